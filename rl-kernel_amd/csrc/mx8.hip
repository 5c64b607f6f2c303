// Eight-bit copies of activations for gfx950, and SwiGLU that keeps its operands in them for its backward.
//
// A run of 32 columns of a row shares a scale, a power of two: 2^e with e = floor(log2 of its largest magnitude) - 6, at least
// -126. Its values are whole numbers of scales in [-127, 127], the nearest ones (halves to even), held as int8; the scale as the
// byte e + 127. Whole numbers and not an eight-bit floating type: within a run what counts is the error against its largest value,
// 2^-7 of it at most, where three bits of significand are 2^-4 off for every value (normal values: 39 against 31 dB). A power
// of two, because products with it are exact: code * scale is a bf16 number, so the backward of the copies is the backward of
// bf16 tensors, bit for bit. A run with a value that is not finite gets the byte 255 and is NaN throughout.
//
// HBM-bound. A thread takes 16 columns (32 bytes of bf16, one 16-byte store of codes) and shares a run with its neighbour. bf16: 4120 x 4096
// encoded in 11.2 us, decoded in 11.9 (51 MB: 4.5 and 4.3 TB/s), 4096 x 12288 SwiGLU 74 us forward, 76 backward (406 MB: 5.5 and 5.3 TB/s).
// Through the codes a training step moves 8 bytes of an element forward and 8 backward where bf16 tensors take 6 and 10, and keeps 2 and a
// sixteenth in place of 4 (or 6 with the activation).
#include "logits_vector.h"

namespace rlk {

constexpr int kRunCols = 32;
constexpr int kThreadCols = 16;
constexpr int kMx8Threads = 256;

typedef u32x4_t u32x4_at1_t __attribute__((aligned(1)));

// n / d for n < 2^31 by a product (d is the pieces of a row, the same for a whole launch).
struct Divider {
  uint32_t factor, shift, d;
};
static Divider divider(uint32_t d) {
  uint32_t shift = 0;
  while (((uint64_t)1 << shift) < d) ++shift;
  const uint64_t factor = (((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1;
  return {(uint32_t)factor, shift, d};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider& by) { return (__umulhi(n, by.factor) + n) >> by.shift; }

// Sixteen columns of a row, as loaded.
template <int ELEM>
struct Columns16 {
  RowVector<ELEM> half[2];
  __device__ __forceinline__ void load(const typename LogitElem<ELEM>::type* row, int col, int cols) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (col + 8 * h < cols) half[h].template load_edge<false>(row, col / 8 + h, cols);
  }
  __device__ __forceinline__ void unpack(int col, int cols, float (&v)[16]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[8];
      half[h].unpack(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * h + i] = col + 8 * h + i < cols ? y[i] : 0.f;
    }
  }
  __device__ __forceinline__ void pack(const float (&v)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[8 * h + i];
      half[h].pack(y);
    }
  }
  __device__ __forceinline__ void store(typename LogitElem<ELEM>::type* row, int col, int cols) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) half[h].template store_edge<false>(row, col + 8 * h, cols);
  }
};

__device__ __forceinline__ u32x4_t load_codes(const int8_t* row, int col, int cols) {
  if (col + kThreadCols <= cols) return *reinterpret_cast<const u32x4_at1_t*>(row + col);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kThreadCols; ++i)
    if (col + i < cols) w[i >> 2] |= (uint32_t)(uint8_t)row[col + i] << (8 * (i & 3));
  return u32x4_t{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ void store_codes(int8_t* row, int col, int cols, const u32x4_t& codes) {
  if (col + kThreadCols <= cols) {
    *reinterpret_cast<u32x4_at1_t*>(row + col) = codes;
  } else {
#pragma unroll
    for (int i = 0; i < kThreadCols; ++i)
      if (col + i < cols) row[col + i] = (int8_t)(codes[i >> 2] >> (8 * (i & 3)));
  }
}

// The codes of a thread's sixteen values and the scale byte of the run that it shares with the other lane of its pair.
__device__ __forceinline__ u32x4_t encode16(const float (&v)[16], uint32_t& scale_byte) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);  // (the order of magnitudes, NaN on top)
  most = max(most, (uint32_t)__builtin_amdgcn_update_dpp((int)most, (int)most, 0xB1, 0xf, 0xf, false));
  const bool finite = most < 0x7f800000u;
  const int exponent = max((int)(most >> 23) - 6, 1);  // of the scale, + 127
  scale_byte = finite ? (uint32_t)exponent : 255u;
  const float up = __uint_as_float((uint32_t)(254 - exponent) << 23);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float whole = fminf(fmaxf(rintf(v[4 * q + i] * up), -127.f), 127.f);
      w[q] |= ((uint32_t)(int)whole & 0xffu) << (8 * i);
    }
    w[q] = finite ? w[q] : 0u;
  }
  return u32x4_t{w[0], w[1], w[2], w[3]};
}

__device__ __forceinline__ void decode16(const u32x4_t& codes, uint32_t scale_byte, float (&v)[16]) {
  const float scale = scale_byte == 255u ? __builtin_nanf("") : __uint_as_float(scale_byte << 23);
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = (float)(int8_t)(codes[i >> 2] >> (8 * (i & 3))) * scale;
}

struct Mx8Args {
  const void* in[2];  // x; gate, up; or dy
  int64_t ld_in[2];
  void* out[3];  // x; y; or d_gate, d_up, y
  int64_t ld_out;
  int8_t* codes[2];
  uint8_t* scales[2];
  int cols, runs;  // runs: scale bytes of a row
  uint32_t pieces;  // of sixteen columns, over all rows
  Divider per_row;  // pieces of a row: an even number
};

// A thread's piece: its row and first column. Threads without one stay for the exchange with the other lane of their pair.
__device__ __forceinline__ bool piece_of(const Mx8Args& a, int64_t& row, int& col) {
  const uint32_t piece = blockIdx.x * kMx8Threads + threadIdx.x;
  const bool have = piece < a.pieces;
  const uint32_t n = have ? piece : 0;
  row = divide(n, a.per_row);
  col = (int)(n - (uint32_t)row * a.per_row.d) * kThreadCols;
  return have;
}

template <int ELEM>
__global__ __launch_bounds__(kMx8Threads) void mx8_encode_kernel(Mx8Args a) {
  using E = typename LogitElem<ELEM>::type;
  int64_t row;
  int col;
  const bool have = piece_of(a, row, col);
  Columns16<ELEM> x;
  x.load(reinterpret_cast<const E*>(a.in[0]) + row * a.ld_in[0], col, a.cols);
  float v[16];
  x.unpack(col, a.cols, v);
  uint32_t scale;
  const u32x4_t codes = encode16(v, scale);
  if (!have) return;
  store_codes(a.codes[0] + row * a.cols, col, a.cols, codes);
  if ((threadIdx.x & 1) == 0) a.scales[0][row * a.runs + col / kRunCols] = (uint8_t)scale;
}

template <int ELEM>
__global__ __launch_bounds__(kMx8Threads) void mx8_decode_kernel(Mx8Args a) {
  using E = typename LogitElem<ELEM>::type;
  int64_t row;
  int col;
  if (!piece_of(a, row, col)) return;
  float v[16];
  decode16(load_codes(a.codes[0] + row * a.cols, col, a.cols), a.scales[0][row * a.runs + col / kRunCols], v);
  Columns16<ELEM> x;
  x.pack(v);
  x.store(reinterpret_cast<E*>(a.out[0]) + row * a.ld_out, col, a.cols);
}

template <int ELEM>
__global__ __launch_bounds__(kMx8Threads) void mx8_swiglu_forward_kernel(Mx8Args a) {
  using E = typename LogitElem<ELEM>::type;
  int64_t row;
  int col;
  const bool have = piece_of(a, row, col);
  Columns16<ELEM> raw[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) raw[n].load(reinterpret_cast<const E*>(a.in[n]) + row * a.ld_in[n], col, a.cols);
  float g[16], u[16], y[16];
  raw[0].unpack(col, a.cols, g);
  raw[1].unpack(col, a.cols, u);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = swiglu_f32(g[i], u[i]);
  uint32_t scale[2];
  const u32x4_t codes[2] = {encode16(g, scale[0]), encode16(u, scale[1])};
  if (!have) return;
  Columns16<ELEM> out;
  out.pack(y);
  out.store(reinterpret_cast<E*>(a.out[0]) + row * a.cols, col, a.cols);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    store_codes(a.codes[n] + row * a.cols, col, a.cols, codes[n]);
    if ((threadIdx.x & 1) == 0) a.scales[n][row * a.runs + col / kRunCols] = (uint8_t)scale[n];
  }
}

template <int ELEM>
__global__ __launch_bounds__(kMx8Threads) void mx8_swiglu_backward_kernel(Mx8Args a) {
  using E = typename LogitElem<ELEM>::type;
  int64_t row;
  int col;
  if (!piece_of(a, row, col)) return;
  Columns16<ELEM> raw;
  raw.load(reinterpret_cast<const E*>(a.in[0]) + row * a.ld_in[0], col, a.cols);
  u32x4_t codes[2];
  uint32_t scale[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    codes[n] = load_codes(a.codes[n] + row * a.cols, col, a.cols);
    scale[n] = a.scales[n][row * a.runs + col / kRunCols];
  }
  float dy[16], g[16], u[16];
  raw.unpack(col, a.cols, dy);
  decode16(codes[0], scale[0], g);
  decode16(codes[1], scale[1], u);
  // the arithmetic of rlk_swiglu_bwd
  float dg[16], du[16], y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float s = sigmoid_f32(g[i]);
    du[i] = dy[i] * (g[i] * s);
    dg[i] = (dy[i] * u[i]) * (s * (1.0f + g[i] * (1.0f - s)));
    y[i] = (g[i] * s) * u[i];
  }
  Columns16<ELEM> out;
  out.pack(dg);
  out.store(reinterpret_cast<E*>(a.out[0]) + row * a.cols, col, a.cols);
  out.pack(du);
  out.store(reinterpret_cast<E*>(a.out[1]) + row * a.cols, col, a.cols);
  if (a.out[2]) {
    out.pack(y);
    out.store(reinterpret_cast<E*>(a.out[2]) + row * a.cols, col, a.cols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

enum class Mx8Op { kEncode, kDecode, kForward, kBackward };

template <int ELEM>
static void launch_mx8_typed(const Mx8Args& a, Mx8Op op, hipStream_t stream) {
  const dim3 grid((a.pieces + kMx8Threads - 1) / kMx8Threads), block(kMx8Threads);
  if (op == Mx8Op::kEncode) hipLaunchKernelGGL((mx8_encode_kernel<ELEM>), grid, block, 0, stream, a);
  else if (op == Mx8Op::kDecode) hipLaunchKernelGGL((mx8_decode_kernel<ELEM>), grid, block, 0, stream, a);
  else if (op == Mx8Op::kForward) hipLaunchKernelGGL((mx8_swiglu_forward_kernel<ELEM>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((mx8_swiglu_backward_kernel<ELEM>), grid, block, 0, stream, a);
}

// Rows in parts of fewer than 2^31 pieces (a part has 2^35 columns: one launch but for tensors of tens of gigabytes).
static hipError_t launch_mx8(Mx8Args a, int dtype, int64_t rows, Mx8Op op, hipStream_t stream) {
  a.runs = (a.cols + kRunCols - 1) / kRunCols;
  const uint32_t per_row = 2 * (uint32_t)a.runs;
  a.per_row = divider(per_row);
  const int64_t most = 0x7fffff00 / per_row;
  const int64_t bytes = dtype == RLK_DTYPE_FP32 ? 4 : 2;
  for (int64_t first = 0; first < rows; first += most) {
    const int64_t some = rows - first < most ? rows - first : most;
    a.pieces = (uint32_t)(some * per_row);
    if (dtype == RLK_DTYPE_BF16) launch_mx8_typed<RLK_DTYPE_BF16>(a, op, stream);
    else if (dtype == RLK_DTYPE_FP16) launch_mx8_typed<RLK_DTYPE_FP16>(a, op, stream);
    else launch_mx8_typed<RLK_DTYPE_FP32>(a, op, stream);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    for (int n = 0; n < 2; ++n) {
      if (a.in[n]) a.in[n] = reinterpret_cast<const char*>(a.in[n]) + some * a.ld_in[n] * bytes;
      if (a.codes[n]) a.codes[n] += some * a.cols;
      if (a.scales[n]) a.scales[n] += some * a.runs;
    }
    for (int n = 0; n < 3; ++n)
      if (a.out[n]) a.out[n] = reinterpret_cast<char*>(a.out[n]) + some * a.ld_out * bytes;
  }
  return hipSuccess;
}

hipError_t mx8_encode_launch(const void* x, int64_t ld, int dtype, int8_t* codes, uint8_t* scales, int64_t rows, int cols, hipStream_t stream) {
  Mx8Args a{};
  a.in[0] = x;
  a.ld_in[0] = ld;
  a.codes[0] = codes;
  a.scales[0] = scales;
  a.cols = cols;
  return launch_mx8(a, dtype, rows, Mx8Op::kEncode, stream);
}

hipError_t mx8_decode_launch(const int8_t* codes, const uint8_t* scales, void* x, int64_t ld, int dtype, int64_t rows, int cols,
                             hipStream_t stream) {
  Mx8Args a{};
  a.out[0] = x;
  a.ld_out = ld;
  a.codes[0] = const_cast<int8_t*>(codes);
  a.scales[0] = const_cast<uint8_t*>(scales);
  a.cols = cols;
  return launch_mx8(a, dtype, rows, Mx8Op::kDecode, stream);
}

hipError_t mx8_swiglu_forward_launch(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype, void* y, int8_t* gate_codes,
                                     uint8_t* gate_scales, int8_t* up_codes, uint8_t* up_scales, int64_t rows, int cols, hipStream_t stream) {
  Mx8Args a{{gate, up}, {ld_gate, ld_up}, {y, nullptr, nullptr}, cols, {gate_codes, up_codes}, {gate_scales, up_scales}, cols, 0, 0, {}};
  return launch_mx8(a, dtype, rows, Mx8Op::kForward, stream);
}

hipError_t mx8_swiglu_backward_launch(const void* dy, int64_t ld_dy, int dtype, const int8_t* gate_codes, const uint8_t* gate_scales,
                                      const int8_t* up_codes, const uint8_t* up_scales, void* d_gate, void* d_up, void* y, int64_t rows,
                                      int cols, hipStream_t stream) {
  Mx8Args a{{dy, nullptr}, {ld_dy, 0}, {d_gate, d_up, y}, cols, {const_cast<int8_t*>(gate_codes), const_cast<int8_t*>(up_codes)},
            {const_cast<uint8_t*>(gate_scales), const_cast<uint8_t*>(up_scales)}, cols, 0, 0, {}};
  return launch_mx8(a, dtype, rows, Mx8Op::kBackward, stream);
}

}  // namespace rlk
