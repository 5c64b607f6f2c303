// What lies between two blocks of a transformer, for gfx950: the norm of a block's output, its gate and the residual scale,
// the residual sum, and the norm that the next block reads. Forward and backward, a pass over the rows each.
//
//   u      = block * r1 * w_post,   r1 = 1 / sqrt(mean block^2 + eps)       (u = block without a post norm)
//   total  = residual + scale * gate * u                                    (rounded to the residual's type on its way out only)
//   normed = total * r2 * w_pre,    r2 = 1 / sqrt(mean total^2 + eps)
//
// The gate is one value per channel, per token, per element, or none. r1 and r2 are kept for the backward, which computes
// total again from the inputs (as many bytes as reading it would be, and unrounded):
//   h2 = total r2;  a = g_normed w_pre;     d_total = g_total + r2 (a - h2 mean(a h2));    d w_pre  = sum over rows of g_normed h2
//   d_u = scale gate d_total;               d_gate = scale u d_total (summed over what the gate is shared by)
//   h1 = block r1;  b = d_u w_post;         d_block = r1 (b - h1 mean(b h1));              d w_post = sum over rows of d_u h1
//
// HBM-bound: every tensor is read or written once (forward, bf16 with an fp32 residual, 4096 x 4096, 201 MB: 41 us = 4.9 TB/s, 33 with
// its inputs in the memory-side cache). A row belongs to one workgroup, or to a part of one, and stays in its registers; sums over a row
// are taken in an order that depends on its width alone, so that a row's results never depend on its batch. Sums over rows: a workgroup of
// the backward takes every G-th row, or group of rows (G a function of the row count), adds them up as it goes, and a second launch adds
// the G of them in a fixed order.
#include "logits_vector.h"

namespace rlk {

enum NormGate { kNoGate = RLK_GATE_NONE, kChannelGate = RLK_GATE_CHANNEL, kTokenGate = RLK_GATE_TOKEN, kFullGate = RLK_GATE_FULL };

struct NormArgs {
  const void* block;     // [T, ld_block] or null: total = residual
  const void* residual;  // [T, ld_residual]
  const void* gate;
  const void* w_post;  // [H] or null: no post norm
  const void* w_pre;   // [H] or null: no normed
  int64_t ld_block, ld_residual, ld_gate;
  void* total;   // [T, H] contiguous, or null
  void* normed;  // [T, H] contiguous, or null
  float* rstd;   // [2][T]: r1, r2; written by the forward, or null
  // backward
  const void* g_total;   // [T, H] contiguous or null (= 0)
  const void* g_normed;  // [T, H] contiguous or null (= 0)
  void* d_block;     // [T, H] or null
  void* d_residual;  // [T, H] or null
  void* d_gate;      // kTokenGate [T], kFullGate [T, H]; or null
  float* part;       // [2][G][H]: sums over rows of d w_pre, and of d w_post without a channel gate's factor
  int64_t T;
  int64_t first_row;  // of a launch of the forward
  int H, gate_kind;
  bool gate_wide, post_wide, pre_wide;  // fp32 where the block's type is narrower
  bool sum_pre, sum_post;               // which sums over rows are wanted
  float eps, scale;
};

// Eight columns of a row, at its end moved to the left (RowVector::load_window). SMALL: the row has fewer; kernels of their own take such
// rows, as the code for single elements, never run, made the forward of 8192 columns a third slower.
template <bool SMALL, int E>
__device__ __forceinline__ void load8(RowVector<E>& v, const typename LogitElem<E>::type* row, int col, int cols) {
  if constexpr (SMALL) v.template load_window<false>(row, col, cols);
  else v.template load_at<false>(row, (uint32_t)min(col, cols - 8));
}
template <bool SMALL, int E>
__device__ __forceinline__ void store8(const RowVector<E>& v, typename LogitElem<E>::type* row, int col, int cols) {
  using T = typename LogitElem<E>::type;
  if constexpr (SMALL) v.template store_edge<false>(row, 0, cols);
  else v.template store<false>(reinterpret_cast<T*>(reinterpret_cast<char*>(row) + (uint32_t)min(col, cols - 8) * (uint32_t)sizeof(T)));
}

// Eight values of a vector whose type is that of the block, or fp32.
template <int A, bool SMALL>
struct EitherVector {
  u32x4_t w[2];
  __device__ __forceinline__ void load(const void* p, int64_t base, bool wide, int col, int cols) {
    if (wide || A == RLK_DTYPE_FP32) {
      RowVector<RLK_DTYPE_FP32> v;
      load8<SMALL>(v, reinterpret_cast<const float*>(p) + base, col, cols);
      w[0] = v.w[0];
      w[1] = v.w[1];
    } else {
      RowVector<A> v;
      load8<SMALL>(v, reinterpret_cast<const typename LogitElem<A>::type*>(p) + base, col, cols);
      w[0] = v.w[0];
    }
  }
  __device__ __forceinline__ void unpack(bool wide, float (&out)[8]) const {
    if (wide || A == RLK_DTYPE_FP32) {
      RowVector<RLK_DTYPE_FP32> v;
      v.w[0] = w[0];
      v.w[1] = w[1];
      v.unpack(out);
    } else {
      RowVector<A> v;
      v.w[0] = w[0];
      v.unpack(out);
    }
  }
};
template <int A, bool SMALL>
__device__ __forceinline__ void load_either(const void* p, int64_t base, bool wide, int col, int cols, float (&out)[8]) {
  if (wide || A == RLK_DTYPE_FP32) {
    RowVector<RLK_DTYPE_FP32> v;
    load8<SMALL>(v, reinterpret_cast<const float*>(p) + base, col, cols);
    v.unpack(out);
  } else {
    RowVector<A> v;
    load8<SMALL>(v, reinterpret_cast<const typename LogitElem<A>::type*>(p) + base, col, cols);
    v.unpack(out);
  }
}
template <int A>
__device__ __forceinline__ float load_one(const void* p, int64_t at, bool wide) {
  return wide ? reinterpret_cast<const float*>(p)[at] : LogitElem<A>::to_float(reinterpret_cast<const typename LogitElem<A>::type*>(p)[at]);
}

// A row is the work of LANES threads: part of a wave up to 256 columns, so that no lane is idle (262144 rows of 128 columns, a wave
// each / sixteen lanes each: forward 140 / 50 us, backward 253 / 82), else whole waves.
template <int LANES>
struct NormShape {
  static constexpr int kThreads = LANES <= kWave ? 256 : LANES;
  static constexpr int kRows = kThreads / LANES;  // of a workgroup at a time
  static constexpr int kWaves = LANES <= kWave ? 1 : LANES / kWave;  // of a row

  // The sum over the threads of a row, in all of them: within sixteen lanes, across them, then the waves ascending. One barrier:
  // a slot is written again only behind another one.
  template <int N>
  static __device__ __forceinline__ void sum(float (&v)[N], float (*slot)[kWaves]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = v[n] + xor_lane<1>(v[n]);
      v[n] = v[n] + xor_lane<2>(v[n]);
      v[n] = v[n] + dpp<0x141>(v[n]);  // row_half_mirror, row_mirror: the other four, the other eight
      v[n] = v[n] + dpp<0x140>(v[n]);
      if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[n]), __float_as_uint(v[n]), false, false);
        v[n] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }
      if constexpr (LANES >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[n]), __float_as_uint(v[n]), false, false);
        v[n] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }
    }
    if constexpr (kWaves > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) slot[n][wave] = v[n];
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) {
        v[n] = slot[n][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v[n] = v[n] + slot[n][w];
      }
    }
  }
  template <int CONTROL>
  static __device__ __forceinline__ float dpp(float v) {
    const int bits = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, CONTROL, 0xf, 0xf, false));
  }
};

// A thread's c-th vector: eight columns from `col` on. One that would run past the row is moved to its end (RowVector::load_window)
// and shares columns with its neighbour: both compute and store the same values, sums over the row take a column once.
struct NormColumns {
  int col, cols;
  bool have, ragged;
  __device__ __forceinline__ NormColumns(int lane, int lanes, int c, int width)
      : col((c * lanes + lane) * 8), cols(width), have(col < width), ragged(col + 8 > width) {}
  __device__ __forceinline__ void once(const float (&x)[8], float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = x[i];
    if (ragged) {
      const int at = window_of(col, cols);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = at + i >= col && at + i < cols ? x[i] : 0.f;
    }
  }
};

// A: type of block, normed and (where they are not fp32) weights and gate. R: type of the residual. C: vectors of eight columns
// per thread.
template <int A, int R, int LANES, int C, bool SMALL>
__global__ __launch_bounds__(NormShape<LANES>::kThreads) void norm_forward_kernel(NormArgs a) {
  using Shape = NormShape<LANES>;
  using EA = typename LogitElem<A>::type;
  using ER = typename LogitElem<R>::type;
  __shared__ float slots[2][1][Shape::kWaves];
  const int lane = threadIdx.x % LANES;
  const int64_t row = Shape::kRows == 1 ? a.first_row + blockIdx.x : a.first_row + (int64_t)blockIdx.x * Shape::kRows + threadIdx.x / LANES;
  if (Shape::kRows > 1 && row >= a.T) return;
  const float inv_width = 1.0f / (float)a.H;
  RowVector<A> raw_block[C];
  RowVector<R> raw_residual[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const NormColumns at(lane, LANES, c, a.H);
    if (!at.have) continue;
    if (a.block) load8<SMALL>(raw_block[c], reinterpret_cast<const EA*>(a.block) + row * a.ld_block, at.col, a.H);
    load8<SMALL>(raw_residual[c], reinterpret_cast<const ER*>(a.residual) + row * a.ld_residual, at.col, a.H);
  }
  float x[C][8], t[C][8];
  float sum[1] = {0.f};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const NormColumns at(lane, LANES, c, a.H);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] = t[c][i] = 0.f;
    if (!at.have) continue;
    if (a.block) raw_block[c].unpack(x[c]);
    raw_residual[c].unpack(t[c]);
    float v[8];
    at.once(x[c], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(v[i], v[i], sum[0]);
  }
  float r1 = 1.f;
  if (a.w_post) {
    Shape::sum(sum, slots[0]);
    r1 = 1.0f / sqrtf(__builtin_fmaf(sum[0], inv_width, a.eps));
  }
  const float token_gate = a.gate_kind == kTokenGate ? load_one<A>(a.gate, row * a.ld_gate, a.gate_wide) : 1.f;
  sum[0] = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const NormColumns at(lane, LANES, c, a.H);
    if (!at.have) continue;
    if (a.block) {
      if (a.w_post) {
        float w[8];
        load_either<A, SMALL>(a.w_post, 0, a.post_wide, at.col, a.H, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] = x[c][i] * r1 * w[i];
      }
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = token_gate;
      if (a.gate_kind == kChannelGate) load_either<A, SMALL>(a.gate, 0, a.gate_wide, at.col, a.H, g);
      if (a.gate_kind == kFullGate) load_either<A, SMALL>(a.gate, row * a.ld_gate, a.gate_wide, at.col, a.H, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[c][i] = __builtin_fmaf(a.scale * g[i], x[c][i], t[c][i]);
    }
    if (a.total) {
      RowVector<R> out;
      out.pack(t[c]);
      store8<SMALL>(out, reinterpret_cast<ER*>(a.total) + row * a.H, at.col, a.H);
    }
    float v[8];
    at.once(t[c], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(v[i], v[i], sum[0]);
  }
  float r2 = 0.f;
  if (a.w_pre) {
    Shape::sum(sum, slots[1]);
    r2 = 1.0f / sqrtf(__builtin_fmaf(sum[0], inv_width, a.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const NormColumns at(lane, LANES, c, a.H);
      if (!at.have) continue;
      float w[8];
      load_either<A, SMALL>(a.w_pre, 0, a.pre_wide, at.col, a.H, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = t[c][i] * r2 * w[i];
      RowVector<A> out;
      out.pack(w);
      store8<SMALL>(out, reinterpret_cast<EA*>(a.normed) + row * a.H, at.col, a.H);
    }
  }
  if (a.rstd && lane == 0) {
    a.rstd[row] = r1;
    a.rstd[a.T + row] = r2;
  }
}

// What a row's backward needs first, eight columns of a thread.
template <int A, int R, bool FULL, bool SMALL>
struct NormRow {
  RowVector<A> block, normed;
  RowVector<R> residual;
  EitherVector<A, SMALL> gate;  // FULL

  __device__ __forceinline__ void fetch(const NormArgs& a, int64_t row, int col) {
    using EA = typename LogitElem<A>::type;
    using ER = typename LogitElem<R>::type;
    if (a.block) load8<SMALL>(block, reinterpret_cast<const EA*>(a.block) + row * a.ld_block, col, a.H);
    load8<SMALL>(residual, reinterpret_cast<const ER*>(a.residual) + row * a.ld_residual, col, a.H);
    if (a.g_normed) load8<SMALL>(normed, reinterpret_cast<const EA*>(a.g_normed) + row * a.H, col, a.H);
    if constexpr (FULL) gate.load(a.gate, row * a.ld_gate, a.gate_wide, col, a.H);
  }
};

// A workgroup goes through its rows one after the other. Up to 8192 columns (a vector to a thread) the next row is on its way while
// one is worked on, the sums over rows are in registers, and weights and a channel gate wait in LDS, each thread's own columns, to
// be read without a barrier (each row loaded as its turn comes, weights from the caches / so, bf16: 4096 x 8192 110 / 90 us, with an
// fp32 residual 163 / 128, 8192 x 4096 with a full gate 119 / 101 = 5.3 TB/s). Above (two vectors) it is the sums that are in LDS
// (2048 x 16384, sums in registers, most of which spilled / in LDS: 245 / 154 us). A full gate has kernels of its own: its registers
// would have the others spill. Four waves to a SIMD: with fewer the loads of a workgroup have nobody to hide behind.
template <int A, int R, int LANES, int C, bool FULL, bool SMALL>
__global__ __launch_bounds__(NormShape<LANES>::kThreads) __attribute__((amdgpu_waves_per_eu(4))) void norm_backward_kernel(NormArgs a) {
  using Shape = NormShape<LANES>;
  using EA = typename LogitElem<A>::type;
  using ER = typename LogitElem<R>::type;
  constexpr bool kAhead = C == 1;
  constexpr int kPre = 0, kPost = 1, kGate = 2;
  __shared__ float slots[2][3][Shape::kWaves];  // rows take turns: a row may pass one barrier only
  __shared__ f32x4_t own[kAhead ? 6 : 4 * C][Shape::kThreads];
  int turn = 0;
  const int lane = threadIdx.x % LANES;
  const float inv_width = 1.0f / (float)a.H;
  const bool token_sum = a.gate_kind == kTokenGate && a.d_gate;
  auto put = [&](int at, const float (&v)[8]) __attribute__((always_inline)) {
    own[at][threadIdx.x] = f32x4_t{v[0], v[1], v[2], v[3]};
    own[at + 1][threadIdx.x] = f32x4_t{v[4], v[5], v[6], v[7]};
  };
  auto get = [&](int at, float (&v)[8]) __attribute__((always_inline)) {
    const f32x4_t lo = own[at][threadIdx.x], hi = own[at + 1][threadIdx.x];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = lo[i];
      v[4 + i] = hi[i];
    }
  };
  auto weight = [&](int which, int col, float (&w)[8]) __attribute__((always_inline)) {
    if constexpr (kAhead) get(2 * which, w);
    else if (which == kPre) load_either<A, SMALL>(a.w_pre, 0, a.pre_wide, col, a.H, w);
    else if (which == kPost) load_either<A, SMALL>(a.w_post, 0, a.post_wide, col, a.H, w);
    else load_either<A, SMALL>(a.gate, 0, a.gate_wide, col, a.H, w);
  };
  float sum_pre[8], sum_post[8];  // kAhead: else in `own`
#pragma unroll
  for (int i = 0; i < 8; ++i) sum_pre[i] = sum_post[i] = 0.f;
  if constexpr (kAhead) {
    const NormColumns at(lane, LANES, 0, a.H);
    float w[8];
    if (at.have && a.w_pre) {
      load_either<A, SMALL>(a.w_pre, 0, a.pre_wide, at.col, a.H, w);
      put(2 * kPre, w);
    }
    if (at.have && a.w_post) {
      load_either<A, SMALL>(a.w_post, 0, a.post_wide, at.col, a.H, w);
      put(2 * kPost, w);
    }
    if (at.have && a.gate_kind == kChannelGate) {
      load_either<A, SMALL>(a.gate, 0, a.gate_wide, at.col, a.H, w);
      put(2 * kGate, w);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 2 * C; ++c) put(2 * c, sum_pre);
  }

  NormRow<A, R, FULL, SMALL> raw[C];
  const int64_t step = (int64_t)gridDim.x * Shape::kRows;
  int64_t row = Shape::kRows == 1 ? blockIdx.x : (int64_t)blockIdx.x * Shape::kRows + threadIdx.x / LANES;
  if constexpr (kAhead) {
    const NormColumns at(lane, LANES, 0, a.H);
    if (at.have && row < a.T) raw[0].fetch(a, row, at.col);
  }
  for (; row < a.T; row += step, turn ^= 1) {
    const float r1 = a.rstd[row], r2 = a.rstd[a.T + row];
    const float token_gate = a.gate_kind == kTokenGate ? load_one<A>(a.gate, row * a.ld_gate, a.gate_wide) : 1.f;
    if constexpr (!kAhead) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const NormColumns at(lane, LANES, c, a.H);
        if (at.have) raw[c].fetch(a, row, at.col);
      }
    }
    // h1: block * r1 (two vectors: made again from the block where it is used, for want of registers); h2: total, then total * r2;
    // d: g_normed * w_pre, then d_total, then d_u * w_post
    float h1[C][8], h2[C][8], d[C][8];
    auto h1_of = [&](int c, float (&h)[8]) __attribute__((always_inline)) {
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = h1[c][i];
      } else {
        raw[c].block.unpack(h);
        if (a.w_post) {
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = h[i] * r1;
        }
      }
    };
    RowVector<R> raw_total[C];
    EitherVector<A, SMALL> raw_gate[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const NormColumns at(lane, LANES, c, a.H);
#pragma unroll
      for (int i = 0; i < 8; ++i) h1[c][i] = h2[c][i] = d[c][i] = 0.f;
      if (!at.have) continue;
      raw[c].residual.unpack(h2[c]);
      if (kAhead && a.block) raw[c].block.unpack(h1[c]);
      if (a.g_normed) raw[c].normed.unpack(d[c]);
      if (a.g_total) load8<SMALL>(raw_total[c], reinterpret_cast<const ER*>(a.g_total) + row * a.H, at.col, a.H);
      if constexpr (FULL) raw_gate[c] = raw[c].gate;
      if constexpr (kAhead) {
        __builtin_amdgcn_sched_barrier(0);
        raw[c].fetch(a, row + step < a.T ? row + step : row, at.col);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    auto gate_of = [&](int c, int col, float (&g)[8]) __attribute__((always_inline)) {
      if constexpr (FULL) {
        raw_gate[c].unpack(a.gate_wide, g);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = token_gate;
        if (a.gate_kind == kChannelGate) weight(kGate, col, g);
      }
    };
    float dot[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const NormColumns at(lane, LANES, c, a.H);
      if (!at.have) continue;
      if (a.block) {
        float g[8], w[8];
        gate_of(c, at.col, g);
        if (a.w_post) {
          weight(kPost, at.col, w);
          if constexpr (kAhead) {
#pragma unroll
            for (int i = 0; i < 8; ++i) h1[c][i] = h1[c][i] * r1;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = 1.f;
        }
        float h[8];
        h1_of(c, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) h2[c][i] = __builtin_fmaf(a.scale * g[i], h[i] * w[i], h2[c][i]);
      }
      if (a.g_normed) {
        float w[8], v[8];
        weight(kPre, at.col, w);
        if constexpr (!kAhead) get(4 * c, sum_pre);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h2[c][i] = h2[c][i] * r2;
          sum_pre[i] = __builtin_fmaf(d[c][i], h2[c][i], sum_pre[i]);
          d[c][i] = d[c][i] * w[i];
        }
        if constexpr (!kAhead) put(4 * c, sum_pre);
        at.once(d[c], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot[0] = __builtin_fmaf(v[i], h2[c][i], dot[0]);
      }
    }
    if (a.g_normed) Shape::sum(dot, slots[turn]);
    const float mean = dot[0] * inv_width;
    float sums[2] = {0.f, 0.f};  // of b h1, and of the token gate's gradient
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const NormColumns at(lane, LANES, c, a.H);
      if (!at.have) continue;
      float up[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) up[i] = 0.f;
      if (a.g_total) raw_total[c].unpack(up);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[c][i] = a.g_normed ? __builtin_fmaf(r2, __builtin_fmaf(-h2[c][i], mean, d[c][i]), up[i]) : up[i];
      if (a.d_residual) {
        RowVector<R> out;
        out.pack(d[c]);
        store8<SMALL>(out, reinterpret_cast<ER*>(a.d_residual) + row * a.H, at.col, a.H);
      }
      if (!a.block) continue;
      float w[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.f;
      if (a.w_post) weight(kPost, at.col, w);
      gate_of(c, at.col, g);
      if constexpr (!kAhead) get(4 * c + 2, sum_post);
      float dg[8], h[8];
      h1_of(c, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float scaled = a.scale * d[c][i];
        const float shared = scaled * h[i];
        dg[i] = shared * w[i];
        // a channel gate is the same in every row: it is multiplied to the sum
        sum_post[i] = !FULL && a.gate_kind == kChannelGate ? sum_post[i] + shared : __builtin_fmaf(shared, g[i], sum_post[i]);
        d[c][i] = scaled * g[i] * w[i];
      }
      if constexpr (!kAhead) put(4 * c + 2, sum_post);
      if (FULL && a.d_gate) {
        if (a.gate_wide) {
          RowVector<RLK_DTYPE_FP32> out;
          out.pack(dg);
          store8<SMALL>(out, reinterpret_cast<float*>(a.d_gate) + row * a.H, at.col, a.H);
        } else {
          RowVector<A> out;
          out.pack(dg);
          store8<SMALL>(out, reinterpret_cast<EA*>(a.d_gate) + row * a.H, at.col, a.H);
        }
      }
      float v[8];
      at.once(d[c], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[0] = __builtin_fmaf(v[i], h[i], sums[0]);
      if (token_sum) {
        at.once(dg, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[1] = sums[1] + v[i];
      }
    }
    if (a.w_post || token_sum) Shape::sum(sums, slots[turn] + 1);
    if (token_sum && lane == 0) {
      if (a.gate_wide) reinterpret_cast<float*>(a.d_gate)[row] = sums[1];
      else reinterpret_cast<EA*>(a.d_gate)[row] = LogitElem<A>::from_float(sums[1]);
    }
    if (a.d_block) {
      const float mean1 = sums[0] * inv_width;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const NormColumns at(lane, LANES, c, a.H);
        if (!at.have) continue;
        if (a.w_post) {
          float h[8];
          h1_of(c, h);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[c][i] = r1 * __builtin_fmaf(-h[i], mean1, d[c][i]);
        }
        RowVector<A> out;
        out.pack(d[c]);
        store8<SMALL>(out, reinterpret_cast<EA*>(a.d_block) + row * a.H, at.col, a.H);
      }
    }
  }

  // the workgroup's sums over its rows: those of its rows at a time are added in their order, through `own`
  float* mine = a.part + (int64_t)blockIdx.x * a.H;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 ? !a.sum_pre : !a.sum_post) continue;
    float* const to = which == 0 ? mine : mine + (int64_t)gridDim.x * a.H;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const NormColumns at(lane, LANES, c, a.H);
      float total[8];
      if constexpr (!kAhead) {
        get(4 * c + 2 * which, total);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) total[i] = which == 0 ? sum_pre[i] : sum_post[i];
      }
      if constexpr (Shape::kRows > 1) {
        __syncthreads();  // (`own` may still be read)
        put(0, total);
        __syncthreads();
        for (int other = 1; other < Shape::kRows; ++other) {
          const f32x4_t lo = own[0][other * LANES + lane], hi = own[1][other * LANES + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            total[i] = total[i] + lo[i];
            total[4 + i] = total[4 + i] + hi[i];
          }
        }
        if (threadIdx.x >= LANES) continue;
      }
      if (!at.have) continue;
      RowVector<RLK_DTYPE_FP32> out;
      out.pack(total);
      store8<SMALL>(out, to, at.col, a.H);
    }
  }
}

// The sums over rows: column by column, 16 waves of a workgroup take every 16th of the G parts, then ascending over the waves
// (512 parts of 4096 columns, both sums: 5 us).
// Sum 1 is that of scale d_total h1 under a channel gate, which times the gate is d w_post and times w_post d_gate; else d w_post.
struct NormSumArgs {
  const float* part;  // [2][G][H]
  void* d_pre;        // each or null
  void* d_post;
  void* d_gate;
  const void* w_post;  // or null
  const void* gate;    // a channel gate, or null
  int pre_dtype, post_dtype, gate_dtype;
  int G, H;
};
constexpr int kSumWaves = 16;

__device__ __forceinline__ float load_typed(const void* p, int dtype, int at) {
  if (dtype == RLK_DTYPE_FP32) return reinterpret_cast<const float*>(p)[at];
  if (dtype == RLK_DTYPE_BF16) return LogitElem<RLK_DTYPE_BF16>::to_float(reinterpret_cast<const uint16_t*>(p)[at]);
  return LogitElem<RLK_DTYPE_FP16>::to_float(reinterpret_cast<const _Float16*>(p)[at]);
}
__device__ __forceinline__ void store_typed(void* p, int dtype, int at, float v) {
  if (dtype == RLK_DTYPE_FP32) reinterpret_cast<float*>(p)[at] = v;
  else if (dtype == RLK_DTYPE_BF16) reinterpret_cast<uint16_t*>(p)[at] = LogitElem<RLK_DTYPE_BF16>::from_float(v);
  else reinterpret_cast<_Float16*>(p)[at] = LogitElem<RLK_DTYPE_FP16>::from_float(v);
}

__global__ __launch_bounds__(kSumWaves * kWave) void norm_column_sums_kernel(NormSumArgs a) {
  __shared__ float sums[kSumWaves][kWave];
  const bool pre = blockIdx.y == 0;
  if (pre ? a.d_pre == nullptr : (a.d_post == nullptr && a.d_gate == nullptr)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * kWave + lane;
  const float* part = a.part + (int64_t)blockIdx.y * a.G * a.H + col;
  float s = 0.f;
  if (col < a.H) {
#pragma unroll 8
    for (int g = wave; g < a.G; g += kSumWaves) s = s + part[(int64_t)g * a.H];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || col >= a.H) return;
#pragma unroll
  for (int w = 1; w < kSumWaves; ++w) s = s + sums[w][lane];
  if (pre) {
    store_typed(a.d_pre, a.pre_dtype, col, s);
    return;
  }
  if (a.d_post) store_typed(a.d_post, a.post_dtype, col, a.gate ? s * load_typed(a.gate, a.gate_dtype, col) : s);
  if (a.d_gate) store_typed(a.d_gate, a.gate_dtype, col, a.w_post ? s * load_typed(a.w_post, a.post_dtype, col) : s);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Threads of a row: eight columns each up to 8192.
static int norm_lanes(int H) {
  int lanes = 16;
  while (lanes < 1024 && lanes * 8 < H) lanes *= 2;
  return lanes;
}

// Workgroups of the backward: as many as the chip holds at 16 waves to a compute unit.
static int norm_groups(int64_t T, int H) {
  const int lanes = norm_lanes(H), threads = lanes <= kWave ? 256 : lanes;
  const int64_t most = (int64_t)device_cu_count() * (1024 / threads), all = (T + threads / lanes - 1) / (threads / lanes);
  return (int)(all < most ? all : most);
}

size_t block_norm_workspace_bytes(int64_t T, int H) { return T > 0 ? (size_t)2 * norm_groups(T, H) * H * sizeof(float) : 0; }

template <int A, int R, int LANES, int C, bool SMALL = false>
static void launch_norm_shape(NormArgs a, bool backward, hipStream_t stream) {
  using Shape = NormShape<LANES>;
  if (backward) {
    const dim3 grid((unsigned)norm_groups(a.T, a.H)), block(Shape::kThreads);
    if (a.gate_kind == kFullGate) hipLaunchKernelGGL((norm_backward_kernel<A, R, LANES, C, true, SMALL>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((norm_backward_kernel<A, R, LANES, C, false, SMALL>), grid, block, 0, stream, a);
  } else {
    constexpr int64_t kMost = 0x7fffffff / Shape::kThreads;  // (a launch has fewer than 2^32 threads)
    for (; a.first_row < a.T; a.first_row += kMost * Shape::kRows) {
      const int64_t all = (a.T - a.first_row + Shape::kRows - 1) / Shape::kRows;
      const dim3 grid((unsigned)(all < kMost ? all : kMost)), block(Shape::kThreads);
      hipLaunchKernelGGL((norm_forward_kernel<A, R, LANES, C, SMALL>), grid, block, 0, stream, a);
    }
  }
}

template <int A, int R>
static hipError_t launch_norm(const NormArgs& a, bool backward, hipStream_t stream) {
  switch (norm_lanes(a.H)) {
    case 16:
      if (a.H < 8) launch_norm_shape<A, R, 16, 1, true>(a, backward, stream);
      else launch_norm_shape<A, R, 16, 1>(a, backward, stream);
      break;
    case 32: launch_norm_shape<A, R, 32, 1>(a, backward, stream); break;
    case 64: launch_norm_shape<A, R, 64, 1>(a, backward, stream); break;
    case 128: launch_norm_shape<A, R, 128, 1>(a, backward, stream); break;
    case 256: launch_norm_shape<A, R, 256, 1>(a, backward, stream); break;
    case 512: launch_norm_shape<A, R, 512, 1>(a, backward, stream); break;
    default:
      if (a.H <= 8192) launch_norm_shape<A, R, 1024, 1>(a, backward, stream);
      else if (a.H <= RLK_NORM_MAX_WIDTH) launch_norm_shape<A, R, 1024, 2>(a, backward, stream);
      else return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

static hipError_t norm_dispatch(const NormArgs& a, int dtype, int residual_dtype, bool backward, hipStream_t stream) {
  if (dtype == RLK_DTYPE_BF16 && residual_dtype == dtype) return launch_norm<RLK_DTYPE_BF16, RLK_DTYPE_BF16>(a, backward, stream);
  if (dtype == RLK_DTYPE_BF16 && residual_dtype == RLK_DTYPE_FP32) return launch_norm<RLK_DTYPE_BF16, RLK_DTYPE_FP32>(a, backward, stream);
  if (dtype == RLK_DTYPE_FP16 && residual_dtype == dtype) return launch_norm<RLK_DTYPE_FP16, RLK_DTYPE_FP16>(a, backward, stream);
  if (dtype == RLK_DTYPE_FP16 && residual_dtype == RLK_DTYPE_FP32) return launch_norm<RLK_DTYPE_FP16, RLK_DTYPE_FP32>(a, backward, stream);
  if (dtype == RLK_DTYPE_FP32 && residual_dtype == dtype) return launch_norm<RLK_DTYPE_FP32, RLK_DTYPE_FP32>(a, backward, stream);
  return hipErrorInvalidValue;
}

static NormArgs norm_args(const rlk_block_norm* n) {
  NormArgs a{};
  a.block = n->block;
  a.residual = n->residual;
  a.gate = n->gate;
  a.w_post = n->post_weight;
  a.w_pre = n->pre_weight;
  a.ld_block = n->block_row_stride;
  a.ld_residual = n->residual_row_stride;
  a.ld_gate = n->gate_row_stride;
  a.T = n->tokens;
  a.H = n->width;
  a.gate_kind = n->block ? n->gate_kind : RLK_GATE_NONE;
  a.gate_wide = n->gate_dtype == RLK_DTYPE_FP32;
  a.post_wide = n->post_dtype == RLK_DTYPE_FP32;
  a.pre_wide = n->pre_dtype == RLK_DTYPE_FP32;
  a.eps = n->eps;
  a.scale = n->residual_scale;
  a.rstd = n->rstd;
  return a;
}

hipError_t block_norm_forward_launch(const rlk_block_norm* n, void* total, void* normed, hipStream_t stream) {
  NormArgs a = norm_args(n);
  a.total = total;
  a.normed = normed;
  return norm_dispatch(a, n->dtype, n->residual_dtype, false, stream);
}

hipError_t block_norm_backward_launch(const rlk_block_norm* n, const void* g_total, const void* g_normed, void* d_block, void* d_residual,
                                      void* d_gate, void* d_post_weight, void* d_pre_weight, void* workspace, hipStream_t stream) {
  NormArgs a = norm_args(n);
  a.g_total = g_total;
  a.g_normed = n->pre_weight ? g_normed : nullptr;
  a.d_block = d_block;
  a.d_residual = d_residual;
  a.d_gate = d_gate;
  a.part = reinterpret_cast<float*>(workspace);
  const bool channel = a.gate_kind == kChannelGate;
  a.sum_pre = d_pre_weight != nullptr;
  a.sum_post = d_post_weight != nullptr || (d_gate != nullptr && channel);
  hipError_t err = norm_dispatch(a, n->dtype, n->residual_dtype, true, stream);
  if (err != hipSuccess || !(a.sum_pre || a.sum_post)) return err;
  const NormSumArgs s{a.part, d_pre_weight, d_post_weight, channel ? d_gate : nullptr, a.w_post, channel ? a.gate : nullptr, n->pre_dtype,
                      n->post_dtype, n->gate_dtype, norm_groups(a.T, a.H), a.H};
  hipLaunchKernelGGL(norm_column_sums_kernel, dim3((unsigned)((a.H + kWave - 1) / kWave), 2), dim3(kSumWaves * kWave), 0, stream, s);
  return hipGetLastError();
}

}  // namespace rlk
