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
// HBM-bound: every tensor is read or written once. A row belongs to one workgroup and stays in its registers; sums over a row
// are taken in an order that depends on its width alone, so that a row's results never depend on its batch. Sums over rows:
// a workgroup of the backward takes every G-th row (G a function of the row count), keeps its sums in registers, and a second
// launch adds the G of them in a fixed order.
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

// Eight values of a vector whose type is that of the block, or fp32.
template <int A>
__device__ __forceinline__ void load_either(const void* p, int64_t base, bool wide, int col, int cols, float (&out)[8]) {
  if (wide) {
    RowVector<RLK_DTYPE_FP32> v;
    v.load_edge<false>(reinterpret_cast<const float*>(p) + base, col / 8, cols);
    v.unpack(out);
  } else {
    RowVector<A> v;
    v.template load_edge<false>(reinterpret_cast<const typename LogitElem<A>::type*>(p) + base, col / 8, cols);
    v.unpack(out);
  }
}
template <int A>
__device__ __forceinline__ float load_one(const void* p, int64_t at, bool wide) {
  return wide ? reinterpret_cast<const float*>(p)[at] : LogitElem<A>::to_float(reinterpret_cast<const typename LogitElem<A>::type*>(p)[at]);
}

template <int THREADS>
struct RowSum {
  static constexpr int kWaves = THREADS / kWave;
  // The sum over the workgroup's threads, in all of them: butterflies over the lanes, then the waves ascending. One barrier: a slot
  // is written again only behind another one.
  template <int N>
  static __device__ __forceinline__ void over(float (&v)[N], float (*slot)[kWaves]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int offset = 32; offset > 0; offset >>= 1) v[n] = v[n] + __shfl_xor(v[n], offset);
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
};

// A: type of block, normed and (where they are not fp32) weights and gate. R: type of the residual. C: vectors of eight columns
// per thread.
template <int A, int R, int THREADS, int C>
__global__ __launch_bounds__(THREADS) void norm_forward_kernel(NormArgs a) {
  using EA = typename LogitElem<A>::type;
  using ER = typename LogitElem<R>::type;
  __shared__ float slots[2][1][RowSum<THREADS>::kWaves];
  const int64_t row = a.first_row + blockIdx.x;
  const float inv_width = 1.0f / (float)a.H;
  RowVector<A> raw_block[C];
  RowVector<R> raw_residual[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * THREADS + (int)threadIdx.x) * 8;
    if (col >= a.H) continue;
    if (a.block) raw_block[c].template load_edge<false>(reinterpret_cast<const EA*>(a.block) + row * a.ld_block, col / 8, a.H);
    raw_residual[c].template load_edge<false>(reinterpret_cast<const ER*>(a.residual) + row * a.ld_residual, col / 8, a.H);
  }
  float x[C][8], t[C][8];
  float sum[1] = {0.f};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * THREADS + (int)threadIdx.x) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] = t[c][i] = 0.f;
    if (col >= a.H) continue;
    if (a.block) raw_block[c].unpack(x[c]);
    raw_residual[c].unpack(t[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(x[c][i], x[c][i], sum[0]);
  }
  float r1 = 1.f;
  if (a.w_post) {
    RowSum<THREADS>::over(sum, slots[0]);
    r1 = 1.0f / sqrtf(__builtin_fmaf(sum[0], inv_width, a.eps));
  }
  const float token_gate = a.gate_kind == kTokenGate ? load_one<A>(a.gate, row * a.ld_gate, a.gate_wide) : 1.f;
  sum[0] = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * THREADS + (int)threadIdx.x) * 8;
    if (col >= a.H) continue;
    if (a.block) {
      if (a.w_post) {
        float w[8];
        load_either<A>(a.w_post, 0, a.post_wide, col, a.H, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] = x[c][i] * r1 * w[i];
      }
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = token_gate;
      if (a.gate_kind == kChannelGate) load_either<A>(a.gate, 0, a.gate_wide, col, a.H, g);
      if (a.gate_kind == kFullGate) load_either<A>(a.gate, row * a.ld_gate, a.gate_wide, col, a.H, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[c][i] = __builtin_fmaf(a.scale * g[i], x[c][i], t[c][i]);
    }
    if (a.total) {
      RowVector<R> out;
      out.pack(t[c]);
      out.template store_edge<false>(reinterpret_cast<ER*>(a.total) + row * a.H, col, a.H);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(t[c][i], t[c][i], sum[0]);
  }
  float r2 = 0.f;
  if (a.w_pre) {
    RowSum<THREADS>::over(sum, slots[1]);
    r2 = 1.0f / sqrtf(__builtin_fmaf(sum[0], inv_width, a.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * THREADS + (int)threadIdx.x) * 8;
      if (col >= a.H) continue;
      float w[8];
      load_either<A>(a.w_pre, 0, a.pre_wide, col, a.H, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = t[c][i] * r2 * w[i];
      RowVector<A> out;
      out.pack(w);
      out.template store_edge<false>(reinterpret_cast<EA*>(a.normed) + row * a.H, col, a.H);
    }
  }
  if (a.rstd && threadIdx.x == 0) {
    a.rstd[row] = r1;
    a.rstd[a.T + row] = r2;
  }
}

template <int A, int R, int THREADS, int C>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormArgs a) {
  using EA = typename LogitElem<A>::type;
  using ER = typename LogitElem<R>::type;
  __shared__ float slots[2][3][RowSum<THREADS>::kWaves];  // rows take turns: a row may pass one barrier only
  int turn = 0;
  const float inv_width = 1.0f / (float)a.H;
  const bool token_sum = a.gate_kind == kTokenGate && a.d_gate;
  float sum_pre[C][8], sum_post[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum_pre[c][i] = sum_post[c][i] = 0.f;

  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, turn ^= 1) {
    RowVector<A> raw_block[C], raw_normed[C];
    RowVector<R> raw_residual[C], raw_total[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * THREADS + (int)threadIdx.x) * 8;
      if (col >= a.H) continue;
      if (a.block) raw_block[c].template load_edge<false>(reinterpret_cast<const EA*>(a.block) + row * a.ld_block, col / 8, a.H);
      raw_residual[c].template load_edge<false>(reinterpret_cast<const ER*>(a.residual) + row * a.ld_residual, col / 8, a.H);
      if (a.g_normed) raw_normed[c].template load_edge<false>(reinterpret_cast<const EA*>(a.g_normed) + row * a.H, col / 8, a.H);
      if (a.g_total) raw_total[c].template load_edge<false>(reinterpret_cast<const ER*>(a.g_total) + row * a.H, col / 8, a.H);
    }
    const float r1 = a.rstd[row], r2 = a.rstd[a.T + row];
    const float token_gate = a.gate_kind == kTokenGate ? load_one<A>(a.gate, row * a.ld_gate, a.gate_wide) : 1.f;
    // h2: total, then total * r2; d: g_normed * w_pre, then d_total, then d_u * w_post
    float h1[C][8], h2[C][8], d[C][8], g[C][8];
    float dot[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * THREADS + (int)threadIdx.x) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h1[c][i] = h2[c][i] = d[c][i] = 0.f;
        g[c][i] = token_gate;
      }
      if (col >= a.H) continue;
      raw_residual[c].unpack(h2[c]);
      if (a.block) {
        raw_block[c].unpack(h1[c]);
        if (a.gate_kind == kChannelGate) load_either<A>(a.gate, 0, a.gate_wide, col, a.H, g[c]);
        if (a.gate_kind == kFullGate) load_either<A>(a.gate, row * a.ld_gate, a.gate_wide, col, a.H, g[c]);
        float w[8];
        if (a.w_post) {
          load_either<A>(a.w_post, 0, a.post_wide, col, a.H, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) h1[c][i] = h1[c][i] * r1;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h2[c][i] = __builtin_fmaf(a.scale * g[c][i], h1[c][i] * w[i], h2[c][i]);
      }
      if (a.g_normed) {
        float w[8];
        raw_normed[c].unpack(d[c]);
        load_either<A>(a.w_pre, 0, a.pre_wide, col, a.H, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h2[c][i] = h2[c][i] * r2;
          sum_pre[c][i] = __builtin_fmaf(d[c][i], h2[c][i], sum_pre[c][i]);
          d[c][i] = d[c][i] * w[i];
          dot[0] = __builtin_fmaf(d[c][i], h2[c][i], dot[0]);
        }
      }
    }
    if (a.g_normed) RowSum<THREADS>::over(dot, slots[turn]);
    const float mean = dot[0] * inv_width;
    float sums[2] = {0.f, 0.f};  // of b h1, and of the token gate's gradient
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * THREADS + (int)threadIdx.x) * 8;
      if (col >= a.H) continue;
      float up[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) up[i] = 0.f;
      if (a.g_total) raw_total[c].unpack(up);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[c][i] = a.g_normed ? __builtin_fmaf(r2, __builtin_fmaf(-h2[c][i], mean, d[c][i]), up[i]) : up[i];
      if (a.d_residual) {
        RowVector<R> out;
        out.pack(d[c]);
        out.template store_edge<false>(reinterpret_cast<ER*>(a.d_residual) + row * a.H, col, a.H);
      }
      if (!a.block) continue;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.f;
      if (a.w_post) load_either<A>(a.w_post, 0, a.post_wide, col, a.H, w);
      float dg[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float scaled = a.scale * d[c][i];
        const float shared = scaled * h1[c][i];
        dg[i] = shared * w[i];
        sums[1] = sums[1] + dg[i];
        // a channel gate is the same in every row: it is multiplied to the sum
        sum_post[c][i] = a.gate_kind == kChannelGate ? sum_post[c][i] + shared : __builtin_fmaf(shared, g[c][i], sum_post[c][i]);
        d[c][i] = scaled * g[c][i] * w[i];
        sums[0] = __builtin_fmaf(d[c][i], h1[c][i], sums[0]);
      }
      if (a.gate_kind == kFullGate && a.d_gate) {
        if (a.gate_wide) {
          RowVector<RLK_DTYPE_FP32> out;
          out.pack(dg);
          out.store_edge<false>(reinterpret_cast<float*>(a.d_gate) + row * a.H, col, a.H);
        } else {
          RowVector<A> out;
          out.pack(dg);
          out.template store_edge<false>(reinterpret_cast<EA*>(a.d_gate) + row * a.H, col, a.H);
        }
      }
    }
    if (a.w_post || token_sum) RowSum<THREADS>::over(sums, slots[turn] + 1);
    if (token_sum && threadIdx.x == 0) {
      if (a.gate_wide) reinterpret_cast<float*>(a.d_gate)[row] = sums[1];
      else reinterpret_cast<EA*>(a.d_gate)[row] = LogitElem<A>::from_float(sums[1]);
    }
    if (a.d_block) {
      const float mean1 = sums[0] * inv_width;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * THREADS + (int)threadIdx.x) * 8;
        if (col >= a.H) continue;
        if (a.w_post) {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[c][i] = r1 * __builtin_fmaf(-h1[c][i], mean1, d[c][i]);
        }
        RowVector<A> out;
        out.pack(d[c]);
        out.template store_edge<false>(reinterpret_cast<EA*>(a.d_block) + row * a.H, col, a.H);
      }
    }
  }
  float* mine = a.part + (int64_t)blockIdx.x * a.H;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * THREADS + (int)threadIdx.x) * 8;
    if (col >= a.H) continue;
    RowVector<RLK_DTYPE_FP32> out;
    if (a.sum_pre) {
      out.pack(sum_pre[c]);
      out.store_edge<false>(mine, col, a.H);
    }
    if (a.sum_post) {
      out.pack(sum_post[c]);
      out.store_edge<false>(mine + (int64_t)gridDim.x * a.H, col, a.H);
    }
  }
}

// The sums over rows: column by column, 16 waves of a workgroup take every 16th of the G parts, then ascending over the waves.
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

// Threads of a workgroup: eight columns each up to 8192, in whole waves of a power of two.
static int norm_threads(int H) {
  int threads = 64;
  while (threads < 1024 && threads * 8 < H) threads *= 2;
  return threads;
}

// Workgroups of the backward: as many as the chip holds at 16 waves to a compute unit.
static int norm_groups(int64_t T, int H) {
  const int64_t most = (int64_t)device_cu_count() * (1024 / norm_threads(H));
  return (int)(T < most ? T : most);
}

size_t block_norm_workspace_bytes(int64_t T, int H) { return T > 0 ? (size_t)2 * norm_groups(T, H) * H * sizeof(float) : 0; }

template <int A, int R, int THREADS, int C>
static void launch_norm_shape(NormArgs a, bool backward, hipStream_t stream) {
  if (backward) {
    hipLaunchKernelGGL((norm_backward_kernel<A, R, THREADS, C>), dim3((unsigned)norm_groups(a.T, a.H)), dim3(THREADS), 0, stream, a);
  } else {
    constexpr int64_t kMost = 0x7fffffff / THREADS;  // (a launch has fewer than 2^32 threads)
    for (; a.first_row < a.T; a.first_row += kMost) {
      const int64_t some = a.T - a.first_row < kMost ? a.T - a.first_row : kMost;
      hipLaunchKernelGGL((norm_forward_kernel<A, R, THREADS, C>), dim3((unsigned)some), dim3(THREADS), 0, stream, a);
    }
  }
}

template <int A, int R>
static hipError_t launch_norm(const NormArgs& a, bool backward, hipStream_t stream) {
  switch (norm_threads(a.H)) {
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
