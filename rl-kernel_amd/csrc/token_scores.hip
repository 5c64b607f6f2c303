// Scores of given tokens from materialised logits for gfx950: log-probability, log-sum-exp, entropy of the row's
// distribution and its most likely alternatives, with the gradient of the logits.
//
//   y_c = z_c / temperature over the real columns c;   M = max y;   S = sum e(y_c - M);   W = sum e(y_c - M) (y_c - M)
//   lse = M + log S;   logp = y_target - lse;   entropy = log S - W / S    (both terms >= 0: nothing cancels)
//   alternatives: the top_k columns by (z descending, column ascending), their log-probabilities y - lse
//
// One pass over the logits. The running (M, S) follow the reduction contract of logits_logp.hip with 64 tiles to a row
// (tile = ceil(V / 64) columns), so that logp and lse are that entry's bits wherever 64 divides V and the logits are numbers; W is
// carried beside S: a state (m, s, w) seen from a larger maximum n is (s e(m - n), e(m - n) (w + s (m - n))).
//
// The alternatives cost the pass two instructions for each vector of eight logits. A lane of a tile sees a fixed slice of
// the row (every sixteenth vector of its tile), 1024 slices in all, and notes the largest logit of each, the vector
// that held it first, and the largest logit outside of that vector. Under the order (value descending, column ascending) the k
// best columns of a row lie in the k slices whose best columns come first: a column outside of them has k better ones. So a
// second, small kernel picks those slices, reads of each that one vector again (the whole slice only where another of its
// vectors reaches the k-th slice's best as well) and ranks what does. It is right however a row's values are spread: equal
// logits, rows of one value and masked rows take the same steps, some of them more often.
//
// HBM-bound: a logit is read once.
#include "logits_vector.h"

namespace rlk {

constexpr int kScoreTiles = 64;
constexpr int kScoreSlices = kScoreTiles * kTileLanes;
constexpr int kGroupTiles = 4 * kTilesPerWave;  // of a workgroup: a row has four
constexpr int kScorePlanes = 4;  // max, sum, target, weighted sum: stats[row][plane][tile]

struct ScoreArgs {
  const void* logits;
  int64_t row_stride;  // elements
  const int64_t* target;     // [T] columns
  const float* temperature;  // [T] or null
  float* stats;              // [T][kScorePlanes][kScoreTiles]
  uint32_t* best;   // [T][kScoreSlices] largest logit of the slice (ordered bits), 0 for a slice without columns
  uint32_t* where;  // [T][kScoreSlices] the upper half of the largest logit in its other vectors | number of the first vector that holds the best
  int T, V, real, tile_size;
  int64_t streamed;  // workgroups, in the order of their ids, that read past the caches
};

// Whole numbers in the order of the values (-0 as +0); a NaN, which the maxima of a row pass over, counts as -inf.
__device__ __forceinline__ uint32_t ordered_bits(float v) {
  v = v == v ? v + 0.f : kNegInf;
  const uint32_t b = __float_as_uint(v);
  return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered_bits(uint32_t o) {
  return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu));
}

struct ScoreState {
  float m, s, w;  // scaled maximum, sum, weighted sum
  float raw;      // largest logit before the temperature
  float other;    // largest logit outside of the first vector that held it
  int at;         // that vector
};

// The eight logits of vector g folded into a lane's state. The maximum is taken before the temperature (times a positive
// number it is the maximum of the products, to the bit), so that alternatives are told apart that scaling makes equal. A NaN stays in
// the sums, wherever it stands (kLowest).
template <bool HAS_TEMP, bool TOP>
__device__ __forceinline__ void fold_score_vector(float (&y)[8], float inv_t, int g, ScoreState& st) {
  const float most = max3_f32(max3_f32(max3_f32(y[0], y[1], y[2]), y[3], y[4]), y[5], y[6]);
  if constexpr (TOP) {
    const float here = max3_f32(most, y[7], y[7]);
    st.at = here > st.raw ? g : st.at;
    st.other = __builtin_amdgcn_fmed3f(here, st.raw, st.other);  // (other <= raw: the second of the three)
  }
  st.raw = max3_f32(most, y[7], st.raw);
  float n = st.raw;
  if constexpr (HAS_TEMP) {
    n = n * inv_t;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * inv_t;
  }
  const float from = fmaxf(n, kLowest);
  float d = y[0] - from;
  float e = pinned_exp(d);
  float sum = e, weighted = e * fmaxf(d, kFarBelow);  // (a masked logit is -inf below: 0 times that is no number)
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    d = y[i] - from;
    e = pinned_exp(d);
    sum = sum + e;
    weighted = __builtin_fmaf(e, fmaxf(d, kFarBelow), weighted);
  }
  const float back = st.m - from;
  const float shrink = pinned_exp(back);
  st.w = __builtin_fmaf(shrink, __builtin_fmaf(st.s, fmaxf(back, kFarBelow), st.w), weighted);
  st.s = st.s * shrink + sum;
  st.m = n;
}

// merge_lane_states of logits_logp.hip with the weighted sum beside.
template <int OFFSET>
__device__ __forceinline__ void merge_score_lanes(int lane, ScoreState& st) {
  const float om = xor_lane<OFFSET>(st.m), os = xor_lane<OFFSET>(st.s), ow = xor_lane<OFFSET>(st.w);
  const float n = fmaxf(st.m, om), from = fmaxf(n, kLowest);
  const float my_shrink = pinned_exp(st.m - from), other_shrink = pinned_exp(om - from);
  const float mine = st.s * my_shrink, theirs = os * other_shrink;
  const float my_w = my_shrink * __builtin_fmaf(st.s, fmaxf(st.m - from, kFarBelow), st.w);
  const float their_w = other_shrink * __builtin_fmaf(os, fmaxf(om - from, kFarBelow), ow);
  // the lower lane's term first on both sides, so that both lanes add in the same order
  st.s = (lane & OFFSET) ? theirs + mine : mine + theirs;
  st.w = (lane & OFFSET) ? their_w + my_w : my_w + their_w;
  st.m = n;
}

// HBM-bound: 2048 x 131072 bf16 104 us = 5.2 TB/s, with alternatives 115 (logits that rotate through 1.6 GB); one row of 151936 7 us, launch
// and latency. (A form for few rows, one wave to a workgroup and eight vectors of a lane on their way, took 0.3 us less up to 64 rows of
// 151936 bf16 logits, 0.3 to 2 more at the other sizes.)
template <int ELEM, bool HAS_TEMP, bool TOP, bool NT>
__device__ __forceinline__ void score_tiles(const ScoreArgs& a) {
  using E = typename LogitElem<ELEM>::type;
  constexpr int kBatch = 4;                   // vectors that a lane has on their way
  constexpr int kStep = kTileLanes * kBatch;  // vectors of a tile per batch
  const int row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & (kTileLanes - 1);
  const int grp = lane / kTileLanes;
  const E* row_ptr = reinterpret_cast<const E*>(a.logits) + (int64_t)row * a.row_stride;
  const float inv_t = HAS_TEMP ? 1.0f / a.temperature[row] : 1.0f;
  const int tile = blockIdx.y * kGroupTiles + wave * kTilesPerWave + grp;
  const int64_t lo64 = (int64_t)tile * a.tile_size, hi64 = lo64 + a.tile_size;
  const int lo_col = lo64 < a.real ? (int)lo64 : a.real;
  const int hi_col = hi64 < a.real ? (int)hi64 : a.real;
  const int g0 = lo_col / 8;
  const int g1 = hi_col > lo_col ? (hi_col + 7) / 8 : g0;
  const int g_last = g1 > g0 ? g1 - 1 : 0;  // a valid vector to clamp loads to
  // Batches in which all four vectors of every lane are whole vectors of the lane's tile need no masks, but for the first vector
  // of a tile, which may start before it.
  const int g_whole = (hi_col % 8) ? g1 - 1 : g1;
  const int my_clean = g_whole > g0 ? (g_whole - g0) / kStep : 0;
  const int my_slots = (g1 - g0 + kTileLanes - 1) / kTileLanes;
  int clean = __builtin_amdgcn_readlane(my_clean, 0), slots = __builtin_amdgcn_readlane(my_slots, 0);
#pragma unroll
  for (int other = kTileLanes; other < kWave; other += kTileLanes) {  // uniform over the wave's four tiles
    clean = min(clean, __builtin_amdgcn_readlane(my_clean, other));
    slots = max(slots, __builtin_amdgcn_readlane(my_slots, other));
  }

  ScoreState st{kNegInf, 0.f, 0.f, kNegInf, kNegInf, g0 + l16};
  int g = g0 + l16;  // this lane's next vector
  // The loads rotate through the raw vectors: a vector's registers are free once it is unpacked, and the same vector of the next
  // batch is fetched into them before the fold, so a lane always has that many loads, or one less, in flight. (Behind the
  // tile its last vector is fetched again.)
  RowVector<ELEM> raw[kBatch];
  auto fetch = [&](int u, int at) __attribute__((always_inline)) {
    raw[u].template load_window<NT>(row_ptr, (at < g1 ? at : g_last) * 8, a.V);
  };
  auto fetch_of_many = [&](int u, int at) __attribute__((always_inline)) {  // of a row that has a window to spare
    raw[u].template load_at<NT>(row_ptr, (uint32_t)min((at < g1 ? at : g_last) * 8, a.V - 8));
  };
#pragma unroll
  for (int u = 0; u < kBatch; ++u) fetch(u, g + u * kTileLanes);
  const int64_t target = a.target[row];
  const bool holds_target = l16 == 0 && target >= lo_col && target < hi_col;
  E target_logit{};
  if (holds_target) target_logit = row_ptr[target];
  int b = 0;
  for (; b < clean; ++b, g += kStep) {  // without a branch between the folds
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int gu = g + u * kTileLanes;
      float y[8];
      raw[u].unpack(y);
      __builtin_amdgcn_sched_barrier(0);
      fetch_of_many(u, gu + kStep);
      if (u == 0) {
        const int lo = lo_col - gu * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = i >= lo ? y[i] : kNegInf;
      }
      fold_score_vector<HAS_TEMP, TOP>(y, inv_t, gu, st);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The rest, mostly what is on its way, a vector at a time: the loads move up through the registers.
#pragma unroll 1
  for (int slot = b * kBatch; slot < slots; ++slot, g += kTileLanes) {
    float y[8];
    raw[0].unpack(y);
#pragma unroll
    for (int u = 0; u + 1 < kBatch; ++u) raw[u] = raw[u + 1];
    if (slot + kBatch < slots) fetch(kBatch - 1, g + kStep);
    const int first = window_of(g * 8, a.V);
    const int lo = max(lo_col, g * 8) - first;  // columns [lo, hi) of the window count: none of a vector behind the tile
    const int hi = g < g1 ? min(hi_col, g * 8 + 8) - first : lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (uint32_t)(i - lo) < (uint32_t)(hi - lo) ? y[i] : kNegInf;
    fold_score_vector<HAS_TEMP, TOP>(y, inv_t, g, st);  // a vector of -inf changes nothing
  }
  if constexpr (TOP) {
    const int64_t slice = (int64_t)row * kScoreSlices + tile * kTileLanes + l16;
    a.best[slice] = g0 + l16 < g1 ? ordered_bits(st.raw) : 0u;
    a.where[slice] = (ordered_bits(st.other) & 0xffff0000u) | (uint32_t)((st.at - g0 - l16) / kTileLanes);
  }
  merge_score_lanes<8>(lane, st);
  merge_score_lanes<4>(lane, st);
  merge_score_lanes<2>(lane, st);
  merge_score_lanes<1>(lane, st);
  if (l16 == 0) {
    float zt = holds_target ? LogitElem<ELEM>::to_float(target_logit) : 0.f;
    if (HAS_TEMP) zt = holds_target ? zt * inv_t : zt;
    float* out = a.stats + (int64_t)row * kScorePlanes * kScoreTiles + tile;
    out[0] = st.m;
    out[kScoreTiles] = st.s;
    out[2 * kScoreTiles] = zt;
    out[3 * kScoreTiles] = st.w;
  }
}

template <int ELEM, bool HAS_TEMP, bool TOP>
__global__ __launch_bounds__(256) void score_tiles_kernel(ScoreArgs a) {
  if ((int64_t)blockIdx.y * gridDim.x + blockIdx.x < a.streamed) {
    score_tiles<ELEM, HAS_TEMP, TOP, true>(a);
  } else {
    score_tiles<ELEM, HAS_TEMP, TOP, false>(a);
  }
}

// ---------------------------------------------------------------------------
// A wave per row, a workgroup of its own (four to a workgroup: 1 us more at 16 to 64 rows, the same at 2048): the tiles of the row merged, and
// its alternatives.
// ---------------------------------------------------------------------------

// LINEAR: from the partials and stored logits of the fused linear-LogP, see below.
struct ScoreFinishArgs {
  const void* logits;
  int64_t row_stride;
  const int64_t* target;
  const float* temperature;
  const float* stats;
  const uint32_t* best;
  const uint32_t* where;
  float* logp;
  float* lse;
  float* entropy;
  float* top_logp;   // [T][top_k]
  int64_t* top_ids;  // [T][top_k]
  int T, V, real, tile_size, top_k;
  const float* part;      // LINEAR: [n_split][T] maxima, sums, target logits
  const float* weighted;  // LINEAR: [n_split][T]
  int n_split;
};

constexpr int kFinishKeys = 512;     // candidates that are held at a time
constexpr int kFinishPicked = 128;   // slices
constexpr int kScoreMostTop = 64;

// A reduction over the wave in six steps of the data-parallel primitives: rows of 16 first, then across them; the result, which
// ends in the last lane, in all of them. (Shuffles go through the LDS unit: 2.4 us for the merge of a row, now 1.3.)
template <class Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, uint32_t neutral, Op op) {
#define RLK_REDUCE_STEP(CONTROL, ROWS) v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)neutral, (int)v, CONTROL, ROWS, 0xf, false))
  RLK_REDUCE_STEP(0x111, 0xf);  // row_shr 1, 2, 4, 8
  RLK_REDUCE_STEP(0x112, 0xf);
  RLK_REDUCE_STEP(0x114, 0xf);
  RLK_REDUCE_STEP(0x118, 0xf);
  RLK_REDUCE_STEP(0x142, 0xa);  // row_bcast 15: into rows 1 and 3
  RLK_REDUCE_STEP(0x143, 0xc);  // row_bcast 31: into rows 2 and 3
#undef RLK_REDUCE_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_sum_f32(float v) {
  auto add = [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); };
  return __uint_as_float(wave_reduce(__float_as_uint(v), 0u, add));
}
__device__ __forceinline__ float wave_max_f32(float v) {
  auto larger = [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); };
  return __uint_as_float(wave_reduce(__float_as_uint(v), __float_as_uint(kNegInf), larger));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) { return wave_reduce(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) { return wave_reduce(v, ~0u, [](uint32_t a, uint32_t b) { return a < b ? a : b; }); }

// From this size on lse = M + log S loses log S to rounding, all of it where a row is masked throughout with a finite lowest value (its
// tokens would all look certain): log-probabilities are y - M - log S then, as they are in the row's entropy.
constexpr float kFarOut = 65536.f;

// What one lane of a wave wrote to LDS is seen by the others behind it.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Bits at the end of an ordered logit that its type leaves the same in all logits of a sign: thresholds need not tell them apart.
template <int ELEM>
constexpr int kIdleBits = ELEM == RLK_DTYPE_BF16 ? 16 : ELEM == RLK_DTYPE_FP16 ? 13 : 0;

// The largest threshold in [low, high] that at least k values reach, where `reach(low)` >= k: halvings, each a count over the wave.
// Ends early at a threshold that at most `enough` reach.
template <class Count>
__device__ __forceinline__ uint32_t threshold_of(uint32_t low, uint32_t high, int k, int enough, int& reached, Count reach) {
  while (reached > enough && low < high) {
    const uint32_t mid = low + (high - low + 1) / 2;
    const int count = reach(mid);
    if (count >= k) {
      low = mid;
      reached = count;
    } else {
      high = mid - 1;
    }
  }
  return low;
}

// The k largest of n different keys (k <= n <= kFinishKeys; their upper words in [low, high], their columns under V) move to the front
// of `keys`; returns the smallest of them. First the k-th logit, then, among the keys that have it, the last column.
template <int ELEM>
__device__ __noinline__ uint64_t keep_largest(uint64_t* keys, int n, int k, int lane, uint32_t low, uint32_t high, int V) {
  constexpr int EACH = kFinishKeys / kWave;
  uint64_t mine[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) mine[i] = i * kWave + lane < n ? keys[i * kWave + lane] : 0;
  constexpr int kIdle = kIdleBits<ELEM>;
  int reached = n;
  const uint32_t at = threshold_of(low >> kIdle, high >> kIdle, k, k, reached, [&](uint32_t t) __attribute__((always_inline)) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) count += __popcll(__ballot((uint32_t)(mine[i] >> 32) >> kIdle >= t));
    return count;
  });
  uint64_t floor = (uint64_t)at << kIdle << 32;
  if (reached > k) {  // (the columns of the keys above `at` count in full)
    const uint32_t last = threshold_of(0u, (uint32_t)V - 1, k, k, reached, [&](uint32_t t) __attribute__((always_inline)) {
      int count = 0;
      const uint32_t tail = ~((uint32_t)V - 1 - t);  // columns up to V - 1 - t
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const uint32_t upper = (uint32_t)(mine[i] >> 32) >> kIdle;
        count += __popcll(__ballot(upper > at || (upper == at && (uint32_t)mine[i] >= tail)));
      }
      return count;
    });
    uint64_t smallest = ~(uint64_t)0;  // of the keys that are left: their upper words agree in what the type leaves idle
    const uint32_t tail = ~((uint32_t)V - 1 - last);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const uint32_t upper = (uint32_t)(mine[i] >> 32) >> kIdle;
      if (upper == at && (uint32_t)mine[i] >= tail && mine[i] < smallest) smallest = mine[i];
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) {
      const uint64_t other = (uint64_t)__shfl_xor((long long)smallest, offset);
      smallest = other < smallest ? other : smallest;
    }
    floor = smallest;
  }
  wave_lds_sync();
  int kept = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const bool keep = mine[i] != 0 && mine[i] >= floor;
    const uint64_t mask = __ballot(keep);
    if (keep) keys[kept + lanes_below(mask)] = mine[i];
    kept += __popcll(mask);
  }
  wave_lds_sync();
  return floor;
}

// The vector that is number `step` of a slice, and the columns of its tile. A slice of materialised logits is every sixteenth vector of
// a tile; one of the fused linear-LogP is a stream of every 64th split: 16 columns of each of its four tiles.
template <bool LINEAR>
__device__ __forceinline__ int slice_vector(const ScoreFinishArgs& a, int tile, int l16, int step) {
  if constexpr (LINEAR) {
    return (tile + kScoreTiles * (step >> 3)) * (kLogpSplitCols / 8) + (step >> 1 & 3) * (kLogpTileCols / 8) + 2 * l16 + (step & 1);
  } else {
    const int64_t lo64 = (int64_t)tile * a.tile_size;
    return (int)((lo64 < a.real ? lo64 : a.real) / 8) + l16 + step * kTileLanes;
  }
}
template <bool LINEAR>
__device__ __forceinline__ void tile_columns(const ScoreFinishArgs& a, int tile, int& lo_col, int& hi_col) {
  lo_col = 0;
  hi_col = a.real;
  if constexpr (!LINEAR) {
    const int64_t lo64 = (int64_t)tile * a.tile_size, hi64 = lo64 + a.tile_size;
    lo_col = lo64 < a.real ? (int)lo64 : a.real;
    hi_col = hi64 < a.real ? (int)hi64 : a.real;
  }
}

template <int ELEM, bool LINEAR>
__device__ __forceinline__ void finish_alternatives(const ScoreFinishArgs& a, int row, int lane, const uint32_t (&most)[kTileLanes],
                                                    const uint32_t (&at)[kTileLanes], float base, float rest, float inv_t, uint64_t* keys,
                                                    uint32_t* picked, uint32_t* where) {
  using E = typename LogitElem<ELEM>::type;
  const int k = a.top_k;
  constexpr int kEach = kScoreSlices / kWave;  // a lane has the sixteen slices of one tile
  static_assert(kEach == kTileLanes, "a lane per tile");
#pragma unroll
  for (int i = 0; i < kEach; ++i) where[i * kWave + lane] = at[i];
  auto count_from = [&](uint32_t limit) __attribute__((always_inline)) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) count += __popcll(__ballot(most[i] >= limit));
    return count;
  };
  uint32_t tile_most = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) tile_most = max(tile_most, most[i]);
  const uint32_t high = wave_max_u32(tile_most);

  // Slices from a limit on that at least k of them reach and not many more (any such limit is as good as the k-th best): first the
  // limit that k of the 64 tiles reach, where a step of the search is one comparison; of its slices there are few more unless k is
  // near 64.
  constexpr int kIdle = kIdleBits<ELEM>;
  uint32_t low = max(wave_min_u32(tile_most), 1u);  // 0: a slice without columns
  int reach = kScoreTiles;
  low = max(threshold_of(low >> kIdle, high >> kIdle, k, k, reach, [&](uint32_t t) __attribute__((always_inline)) {
              return (int)__popcll(__ballot(tile_most >> kIdle >= t));
            }) << kIdle, 1u);
  reach = count_from(low);
  low = max(threshold_of(low >> kIdle, high >> kIdle, k, k + kWave / 2, reach, [&](uint32_t t) __attribute__((always_inline)) {
              return count_from(t << kIdle);
            }) << kIdle, 1u);
  uint64_t floor = (uint64_t)low << 32;  // candidates are not under it; key = (ordered logit, columns behind it)

  uint32_t last_at = 0xffffffffu;
  if (reach > kFinishPicked) {  // many slices with the same best logit: the first of them, by the vector that holds it
    const uint32_t same = low >> kIdle;
    const int above = count_from((same + 1) << kIdle);  // (the largest ordered logit, that of +inf, ends in 23 zeros)
    uint32_t first = 0, end = (uint32_t)(a.V / 8);  // the smallest vector number up to which there are enough
    while (first < end) {
      const uint32_t mid = first + (end - first) / 2;
      int count = above;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        count += __popcll(__ballot(most[i] >> kIdle == same && (uint32_t)slice_vector<LINEAR>(a, lane, i, at[i] & 0xffffu) <= mid));
      if (count >= k) end = mid; else first = mid + 1;
    }
    last_at = first;
    floor |= 0xffffffffu - min((uint64_t)0xffffffffu, (uint64_t)last_at * 8 + 7);
  }
  // Of a picked slice its best vector is read, from the front of the list on, or all of it, from the back. The wave takes one slice of
  // each lane at a time, which leaves two or three turns of a short loop: straight code for all sixteen took 1.7 us a row, most of it to
  // be fetched.
  uint32_t takes = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) takes |= most[i] >= low ? 1u << i : 0u;
  if (last_at != 0xffffffffu) {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (most[i] >> kIdle == low >> kIdle && (uint32_t)slice_vector<LINEAR>(a, lane, i, at[i] & 0xffffu) > last_at) takes &= ~(1u << i);
  }
  int singles = 0, wholes = 0;
#pragma unroll 1
  while (__ballot(takes != 0) != 0) {
    const int i = __builtin_ctz(takes | 1u << (kEach - 1));
    const uint32_t v = where[i * kWave + lane];
    const bool whole = v >> 16 >= low >> 16;  // another of its vectors may reach the limit
    const uint64_t single_mask = __ballot(takes != 0 && !whole), whole_mask = __ballot(takes != 0 && whole);
    if (takes != 0) {
      if (whole) picked[kFinishPicked - 1 - (wholes + lanes_below(whole_mask))] = (uint32_t)(lane * kEach + i);
      else picked[singles + lanes_below(single_mask)] = (uint32_t)lane << 26 | (uint32_t)slice_vector<LINEAR>(a, lane, i, v & 0xffffu);
    }
    singles += __popcll(single_mask);
    wholes += __popcll(whole_mask);
    takes &= takes - 1;
  }
  wave_lds_sync();

  // The vectors, a lane each, one on its way while one is looked at. (Four on their way took four times the code: 0.8 us more for one
  // row, nothing less for 2048.) An element costs a comparison with the floor's logit; a lane's candidates of a vector are the bits of a
  // mask, and the wave takes one of each lane at a time.
  const E* row_ptr = reinterpret_cast<const E*>(a.logits) + (int64_t)row * a.row_stride;
  // vectors of a slice, at most (2^28 / 64 / 128 + 1)
  const int rounds = LINEAR ? (a.n_split + kScoreTiles - 1) / kScoreTiles * 8 : ((a.tile_size + 14) / 8 + kTileLanes - 1) / kTileLanes;
  const uint32_t jobs = (uint32_t)(singles + wholes * rounds);
  RowVector<ELEM> next;
  int next_first = 0;    // the window's first column,
  uint32_t next_of = 0;  // and which of its eight are the slice's, as bits
  int n = 0;
  float least = low > ordered_bits(kNegInf) ? from_ordered_bits(low) : kNegInf;  // the floor's logit
  for (uint32_t first = 0; first < jobs + kWave; first += kWave) {  // (the first turn only loads, the last only looks)
    float y[8];
    uint32_t mine = 0;
    const int from = next_first;
    if (first > 0) {
      next.unpack(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = fmaxf(y[i], kNegInf);  // (a NaN counts as -inf)
        mine |= y[i] >= least ? 1u << i : 0u;
      }
      mine &= next_of;
    }
    const uint32_t job = first + lane;
    next_of = 0;
    if (job < jobs) {
      int tile, g;
      if (job < (uint32_t)singles) {
        tile = picked[job] >> 26;
        g = picked[job] & 0x3ffffffu;
      } else {
        const uint32_t rest = job - singles, slice = picked[kFinishPicked - 1 - rest / (uint32_t)rounds];
        tile = slice / kTileLanes;
        g = slice_vector<LINEAR>(a, tile, slice % kTileLanes, rest % (uint32_t)rounds);
      }
      int lo_col, hi_col;
      tile_columns<LINEAR>(a, tile, lo_col, hi_col);
      if ((int64_t)g * 8 < hi_col) {
        const int at = window_of(g * 8, a.V);
        const int lo = max(lo_col, g * 8) - at, hi = min(hi_col, g * 8 + 8) - at;
        next_of = (1u << hi) - (1u << lo);
        next_first = at;
        next.template load_window<false>(row_ptr, at, a.V);
      }
    }
    while (__ballot(mine != 0) != 0) {
      const int i = __builtin_ctz(mine | 256u);
      float v = y[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) v = i == e ? y[e] : v;
      const uint64_t key = (uint64_t)ordered_bits(v) << 32 | (0xffffffffu - (uint32_t)(from + i));
      const bool take = mine != 0 && key >= floor;
      const uint64_t mask = __ballot(take);
      if (take) keys[n + lanes_below(mask)] = key;
      n += __popcll(mask);
      mine &= mine - 1;
      if (n > kFinishKeys - kWave) {
        wave_lds_sync();
        floor = keep_largest<ELEM>(keys, n, k, lane, low, high, a.V);
        least = from_ordered_bits((uint32_t)(floor >> 32));
        n = k;
      }
    }
  }
  wave_lds_sync();
  if (n > 2 * kWave) {
    keep_largest<ELEM>(keys, n, k, lane, low, high, a.V);
    n = k;
  }

  // A key's rank is the number of larger ones: all of them read from LDS, four at a time, the same for every lane.
  if (lane < 4) keys[n + lane] = 0;
  wave_lds_sync();
  uint64_t mine[2];
  int rank[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) mine[i] = i * kWave + lane < n ? keys[i * kWave + lane] : 0;
  auto rank_all = [&](auto both) __attribute__((always_inline)) {
    for (int j = 0; j < n; j += 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t other = keys[j + e];
        rank[0] += other > mine[0] ? 1 : 0;
        if constexpr (decltype(both)::value) rank[1] += other > mine[1] ? 1 : 0;
      }
    }
  };
  if (n <= kWave) rank_all(BoolConstant<false>{});
  else rank_all(BoolConstant<true>{});
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i * kWave + lane >= n || rank[i] >= k) continue;
    float v = (from_ordered_bits((uint32_t)(mine[i] >> 32)) * inv_t - base) - rest;
    if (LINEAR && v > 0.f) v = 0.f;  // the fused linear-LogP clamps its log-probabilities
    const int64_t out = (int64_t)row * k + rank[i];
    a.top_ids[out] = (int64_t)(0xffffffffu - (uint32_t)mine[i]);
    a.top_logp[out] = v;
  }
}

// 2048 rows: 5 us, 17 with 64 alternatives (17 MB of slices, then two lines of logits for each of some 80 vectors of a row); one row: 2 us,
// 5 with 20 alternatives, a chain of dependent reads and searches whose code is fetched as it is run: short loops throughout.
template <int ELEM, bool LINEAR>
__global__ __launch_bounds__(kWave) void score_finish_kernel(ScoreFinishArgs a) {
  __shared__ __align__(16) uint64_t keys[kFinishKeys];
  __shared__ uint32_t picked[kFinishPicked];
  __shared__ uint32_t slices[kScoreSlices];
  const int lane = threadIdx.x;
  const int row = blockIdx.x;
  uint32_t most[kTileLanes], at[kTileLanes];  // on their way while the tiles are merged
  if (a.top_k > 0) {
    const u32x4_t* best = reinterpret_cast<const u32x4_t*>(a.best + (int64_t)row * kScoreSlices + lane * kTileLanes);
    const u32x4_t* where = reinterpret_cast<const u32x4_t*>(a.where + (int64_t)row * kScoreSlices + lane * kTileLanes);
#pragma unroll
    for (int i = 0; i < kTileLanes / 4; ++i) {
      const u32x4_t v = best[i], w = where[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most[4 * i + e] = v[e];
        at[4 * i + e] = w[e];
      }
    }
  }
  const float inv_t = a.temperature ? 1.0f / a.temperature[row] : 1.0f;
  const bool bad_temperature = !(inv_t > 0.f && inv_t < -kNegInf);  // (0 or infinity times a masked logit, or one of 0, is no number)
  const float nan = __builtin_nanf("");
  float base, rest;  // log p = y - base - rest
  if constexpr (LINEAR) {  // a lane takes every 64th split; the sums of all are added ascending, as in linear_logp_merge_kernel
    const int64_t plane = (int64_t)a.n_split * a.T;
    const int64_t target = a.target[row];
    const bool bad_target = target < 0 || target >= a.real;
    const float zt = bad_target ? nan : a.part[2 * plane + target / kLogpSplitCols * a.T + row];
    constexpr int kHeld = 4;  // splits of a lane at a time, as loaded: up to a vocabulary of 262144 all of them
    float pm[kHeld], ps[kHeld], pw[kHeld];
    auto fetch = [&](int base) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        const int p = base + r * kWave + lane;
        const int64_t at = (int64_t)p * a.T + row;
        pm[r] = p < a.n_split ? a.part[at] : kNegInf;
        ps[r] = p < a.n_split ? a.part[plane + at] : 0.f;
        pw[r] = p < a.n_split ? a.weighted[at] : 0.f;
      }
    };
    fetch(0);
    float m = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), w = 0.f, sum = 0.f;
    for (int p = kHeld * kWave + lane; p < a.n_split; p += kWave) m = fmaxf(m, a.part[(int64_t)p * a.T + row]);
    const float big = wave_max_f32(m);
    float* const terms = reinterpret_cast<float*>(keys);  // (not in use yet)
    for (int base = 0; base < a.n_split; base += kHeld * kWave) {
      if (base > 0) fetch(base);
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        const float scaled = ps[r] * pinned_exp(pm[r] - big);
        terms[r * kWave + lane] = pm[r] > kNegInf ? scaled : 0.f;
        w = w + logp_weighted_term(pm[r], ps[r], pw[r], big);
      }
      wave_lds_sync();
      const int count = min(kHeld * kWave, a.n_split - base);
      for (int j = 0; j < count; j += 4) {  // (terms behind the last split are 0)
        const f32x4_t four = *reinterpret_cast<const f32x4_t*>(terms + j);
        sum = (((sum + four[0]) + four[1]) + four[2]) + four[3];
      }
      wave_lds_sync();
    }
    const float weighted = wave_sum_f32(w);
    const float log_sum = logf(sum);
    const bool diverged = weighted != weighted;  // (the linear-LogP's maxima and sums pass over a NaN that stands among masked logits)
    const float lse = bad_temperature || diverged ? nan : big + log_sum;
    const bool far = fabsf(lse) >= kFarOut && lse > kNegInf;
    base = far ? big : lse;
    rest = far ? log_sum : 0.f;
    if (lane == 0) {
      a.entropy[row] = bad_temperature ? nan : log_sum - weighted / sum;
      a.lse[row] = lse;
      const float value = (zt - base) - rest;
      a.logp[row] = bad_temperature || bad_target ? nan : value > 0.f ? 0.f : value;  // (fminf would drop a NaN)
    }
  } else {
    const float* stats = a.stats + (int64_t)row * kScorePlanes * kScoreTiles + lane;
    const float m = stats[0], s = stats[kScoreTiles], w = stats[3 * kScoreTiles];
    const float big = wave_max_f32(m), from = fmaxf(big, kLowest);
    const float shrink = pinned_exp(m - from);
    const float term = s * shrink;
    float sum = 0.f;  // (ascending)
#pragma unroll 8
    for (int t = 0; t < kScoreTiles; ++t) sum = sum + __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(term), t));
    const float weighted = wave_sum_f32(shrink * __builtin_fmaf(s, fmaxf(m - from, kFarBelow), w));
    const float log_sum = logf(sum);
    const float lse = bad_temperature ? nan : big + log_sum;
    const bool far = fabsf(lse) >= kFarOut && lse > kNegInf;
    base = far ? big : lse;
    rest = far ? log_sum : 0.f;
    const float zt = wave_sum_f32(stats[2 * kScoreTiles]);
    if (lane == 0) {
      const bool bad_target = a.target[row] < 0 || a.target[row] >= a.real;
      a.entropy[row] = bad_temperature ? nan : log_sum - weighted / sum;
      a.lse[row] = lse;
      a.logp[row] = bad_target ? nan : (zt - base) - rest;
    }
  }
  if (a.top_k > 0) finish_alternatives<ELEM, LINEAR>(a, row, lane, most, at, base, rest, inv_t, keys, picked, slices);
}

// ---------------------------------------------------------------------------
// The scores of the fused linear-LogP. Its partials have the maxima and sums of the splits; the weighted sums follow its reduction
// contract: a chain per stream of a split, tile by tile (logp_fold_run_weighted), the streams of a split in pairs, from their
// maximum. The four-wave kernel above 1024 tokens has them in its fold. Where it does not run, or alternatives are asked for, they
// come from the logits that the launch stored, by the kernel below: the same steps on the same values, so the same bits for a token
// whatever batch it arrives in. A lane has one stream, sixteen of them a split, and goes through every 64th split: these are the
// slices of the alternatives. HBM-bound: 2048 x 151936 fp32 logits 258 us with alternatives = 4.8 TB/s; 16 rows 5.4.
// ---------------------------------------------------------------------------

struct LinearRowArgs {
  const float* logits;  // [T, logits_ld], rows of whole 64-column spans, 16-byte aligned
  int64_t logits_ld;
  const float* temperature;  // or null
  float* weighted;           // [n_split][T]
  uint32_t* best;            // as in ScoreArgs
  uint32_t* where;
  int T, V, real, n_split;
};

template <bool HAS_TEMP, bool TOP>
__global__ __launch_bounds__(256) void linear_score_rows_kernel(LinearRowArgs a) {
  const int row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & (kTileLanes - 1);
  const float* row_ptr = a.logits + (int64_t)row * a.logits_ld;
  const float inv_t = HAS_TEMP ? 1.0f / a.temperature[row] : 1.0f;
  // A wave has four splits at a time. TOP: those of the same classes are the other three waves' and its next ones.
  const int c0 = blockIdx.y * (TOP ? kTilesPerWave : kGroupTiles) + (TOP ? 0 : wave * kTilesPerWave);
  const int mine = c0 + lane / kTileLanes;
  float best = kNegInf, other = kNegInf;
  int at = 0;
  for (int base = TOP ? wave * kScoreTiles : 0; base + c0 < a.n_split; base += 4 * kScoreTiles) {  // uniform
    const int split = base + mine;
    const int col0 = split * kLogpSplitCols + l16 * 16;
    f32x4_t raw[kLogpSplitTiles][4];
#pragma unroll
    for (int t = 0; t < kLogpSplitTiles; ++t) {
      const int col = col0 + t * kLogpTileCols;
      if (split < a.n_split && col < a.V) {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[t][q] = *reinterpret_cast<const f32x4_t*>(row_ptr + col + 4 * q);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[t][q] = f32x4_t{kNegInf, kNegInf, kNegInf, kNegInf};
      }
    }
    float m = kNegInf, s = 0.f, w = 0.f, unused = 0.f;
#pragma unroll
    for (int t = 0; t < kLogpSplitTiles; ++t) {
      const int col = col0 + t * kLogpTileCols;
      float y[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) y[c] = col + c < a.real ? raw[t][c / 4][c % 4] : kNegInf;
      if constexpr (TOP) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* v = y + 8 * h;
          const float here = max3_f32(max3_f32(max3_f32(max3_f32(v[0], v[1], v[2]), v[3], v[4]), v[5], v[6]), v[7], v[7]);
          at = here > best ? base / kScoreTiles * 8 + 2 * t + h : at;
          other = __builtin_amdgcn_fmed3f(here, best, other);
          best = fmaxf(best, here);
        }
      }
      if constexpr (HAS_TEMP) {
#pragma unroll
        for (int c = 0; c < 16; ++c) y[c] = y[c] * inv_t;
      }
      logp_fold_run_weighted(y, -1, m, s, w, unused);
      __builtin_amdgcn_sched_barrier(0);
    }
    float big = fmaxf(m, xor_lane<1>(m));
    big = fmaxf(big, xor_lane<2>(big));
    big = fmaxf(big, xor_lane<4>(big));
    big = fmaxf(big, xor_lane<8>(big));
    float sum = logp_weighted_term(m, s, w, big);
    sum = sum + xor_lane<1>(sum);
    sum = sum + xor_lane<2>(sum);
    sum = sum + xor_lane<4>(sum);
    sum = sum + xor_lane<8>(sum);
    if (l16 == 0 && split < a.n_split) a.weighted[(int64_t)split * a.T + row] = sum;
    if constexpr (!TOP) break;
  }
  if constexpr (TOP) {  // the waves' notes of a slice: the larger best one, of equal ones the first vector, and what is left as the other
    __shared__ float bests[4][kWave], others[4][kWave];
    __shared__ int ats[4][kWave];
    bests[wave][lane] = best;
    others[wave][lane] = other;
    ats[wave][lane] = at;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int v = 1; v < 4; ++v) {
      const float theirs = bests[v][lane];
      const int their_at = ats[v][lane];
      const bool win = theirs > best || (theirs == best && their_at < at);
      other = fmaxf(fmaxf(other, others[v][lane]), win ? best : theirs);
      best = win ? theirs : best;
      at = win ? their_at : at;
    }
    const int64_t slice = (int64_t)row * kScoreSlices + mine * kTileLanes + l16;
    a.best[slice] = mine * kLogpSplitCols + l16 * 16 < a.real ? ordered_bits(best) : 0u;
    a.where[slice] = (ordered_bits(other) & 0xffff0000u) | (uint32_t)at;
  }
}

// ---------------------------------------------------------------------------
// Gradient: dz = 1/T [ p (g_lse - g_logp - sum g_top - g_entropy (y - lse + entropy)) + g_logp [target] + g_top [ids] ],
// p = e(y - lse). Elementwise; rounded once to the element type of the output. HBM-bound: 2047 x 151936 bf16 225 us = 5.5 TB/s, fp32 logits to
// bf16 of 2060 x 151936 364 us = 5.2.
// ---------------------------------------------------------------------------

struct ScoreBackwardArgs {
  const void* logits;
  int64_t row_stride;
  const int64_t* target;
  const float* temperature;  // or null
  const float* lse;
  const float* entropy;      // read with g_entropy
  const float* g_logp;       // each [T] or null (= 0)
  const float* g_lse;
  const float* g_entropy;
  const int64_t* top_ids;    // [T][top_k], read with g_top
  const float* g_top;        // [T][top_k] or null
  void* grad;
  int64_t grad_row_stride;
  int T, V, real, top_k;
  int grad_cols;  // columns written: V and zeros behind it
};

constexpr int kScoreBackThreads = 256;
constexpr int kScoreBackVectors = 4;
constexpr int kScoreBackCols = kScoreBackThreads * kScoreBackVectors * 8;

// A workgroup's sum or maximum of a value per thread, in all of them.
template <class Op>
__device__ __forceinline__ float score_block_reduce(float v, float (*waves)[kScoreBackThreads / kWave], Op op) {
  if ((threadIdx.x & 63) == 0) (*waves)[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (*waves)[0];
#pragma unroll
  for (int w = 1; w < kScoreBackThreads / kWave; ++w) v = op(v, (*waves)[w]);
  return v;
}

// The columns [first, end) of a far-out row (kFarOut): its maximum and the logarithm of its sum, which lse does not hold, from the whole row
// again.
template <int ELEM, int OUT>
__device__ __forceinline__ void far_out_columns(const typename LogitElem<ELEM>::type* row, typename LogitElem<OUT>::type* grad, int first, int end,
                                                int real, float inv_t, float slope, float g_entropy, float entropy, float scale, int hits,
                                                const int* hit_col, const float* hit_grad) {
  __shared__ float waves[2][kScoreBackThreads / kWave];
  auto scaled = [&](int c) __attribute__((always_inline)) { return LogitElem<ELEM>::to_float(row[c]) * inv_t; };
  float big = kNegInf, sum = 0.f;
#pragma unroll 1
  for (int c = threadIdx.x; c < real; c += kScoreBackThreads) big = fmaxf(big, scaled(c));
  big = score_block_reduce(wave_max_f32(big), &waves[0], [](float a, float b) { return fmaxf(a, b); });
#pragma unroll 1
  for (int c = threadIdx.x; c < real; c += kScoreBackThreads) sum = sum + pinned_exp(scaled(c) - big);
  const float log_sum = logf(score_block_reduce(wave_sum_f32(sum), &waves[1], [](float a, float b) { return a + b; }));
#pragma unroll 1
  for (int c = first + threadIdx.x; c < end; c += kScoreBackThreads) {
    float out = 0.f;
    if (c < real) {
      const float d = (scaled(c) - big) - log_sum;
      out = pinned_exp(d) * __builtin_fmaf(-g_entropy, fmaxf(d, kFarBelow) + entropy, slope);
      for (int h = 0; h < hits; ++h) out = hit_col[h] == c ? out + hit_grad[h] : out;
      out = out * scale;
    }
    grad[c] = LogitElem<OUT>::from_float(out);
  }
}

template <int ELEM, int OUT, bool STREAM>
__global__ __launch_bounds__(kScoreBackThreads) void score_backward_kernel(ScoreBackwardArgs a) {
  using E = typename LogitElem<ELEM>::type;
  using O = typename LogitElem<OUT>::type;
  __shared__ int hit_col[kScoreMostTop + 1];
  __shared__ float hit_grad[kScoreMostTop + 1];
  __shared__ int hit_count;
  __shared__ bool any_top;  // a gradient of an alternative that is not 0
  __shared__ float top_sum;
  // from the last row and columns to the first: the forward has left the last ones in the memory-side cache
  const int row = gridDim.x - 1 - blockIdx.x;
  const int first = (int)(gridDim.y - 1 - blockIdx.y) * kScoreBackCols;
  const E* row_in = reinterpret_cast<const E*>(a.logits) + (int64_t)row * a.row_stride;
  O* row_out = reinterpret_cast<O*>(a.grad) + (int64_t)row * a.grad_row_stride;

  RowVector<ELEM> raw[kScoreBackVectors];
#pragma unroll
  for (int u = 0; u < kScoreBackVectors; ++u) {
    const int64_t col = first + (int64_t)(u * kScoreBackThreads + threadIdx.x) * 8;
    if (col < a.real) raw[u].template load_edge<STREAM>(row_in, (int)(col / 8), a.V);
  }

  const float g_logp = a.g_logp ? a.g_logp[row] : 0.f;
  if (threadIdx.x < kWave) {  // the columns of this workgroup with a gradient of their own
    const int lane = threadIdx.x;
    const int64_t wanted = lane < a.top_k && a.g_top ? a.top_ids[(int64_t)row * a.top_k + lane] : -1;
    const float g = wanted >= 0 ? a.g_top[(int64_t)row * a.top_k + lane] : 0.f;
    const float all = wave_sum_f32(g);
    const uint64_t not_zero = __ballot(g != 0.f);
    const int64_t at = wanted - first;
    const bool take = wanted >= 0 && wanted < a.real && at >= 0 && at < kScoreBackCols;
    const uint64_t mask = __ballot(take);
    if (take) {
      hit_col[lanes_below(mask)] = (int)wanted;
      hit_grad[lanes_below(mask)] = g;
    }
    if (lane == 0) {
      int count = __popcll(mask);
      const int64_t target = a.g_logp ? a.target[row] : -1;
      if (target >= first && target < (int64_t)first + kScoreBackCols && target < a.real) {
        hit_col[count] = (int)target;
        hit_grad[count++] = g_logp;
      }
      hit_count = count;
      any_top = not_zero != 0;
      top_sum = all;
    }
  }
  __syncthreads();
  const float lse = a.lse[row];
  const float inv_t = a.temperature ? 1.0f / a.temperature[row] : 1.0f;
  const float g_entropy = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float entropy = a.g_entropy ? a.entropy[row] : 0.f;
  const float g_lse = a.g_lse ? a.g_lse[row] : 0.f;
  const float slope = g_lse - g_logp - top_sum;
  // A row that no gradient reaches has none, whatever it holds: a token that a loss leaves out must not make a weight's gradient NaN.
  const bool reached = g_logp != 0.f || g_lse != 0.f || g_entropy != 0.f || any_top;
  const bool any = reached && lse > kNegInf && lse < -kNegInf;
  // Of a row without a distribution: zeros where everything is masked (lse = -inf), as no answer moves with a logit; NaN where the row is NaN.
  const int hits = any ? hit_count : 0;
  const float scale = any ? inv_t : 1.f;
  const float without = reached && lse != kNegInf ? __builtin_nanf("") : 0.f;
  if (any && fabsf(lse) >= kFarOut) {
    far_out_columns<ELEM, OUT>(row_in, row_out, first, min(first + kScoreBackCols, a.grad_cols), a.real, inv_t, slope, g_entropy, entropy, scale,
                               hits, hit_col, hit_grad);
    return;
  }
  // lse and the gradients of the row in registers: from here on a logit costs an exponential and a few products
#pragma unroll
  for (int u = 0; u < kScoreBackVectors; ++u) {
    const int64_t col = first + (int64_t)(u * kScoreBackThreads + threadIdx.x) * 8;
    if (col >= a.grad_cols) break;
    float out[8];
    if (col < a.real && any) {
      float z[8];
      raw[u].unpack(z);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = __builtin_fmaf(z[i], inv_t, -lse);  // log p
        const float p = pinned_exp(d);
        out[i] = p * __builtin_fmaf(-g_entropy, fmaxf(d, kFarBelow) + entropy, slope);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = without;  // (columns behind the real ones: 0 below)
    }
    for (int h = 0; h < hits; ++h) {
      const int at = hit_col[h] - (int)col;
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = at == i ? out[i] + hit_grad[h] : out[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = col + i < a.real ? out[i] * scale : 0.f;
    RowVector<OUT> packed;
    packed.pack(out);
    packed.template store_edge<STREAM>(row_out, col, a.grad_cols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

size_t token_scores_workspace_bytes(int T, int top_k) {
  return (size_t)T * (kScorePlanes * kScoreTiles * sizeof(float) + (top_k > 0 ? 2 * kScoreSlices * sizeof(uint32_t) : 0));
}

template <int ELEM, bool HAS_TEMP, bool TOP>
static void launch_score_tiles(const ScoreArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.T, kScoreTiles / kGroupTiles);
  hipLaunchKernelGGL((score_tiles_kernel<ELEM, HAS_TEMP, TOP>), grid, dim3(256), 0, stream, a);
}

template <int ELEM>
static hipError_t token_scores_typed(const ScoreArgs& a, const ScoreFinishArgs& f, hipStream_t stream) {
  const bool temp = a.temperature != nullptr, top = f.top_k > 0;
  if (temp && top) launch_score_tiles<ELEM, true, true>(a, stream);
  else if (top) launch_score_tiles<ELEM, false, true>(a, stream);
  else if (temp) launch_score_tiles<ELEM, true, false>(a, stream);
  else launch_score_tiles<ELEM, false, false>(a, stream);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((score_finish_kernel<ELEM, false>), dim3((unsigned)a.T), dim3(kWave), 0, stream, f);
  return hipGetLastError();
}

hipError_t token_scores_launch(const void* logits, int dtype, int64_t row_stride, const int64_t* target, const float* temperature, int T,
                               int V, int real, int top_k, float* logp, float* lse, float* entropy, float* top_logp, int64_t* top_ids,
                               void* workspace, hipStream_t stream) {
  ScoreArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.target = target;
  a.temperature = temperature;
  a.stats = reinterpret_cast<float*>(workspace);
  a.best = reinterpret_cast<uint32_t*>(a.stats + (size_t)T * kScorePlanes * kScoreTiles);
  a.where = a.best + (size_t)T * kScoreSlices;
  a.T = T;
  a.V = V;
  a.real = real;
  a.tile_size = (int)(((int64_t)V + kScoreTiles - 1) / kScoreTiles);
  const int64_t bytes = (int64_t)T * V * (dtype == RLK_DTYPE_FP32 ? 4 : 2);
  a.streamed = bytes > kCachedLogitsBytes ? (int64_t)((double)T * (kScoreTiles / kGroupTiles) * (1.0 - (double)kCachedLogitsBytes / bytes)) : 0;
  const ScoreFinishArgs f{logits, row_stride, target, temperature, a.stats, a.best, a.where, logp, lse, entropy,
                          top_logp, top_ids, T, V, real, a.tile_size, top_k, nullptr, nullptr, 0};
  switch (dtype) {
    case RLK_DTYPE_BF16: return token_scores_typed<RLK_DTYPE_BF16>(a, f, stream);
    case RLK_DTYPE_FP16: return token_scores_typed<RLK_DTYPE_FP16>(a, f, stream);
    case RLK_DTYPE_FP32: return token_scores_typed<RLK_DTYPE_FP32>(a, f, stream);
    default: return hipErrorInvalidValue;
  }
}

size_t linear_scores_extra_bytes(int T, int V, int top_k) {
  const size_t weighted = (size_t)linear_logp_split_count(V) * T * sizeof(float);
  return weighted + 16 + (top_k > 0 ? (size_t)T * 2 * kScoreSlices * sizeof(uint32_t) : 0);
}

hipError_t linear_scores_launch(const float* logits, int64_t logits_ld, const int64_t* target, const float* temperature, const float* part,
                                bool have_weighted, int T, int V, int real, int n_split, int top_k, float* logp, float* lse, float* entropy,
                                float* top_logp, int64_t* top_ids, void* extra, hipStream_t stream) {
  float* weighted = reinterpret_cast<float*>(extra);
  uint32_t* best = reinterpret_cast<uint32_t*>((reinterpret_cast<uintptr_t>(weighted + (size_t)n_split * T) + 15) / 16 * 16);
  uint32_t* where = best + (size_t)T * kScoreSlices;
  if (!have_weighted || top_k > 0) {
    LinearRowArgs a{logits, logits_ld, temperature, weighted, best, where, T, V, real, n_split};
    // (four splits to a wave, and a wave for all of them: with 64 classes of splits, each the work of one lane, 1 to 16 tokens of V = 151936
    // took 4.6 us more)
    const dim3 grid((unsigned)T, top_k > 0 ? kScoreTiles / kTilesPerWave : (n_split + kGroupTiles - 1) / kGroupTiles), block(256);
    if (temperature && top_k > 0) hipLaunchKernelGGL((linear_score_rows_kernel<true, true>), grid, block, 0, stream, a);
    else if (temperature) hipLaunchKernelGGL((linear_score_rows_kernel<true, false>), grid, block, 0, stream, a);
    else if (top_k > 0) hipLaunchKernelGGL((linear_score_rows_kernel<false, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((linear_score_rows_kernel<false, false>), grid, block, 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  const ScoreFinishArgs f{logits, logits_ld, target, temperature, nullptr, best, where, logp, lse, entropy,
                          top_logp, top_ids, T, V, real, 0, top_k, part, weighted, n_split};
  hipLaunchKernelGGL((score_finish_kernel<RLK_DTYPE_FP32, true>), dim3((unsigned)T), dim3(kWave), 0,
                     stream, f);
  return hipGetLastError();
}

template <int ELEM, int OUT>
static hipError_t score_backward_typed(const ScoreBackwardArgs& a, bool streamed, hipStream_t stream) {
  const dim3 grid((unsigned)a.T, (unsigned)(((int64_t)a.grad_cols + kScoreBackCols - 1) / kScoreBackCols));
  if (streamed) hipLaunchKernelGGL((score_backward_kernel<ELEM, OUT, true>), grid, dim3(kScoreBackThreads), 0, stream, a);
  else hipLaunchKernelGGL((score_backward_kernel<ELEM, OUT, false>), grid, dim3(kScoreBackThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t token_scores_backward_launch(const void* logits, int dtype, int64_t row_stride, const int64_t* target,
                                        const float* temperature, const float* lse, const float* entropy, const float* g_logp,
                                        const float* g_lse, const float* g_entropy, const int64_t* top_ids, const float* g_top,
                                        int top_k, void* grad, int grad_dtype, int64_t grad_row_stride, int grad_cols, int T, int V,
                                        int real, hipStream_t stream) {
  const ScoreBackwardArgs a{logits, row_stride, target, temperature, lse, entropy, g_logp, g_lse, g_entropy, top_ids, g_top, grad,
                            grad_row_stride, T, V, real, g_top ? top_k : 0, grad_cols};
  // as in logits_backward_launch: a gradient that the memory-side cache cannot hold beside the logits goes past it
  const bool streamed = (int64_t)T * V * (grad_dtype == RLK_DTYPE_FP32 ? 4 : 2) >= (int64_t)128 << 20;
  if (dtype == RLK_DTYPE_BF16 && grad_dtype == dtype) return score_backward_typed<RLK_DTYPE_BF16, RLK_DTYPE_BF16>(a, streamed, stream);
  if (dtype == RLK_DTYPE_FP16 && grad_dtype == dtype) return score_backward_typed<RLK_DTYPE_FP16, RLK_DTYPE_FP16>(a, streamed, stream);
  if (dtype == RLK_DTYPE_FP32 && grad_dtype == dtype) return score_backward_typed<RLK_DTYPE_FP32, RLK_DTYPE_FP32>(a, streamed, stream);
  if (dtype == RLK_DTYPE_FP32 && grad_dtype == RLK_DTYPE_BF16) return score_backward_typed<RLK_DTYPE_FP32, RLK_DTYPE_BF16>(a, streamed, stream);
  return hipErrorInvalidValue;
}

}  // namespace rlk
