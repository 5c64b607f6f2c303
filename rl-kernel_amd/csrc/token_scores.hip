// Scores of given tokens from materialised logits for gfx950: log-probability, log-sum-exp, entropy of the row's
// distribution and its most likely alternatives, with the gradient of the logits.
//
//   y_c = z_c / temperature over the real columns c;   M = max y;   S = sum e(y_c - M);   W = sum e(y_c - M) (y_c - M)
//   lse = M + log S;   logp = y_target - lse;   entropy = log S - W / S    (both terms >= 0: nothing cancels)
//   alternatives: the top_k columns by (z descending, column ascending), their log-probabilities y - lse
//
// One pass over the logits. The running (M, S) follow the reduction contract of logits_logp.hip with 64 tiles to a row
// (tile = ceil(V / 64) columns), so that logp and lse are that entry's bits wherever 64 divides V; W is carried beside
// S: a state (m, s, w) seen from a larger maximum n is (s e(m - n), e(m - n) (w + s (m - n))).
//
// The alternatives cost the pass one comparison for each vector of eight logits. A lane of a tile sees a fixed slice of
// the row (every sixteenth vector of its tile), 1024 slices in all, and notes the largest logit of each and the vector
// that held it first. Under the order (value descending, column ascending) the k best columns of a row lie in the k
// slices whose best columns come first: a column outside of them has k better ones. So a second, small kernel picks
// those slices, reads them again (k / 1024 of the row) and ranks what is not under the k-th slice's best. Nothing of it
// depends on how a row's values are spread: equal logits, rows of one value and masked rows take the same steps.
//
// HBM-bound: a logit is read once.
#include "logits_vector.h"

namespace rlk {

constexpr int kScoreTiles = 64;
constexpr int kScoreSlices = kScoreTiles * kTileLanes;
constexpr int kScorePlanes = 4;  // max, sum, target, weighted sum: stats[row][plane][tile]
constexpr float kFarBelow = -256.f;  // e(x) is zero from here down

struct ScoreArgs {
  const void* logits;
  int64_t row_stride;  // elements
  const int64_t* target;     // [T] columns
  const float* temperature;  // [T] or null
  float* stats;              // [T][kScorePlanes][kScoreTiles]
  uint32_t* best;            // [T][kScoreSlices] largest logit of the slice (ordered bits), 0 for a slice without columns
  uint32_t* best_at;         // [T][kScoreSlices] first vector that holds it
  int T, V, real, tile_size, tiles_per_group;
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
  int at;         // first vector that held it
};

// The eight logits of vector g folded into a lane's state. The maximum is taken before the temperature (times a positive
// number it is the maximum of the products, to the bit), so that alternatives are told apart that scaling makes equal.
template <bool HAS_TEMP, bool TOP>
__device__ __forceinline__ void fold_score_vector(float (&y)[8], float inv_t, int g, ScoreState& st) {
  const float most = max3_f32(max3_f32(max3_f32(y[0], y[1], y[2]), y[3], y[4]), y[5], y[6]);
  if constexpr (TOP) st.at = fmaxf(most, y[7]) > st.raw ? g : st.at;
  st.raw = max3_f32(most, y[7], st.raw);
  float n = st.raw;
  if constexpr (HAS_TEMP) {
    n = n * inv_t;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * inv_t;
  }
  float d = y[0] - n;
  float e = pinned_exp(d);
  float sum = e, weighted = e * fmaxf(d, kFarBelow);  // (a masked logit is -inf below: 0 times that is no number)
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    d = y[i] - n;
    e = pinned_exp(d);
    sum = sum + e;
    weighted = __builtin_fmaf(e, fmaxf(d, kFarBelow), weighted);
  }
  const float back = st.m - n;
  const float shrink = pinned_exp(back);
  const float scaled = st.s * shrink;
  const float moved = __builtin_fmaf(shrink, __builtin_fmaf(st.s, fmaxf(back, kFarBelow), st.w), weighted);
  const bool any = n > kNegInf;
  st.s = any ? scaled + sum : st.s;
  st.w = any ? moved : st.w;
  st.m = n;
}

// merge_lane_states of logits_logp.hip with the weighted sum beside.
template <int OFFSET>
__device__ __forceinline__ void merge_score_lanes(int lane, ScoreState& st) {
  const float om = xor_lane<OFFSET>(st.m), os = xor_lane<OFFSET>(st.s), ow = xor_lane<OFFSET>(st.w);
  const float n = fmaxf(st.m, om);
  const float my_shrink = pinned_exp(st.m - n), other_shrink = pinned_exp(om - n);
  const float mine = st.m > kNegInf ? st.s * my_shrink : 0.f;
  const float theirs = om > kNegInf ? os * other_shrink : 0.f;
  const float my_w = st.m > kNegInf ? my_shrink * __builtin_fmaf(st.s, st.m - n, st.w) : 0.f;
  const float their_w = om > kNegInf ? other_shrink * __builtin_fmaf(os, om - n, ow) : 0.f;
  // the lower lane's term first on both sides, so that both lanes add in the same order
  st.s = (lane & OFFSET) ? theirs + mine : mine + theirs;
  st.w = (lane & OFFSET) ? their_w + my_w : my_w + their_w;
  st.m = n;
}

template <int ELEM, bool HAS_TEMP, bool TOP, bool NT>
__device__ __forceinline__ void score_tiles(const ScoreArgs& a) {
  using E = typename LogitElem<ELEM>::type;
  constexpr int kBatch = 4;
  constexpr int kStep = kTileLanes * kBatch;  // vectors of a tile per batch
  const int row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int l16 = lane & (kTileLanes - 1);
  const int grp = lane / kTileLanes;
  const E* row_ptr = reinterpret_cast<const E*>(a.logits) + (int64_t)row * a.row_stride;
  const float inv_t = HAS_TEMP ? 1.0f / a.temperature[row] : 1.0f;
  const int64_t wanted = a.target ? a.target[row] : -1;
  const int target = wanted >= 0 && wanted < a.real ? (int)wanted : -1;

  const int tile_first = blockIdx.y * a.tiles_per_group;
  const int tile_last = min(tile_first + a.tiles_per_group, kScoreTiles);
  for (int t0 = tile_first + wave * kTilesPerWave; t0 < tile_last; t0 += waves * kTilesPerWave) {
    const int tile = t0 + grp;  // (a group has a multiple of four tiles)
    const int64_t lo64 = (int64_t)tile * a.tile_size, hi64 = lo64 + a.tile_size;
    const int lo_col = lo64 < a.real ? (int)lo64 : a.real;
    const int hi_col = hi64 < a.real ? (int)hi64 : a.real;
    const int g0 = lo_col / 8;
    const int g1 = hi_col > lo_col ? (hi_col + 7) / 8 : g0;
    const int g_last = g1 > g0 ? g1 - 1 : 0;  // a valid vector to clamp loads to
    // Batches in which all four vectors of every lane are whole vectors of the lane's tile (only the very first one of a
    // tile may start before it) run without clamps and with one mask.
    const int g_whole = (hi_col % 8) ? g1 - 1 : g1;
    const int my_clean = g_whole > g0 ? (g_whole - g0) / kStep : 0;
    const int my_slots = (g1 - g0 + kTileLanes - 1) / kTileLanes;
    int clean = __builtin_amdgcn_readlane(my_clean, 0), slots = __builtin_amdgcn_readlane(my_slots, 0);
#pragma unroll
    for (int other = kTileLanes; other < kWave; other += kTileLanes) {  // uniform over the wave's four tiles
      clean = min(clean, __builtin_amdgcn_readlane(my_clean, other));
      slots = max(slots, __builtin_amdgcn_readlane(my_slots, other));
    }

    ScoreState st{kNegInf, 0.f, 0.f, kNegInf, g0 + l16};
    int g = g0 + l16;  // this lane's next vector
    // The loads rotate through four raw vectors: a vector's registers are free once it is unpacked, and the same vector
    // of the next batch is fetched into them before the fold, so a lane always has three or four loads in flight.
    RowVector<ELEM> raw[kBatch];
    if (clean > 0) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) raw[u].template load<NT>(row_ptr + (int64_t)(g + u * kTileLanes) * 8);
    }
    auto clean_batch = [&](auto more, bool first) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        float y[8];
        raw[u].unpack(y);
        if constexpr (decltype(more)::value) raw[u].template load<NT>(row_ptr + (int64_t)(g + kStep + u * kTileLanes) * 8);
        if (u == 0 && first) {
          const int lo = lo_col - g * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = i >= lo ? y[i] : kNegInf;
        }
        fold_score_vector<HAS_TEMP, TOP>(y, inv_t, g + u * kTileLanes, st);
      }
    };
    for (int b = 0; b + 1 < clean; ++b, g += kStep) clean_batch(BoolConstant<true>{}, b == 0);
    if (clean > 0) {
      clean_batch(BoolConstant<false>{}, clean == 1);
      g += kStep;
    }
    for (int b = clean; b * kBatch < slots; ++b, g += kStep) {  // the rest: clamped loads, both edges masked
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int gu = g + u * kTileLanes;
        raw[u].template load_edge<NT>(row_ptr, gu < g1 ? gu : g_last, a.V);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (b * kBatch + u >= slots) break;  // uniform
        const int gu = g + u * kTileLanes;
        float y[8];
        raw[u].unpack(y);
        const int lo = lo_col - gu * 8;
        const int hi = gu < g1 ? hi_col - gu * 8 : lo;  // columns [lo, hi) of the vector count
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (i >= lo && i < hi) ? y[i] : kNegInf;
        fold_score_vector<HAS_TEMP, TOP>(y, inv_t, gu, st);  // a vector of -inf changes nothing
      }
    }
    if constexpr (TOP) {
      const int64_t slice = (int64_t)row * kScoreSlices + tile * kTileLanes + l16;
      a.best[slice] = g0 + l16 < g1 ? ordered_bits(st.raw) : 0u;
      a.best_at[slice] = (uint32_t)st.at;
    }
    merge_score_lanes<8>(lane, st);
    merge_score_lanes<4>(lane, st);
    merge_score_lanes<2>(lane, st);
    merge_score_lanes<1>(lane, st);
    if (l16 == 0) {
      const bool finite = st.m > kNegInf && st.m < -kNegInf;
      float zt = 0.f;
      if (target >= lo_col && target < hi_col) {
        zt = LogitElem<ELEM>::to_float(row_ptr[target]);
        if (HAS_TEMP) zt = zt * inv_t;
      }
      float* out = a.stats + (int64_t)row * kScorePlanes * kScoreTiles + tile;
      out[0] = st.m;
      out[kScoreTiles] = finite ? st.s : 0.f;
      out[2 * kScoreTiles] = zt;
      out[3 * kScoreTiles] = finite ? st.w : 0.f;
    }
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
// A wave per row: the tiles of the row merged, and its alternatives.
// ---------------------------------------------------------------------------

struct ScoreFinishArgs {
  const void* logits;
  int64_t row_stride;
  const int64_t* target;
  const float* temperature;
  const float* row_lse;  // [T] or null: log-sum-exps that exist; logp and lse are then not written, no alternative is above 0
  const float* stats;
  const uint32_t* best;
  const uint32_t* best_at;
  float* logp;
  float* lse;
  float* entropy;
  float* top_logp;   // [T][top_k]
  int64_t* top_ids;  // [T][top_k]
  int T, V, real, tile_size, top_k;
};

constexpr int kFinishWaves = 4;
constexpr int kFinishKeys = 1024;    // candidates that are held at a time
constexpr int kFinishPicked = 128;   // slices
constexpr int kScoreMostTop = 64;

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v = v + __shfl_xor(v, offset);
  return v;
}
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor(v, offset));
  return v;
}

// What one lane of a wave wrote to LDS is seen by the others behind it.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The k largest of n different keys (k <= n <= kFinishKeys) move to the front of `keys`; returns the smallest of them.
__device__ __forceinline__ uint64_t keep_largest(uint64_t* keys, int n, int k, int lane) {
  constexpr int kEach = kFinishKeys / kWave;
  uint64_t mine[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine[i] = i * kWave + lane < n ? keys[i * kWave + lane] : 0;
  uint64_t floor = 0;  // the largest number that k keys are not under
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t trial = floor | (uint64_t)1 << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) count += __popcll(__ballot(mine[i] >= trial));
    if (count >= k) floor = trial;
  }
  wave_lds_sync();
  int kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint64_t mask = __ballot(mine[i] >= floor);
    if (mine[i] >= floor) keys[kept + lanes_below(mask)] = mine[i];
    kept += __popcll(mask);
  }
  wave_lds_sync();
  return floor;
}

template <int ELEM>
__device__ __forceinline__ void finish_alternatives(const ScoreFinishArgs& a, int row, int lane, float lse, float inv_t,
                                                    uint64_t* keys, uint16_t* picked) {
  using E = typename LogitElem<ELEM>::type;
  const int k = a.top_k;
  constexpr int kEach = kScoreSlices / kWave;  // a lane has the sixteen slices of one tile
  static_assert(kEach == kTileLanes, "a lane per tile");
  uint32_t most[kEach];
  const u32x4_t* src = reinterpret_cast<const u32x4_t*>(a.best + (int64_t)row * kScoreSlices + lane * kEach);
#pragma unroll
  for (int i = 0; i < kEach / 4; ++i) {
    const u32x4_t v = src[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) most[4 * i + e] = v[e];
  }
  auto count_from = [&](uint32_t limit) __attribute__((always_inline)) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) count += __popcll(__ballot(most[i] >= limit));
    return count;
  };
  uint32_t tile_most = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) tile_most = max(tile_most, most[i]);
  uint32_t high = tile_most, low = tile_most;
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    high = max(high, (uint32_t)__shfl_xor((int)high, offset));
    low = min(low, (uint32_t)__shfl_xor((int)low, offset));
  }
  high = __builtin_amdgcn_readfirstlane(high);
  low = max(__builtin_amdgcn_readfirstlane(low), 1u);  // 0: a slice without columns

  // Slices from a limit on that at least k of them reach and not many more (any such limit is as good as the k-th best).
  const int enough = k + k / 8 + 2;
  int reach = count_from(low);
  uint32_t beyond = high + 1;  // (high is the key of a number, under 2^32 - 1)
  while (reach > enough && beyond - low > 1) {
    const uint32_t mid = low + (beyond - low) / 2;
    const int count = count_from(mid);
    if (count >= k) {
      low = mid;
      reach = count;
    } else {
      beyond = mid;
    }
  }
  uint64_t floor = (uint64_t)low << 32;  // candidates are not under it; key = (ordered logit, columns behind it)
  uint32_t last_at = 0xffffffffu;
  uint32_t at[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) at[i] = 0;
  if (reach > enough) {  // many slices with the same best logit: the first of them, by the vector that holds it
    const u32x4_t* where = reinterpret_cast<const u32x4_t*>(a.best_at + (int64_t)row * kScoreSlices + lane * kEach);
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) {
      const u32x4_t v = where[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) at[4 * i + e] = v[e];
    }
    const int above = count_from(low + 1);
    uint32_t first = 0, end = (uint32_t)(a.V / 8);  // the smallest vector number up to which there are enough
    while (first < end) {
      const uint32_t mid = first + (end - first) / 2;
      int count = above;
#pragma unroll
      for (int i = 0; i < kEach; ++i) count += __popcll(__ballot(most[i] == low && at[i] <= mid));
      if (count >= k) end = mid; else first = mid + 1;
    }
    last_at = first;
    floor |= 0xffffffffu - min((uint64_t)0xffffffffu, (uint64_t)last_at * 8 + 7);
  }
  int slices = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool take = most[i] > low || (most[i] == low && at[i] <= last_at);
    const uint64_t mask = __ballot(take);
    if (take) picked[slices + lanes_below(mask)] = (uint16_t)(lane * kEach + i);
    slices += __popcll(mask);
  }
  wave_lds_sync();

  // The picked slices' vectors, a lane each, some of a lane's on their way while as many are looked at. An element costs a comparison with
  // the floor's logit, whose result is a mask over the lanes already; only masks that are not empty go on to the keys.
  const E* row_ptr = reinterpret_cast<const E*>(a.logits) + (int64_t)row * a.row_stride;
  const int rounds = ((a.tile_size + 14) / 8 + kTileLanes - 1) / kTileLanes;  // vectors of a slice, at most
  const uint32_t jobs = (uint32_t)(slices * rounds);  // (rounds <= 2^28 / 64 / 128 + 1)
  constexpr int kAhead = ELEM == RLK_DTYPE_FP32 ? 2 : 4;
  struct Piece {
    RowVector<ELEM> v;
    int g, lo, hi;  // columns [lo, hi) of vector g
  } now[kAhead], next[kAhead];
  auto fetch = [&](uint32_t job, Piece& p) __attribute__((always_inline)) {
    p.g = p.lo = p.hi = 0;
    if (job < jobs) {
      const int slice = picked[job / (uint32_t)rounds];
      const int tile = slice / kTileLanes;
      const int64_t lo64 = (int64_t)tile * a.tile_size, hi64 = lo64 + a.tile_size;
      const int lo_col = lo64 < a.real ? (int)lo64 : a.real;
      const int hi_col = hi64 < a.real ? (int)hi64 : a.real;
      const int g = lo_col / 8 + slice % kTileLanes + (int)(job % (uint32_t)rounds) * kTileLanes;
      if ((int64_t)g * 8 < hi_col) {
        p.g = g;
        p.lo = max(lo_col - g * 8, 0);
        p.hi = min(hi_col - g * 8, 8);
        p.v.template load_edge<false>(row_ptr, g, a.V);
      }
    }
  };
  int n = 0;
  float least = low > ordered_bits(kNegInf) ? from_ordered_bits(low) : kNegInf;  // the floor's logit
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(u * kWave + lane, next[u]);
  for (uint32_t first = 0; first < jobs; first += kAhead * kWave) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now[u] = next[u];
    if (first + kAhead * kWave < jobs) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) fetch(first + (kAhead + u) * kWave + lane, next[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (first + u * kWave >= jobs) break;
      float y[8];
      uint64_t hit[8], any = 0;
      now[u].v.unpack(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = fmaxf(y[i], kNegInf);  // (a NaN counts as -inf)
        hit[i] = __ballot(i >= now[u].lo && i < now[u].hi && y[i] >= least);
        any |= hit[i];
      }
      if (any == 0) continue;
      if (n > kFinishKeys - 8 * kWave) {
        floor = keep_largest(keys, n, k, lane);
        least = from_ordered_bits((uint32_t)(floor >> 32));
        n = k;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (hit[i] == 0) continue;
        const uint64_t key = (uint64_t)ordered_bits(y[i]) << 32 | (0xffffffffu - (uint32_t)(now[u].g * 8 + i));
        const bool take = ((hit[i] >> lane) & 1) != 0 && key >= floor;
        const uint64_t mask = __ballot(take);
        if (take) keys[n + lanes_below(mask)] = key;
        n += __popcll(mask);
      }
    }
    wave_lds_sync();
  }
  if (n > 2 * kWave) {
    keep_largest(keys, n, k, lane);
    n = k;
  }

  uint64_t mine[2];
  int rank[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) mine[i] = i * kWave + lane < n ? keys[i * kWave + lane] : 0;
  auto rank_against = [&](uint64_t of, int count) __attribute__((always_inline)) {
    for (int j = 0; j < count; ++j) {
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(of >> 32), j) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)of, j);
#pragma unroll
      for (int i = 0; i < 2; ++i) rank[i] += other > mine[i] ? 1 : 0;
    }
  };
  rank_against(mine[0], min(n, kWave));
  rank_against(mine[1], max(n - kWave, 0));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i * kWave + lane >= n || rank[i] >= k) continue;
    float v = from_ordered_bits((uint32_t)(mine[i] >> 32)) * inv_t - lse;
    if (a.row_lse != nullptr && v > 0.f) v = 0.f;  // the fused linear-LogP clamps its log-probabilities
    const int64_t out = (int64_t)row * k + rank[i];
    a.top_ids[out] = (int64_t)(0xffffffffu - (uint32_t)mine[i]);
    a.top_logp[out] = v;
  }
}

template <int ELEM>
__global__ __launch_bounds__(kFinishWaves * kWave) void score_finish_kernel(ScoreFinishArgs a) {
  __shared__ uint64_t keys[kFinishWaves][kFinishKeys];
  __shared__ uint16_t picked[kFinishWaves][kFinishPicked];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x * kFinishWaves + wave;
  if (row >= a.T) return;  // (waves share nothing)
  const float* stats = a.stats + (int64_t)row * kScorePlanes * kScoreTiles + lane;
  const float m = stats[0], s = stats[kScoreTiles], w = stats[3 * kScoreTiles];
  const float big = wave_max_f32(m);
  const float shrink = pinned_exp(m - big);
  const float term = m > kNegInf ? s * shrink : 0.f;
  float sum = 0.f;  // (ascending)
#pragma unroll
  for (int t = 0; t < kScoreTiles; ++t) sum = sum + __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(term), t));
  const float weighted = wave_sum_f32(m > kNegInf ? shrink * __builtin_fmaf(s, m - big, w) : 0.f);
  const float log_sum = logf(sum);
  const float temperature = a.temperature ? a.temperature[row] : 1.0f;
  const bool bad_temperature = !(temperature > 0.f);
  const float nan = __builtin_nanf("");
  float lse = a.row_lse ? a.row_lse[row] : big + log_sum;
  if (bad_temperature) lse = nan;
  const float zt = wave_sum_f32(stats[2 * kScoreTiles]);
  if (lane == 0) {
    a.entropy[row] = bad_temperature ? nan : log_sum - weighted / sum;
    if (a.row_lse == nullptr) {
      const bool bad_target = a.target[row] < 0 || a.target[row] >= a.real;
      a.lse[row] = lse;
      a.logp[row] = bad_target ? nan : zt - lse;
    }
  }
  if (a.top_k > 0) finish_alternatives<ELEM>(a, row, lane, lse, a.temperature ? 1.0f / temperature : 1.0f, keys[wave], picked[wave]);
}

// ---------------------------------------------------------------------------
// Gradient: dz = 1/T [ p (g_lse - g_logp - sum g_top - g_entropy (y - lse + entropy)) + g_logp [target] + g_top [ids] ],
// p = e(y - lse). Elementwise; rounded once to the element type of the output.
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

template <int ELEM, int OUT, bool STREAM>
__global__ __launch_bounds__(kScoreBackThreads) void score_backward_kernel(ScoreBackwardArgs a) {
  using E = typename LogitElem<ELEM>::type;
  using O = typename LogitElem<OUT>::type;
  __shared__ int hit_col[kScoreMostTop + 1];
  __shared__ float hit_grad[kScoreMostTop + 1];
  __shared__ int hit_count;
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
      top_sum = all;
    }
  }
  __syncthreads();
  const int hits = hit_count;
  const float lse = a.lse[row];
  const bool finite = lse > kNegInf && lse < -kNegInf;
  const float inv_t = a.temperature ? 1.0f / a.temperature[row] : 1.0f;
  const float g_entropy = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float entropy = a.g_entropy ? a.entropy[row] : 0.f;
  const float slope = (a.g_lse ? a.g_lse[row] : 0.f) - g_logp - top_sum;
  // lse and the gradients of the row in registers: from here on a logit costs an exponential and a few products
#pragma unroll
  for (int u = 0; u < kScoreBackVectors; ++u) {
    const int64_t col = first + (int64_t)(u * kScoreBackThreads + threadIdx.x) * 8;
    if (col >= a.grad_cols) break;
    float out[8];
    if (col < a.real && finite) {
      float z[8];
      raw[u].unpack(z);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = __builtin_fmaf(z[i], inv_t, -lse);  // log p
        const float p = pinned_exp(d);
        out[i] = p * __builtin_fmaf(-g_entropy, fmaxf(d, kFarBelow) + entropy, slope);
        out[i] = col + i < a.real ? out[i] : 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = 0.f;
    }
    for (int h = 0; h < hits; ++h) {
      const int at = hit_col[h] - (int)col;
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = at == i ? out[i] + hit_grad[h] : out[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = out[i] * inv_t;
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

template <int ELEM>
static hipError_t token_scores_typed(ScoreArgs a, const ScoreFinishArgs& f, dim3 grid, int threads, hipStream_t stream) {
  const bool temp = a.temperature != nullptr;
  if (f.top_k > 0) {
    if (temp) hipLaunchKernelGGL((score_tiles_kernel<ELEM, true, true>), grid, dim3(threads), 0, stream, a);
    else hipLaunchKernelGGL((score_tiles_kernel<ELEM, false, true>), grid, dim3(threads), 0, stream, a);
  } else {
    if (temp) hipLaunchKernelGGL((score_tiles_kernel<ELEM, true, false>), grid, dim3(threads), 0, stream, a);
    else hipLaunchKernelGGL((score_tiles_kernel<ELEM, false, false>), grid, dim3(threads), 0, stream, a);
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((score_finish_kernel<ELEM>), dim3((a.T + kFinishWaves - 1) / kFinishWaves), dim3(kFinishWaves * kWave), 0, stream, f);
  return hipGetLastError();
}

hipError_t token_scores_launch(const void* logits, int dtype, int64_t row_stride, const int64_t* target, const float* temperature,
                               const float* row_lse, int T, int V, int real, int top_k, float* logp, float* lse, float* entropy,
                               float* top_logp, int64_t* top_ids, void* workspace, hipStream_t stream) {
  ScoreArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.target = target;
  a.temperature = temperature;
  a.stats = reinterpret_cast<float*>(workspace);
  a.best = reinterpret_cast<uint32_t*>(a.stats + (size_t)T * kScorePlanes * kScoreTiles);
  a.best_at = a.best + (size_t)T * kScoreSlices;
  a.T = T;
  a.V = V;
  a.real = real;
  a.tile_size = (int)(((int64_t)V + kScoreTiles - 1) / kScoreTiles);
  a.tiles_per_group = kScoreTiles;
  while ((int64_t)T * (kScoreTiles / a.tiles_per_group) < 16384 && a.tiles_per_group > 16) a.tiles_per_group /= 2;
  const int groups = kScoreTiles / a.tiles_per_group;
  const int64_t bytes = (int64_t)T * V * (dtype == RLK_DTYPE_FP32 ? 4 : 2);
  a.streamed = bytes > kCachedLogitsBytes ? (int64_t)((double)T * groups * (1.0 - (double)kCachedLogitsBytes / bytes)) : 0;
  const ScoreFinishArgs f{logits, row_stride, target, temperature, row_lse, a.stats, a.best, a.best_at, logp, lse, entropy,
                          top_logp, top_ids, T, V, real, a.tile_size, top_k};
  const dim3 grid((unsigned)T, (unsigned)groups);
  switch (dtype) {
    case RLK_DTYPE_BF16: return token_scores_typed<RLK_DTYPE_BF16>(a, f, grid, 256, stream);
    case RLK_DTYPE_FP16: return token_scores_typed<RLK_DTYPE_FP16>(a, f, grid, 256, stream);
    case RLK_DTYPE_FP32: return token_scores_typed<RLK_DTYPE_FP32>(a, f, grid, 256, stream);
    default: return hipErrorInvalidValue;
  }
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
