// Attention of new tokens over a paged cache for gfx950: single tokens, chunks of a prompt, whole prompts.
//
// Rows. A sequence's new tokens and the heads that share a key head are rows of one matrix, token by token, so that every key and
// value that is read serves all of them. A tile is a run of such rows of one sequence and one key head.
//
// Sums. Scores come transposed, S^T = K Q^T: the matrix instruction's result then has a row's scores in four lanes (and its
// statistics need two lane swaps), and two 16-key blocks of it, rounded to 16 bits, are the operand of O^T = V^T P^T as they
// stand: slot 8 g + e of lane group g holds key 16 (e / 4) + 4 g + e % 4 of 32, and the transposing LDS read brings the values in
// that order. Each of a row's four lanes sums the weights of its own keys; they meet at the end of a run.
//   tile of 64 keys:  m' = max(m, max s),  a = 2^(m - m'),  p = 2^(s - m'),  o = a o + round(p) V,  l = a l + sum p
// with s in units of log2(e) * scale. A run of tiles starts from nothing; runs are combined in ascending order:
//   M' = max(M, m),  O = 2^(m - M') o + 2^(M - M') O  (one fused step), L likewise;  out = O / L,  lse = ln 2 (M + log2 L)
// Which keys form a tile and which tiles a run is a function of their positions, and keys that a row does not see leave its chain as it is (a
// factor of 1, a sum with 0). So a row's bits are the same in every kernel below, however its runs are spread over the chip.
// Statistics and outputs are fp32 throughout; weights are rounded to the inputs' 16 bits for the matrix units (half a step, 2^-9 of a
// weight in bf16, which averages out over the keys), not for their sum: its logarithm is an answer in 32 bits.
//
// What a row does not see may hold anything. Scores are replaced, not added to. Keys and values that no row of a tile sees are
// read as zeros. Where some rows see a value and others do not, a zero weight would not save them from infinities and NaN in
// it: such a tile is looked through before it is used, and if it holds any they are taken out of the product and added to the
// rows that see them.
#include "paged.h"

namespace rlk {

constexpr int kTileKeys = 64;
constexpr int kSlabBytes = kTileKeys * 128;  // 64 keys x 64 elements
constexpr int kMaxWidth = 256;
constexpr int kMostKeys = 0x7fffff00;  // of a sequence

// Runs: their lengths grow with the position, so that a short context still has enough of them for the chip and a long
// one's partial results stay few. Tiles 0 ... 63 in fours, ... 255 in eights, ... 1023 in sixteens, then 32 at a time.
__host__ __device__ __forceinline__ int run_of_tile(int t) {
  return t < 64 ? t >> 2 : t < 256 ? 16 + ((t - 64) >> 3) : t < 1024 ? 40 + ((t - 256) >> 4) : 88 + ((t - 1024) >> 5);
}
__host__ __device__ __forceinline__ int run_first_tile(int r) {
  return r < 16 ? 4 * r : r < 40 ? 64 + 8 * (r - 16) : r < 88 ? 256 + 16 * (r - 40) : 1024 + 32 * (r - 88);
}

// What a lane reads where there is no key (zeros) and where its page is missing (NaN in either type), a head's width of each.
#define RLK_4(x) x, x, x, x
#define RLK_64(x) RLK_4(RLK_4(RLK_4(x)))
__device__ const __align__(16) uint16_t kSpecialRows[2][kMaxWidth] = {{RLK_4(RLK_64(0))}, {RLK_4(RLK_64(0x7fff))}};
#undef RLK_64
#undef RLK_4

struct AttentionArgs {
  rlk_paged_cache cache;
  const char* q;
  char* out;
  float* lse;
  float* part_out;  // [run][token][head][width]
  float* part_max;  // [run][token][head]
  float* part_sum;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // bytes
  int64_t part_rows;  // tokens * heads
  PageDivider by_page, by_group, by_key_heads;
  int tokens, heads, group, causal, window, zero_rest, tiles, chunks;
  float scale;  // times log2(e)
};

template <int DTYPE>
struct Half;
template <>
struct Half<RLK_DTYPE_BF16> {
  static constexpr uint32_t kOnes = 0x3f803f80u, kExponent = 0x7f807f80u, kLowest = 0x00800080u, kFraction = 0x007f007fu;
  static constexpr uint32_t k128 = 0x4300u, k16384 = 0x4680u;
  static __device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) { return mfma_16x16x32(a, b, c); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Half<RLK_DTYPE_FP16> {
  static constexpr uint32_t kOnes = 0x3c003c00u, kExponent = 0x7c007c00u, kLowest = 0x04000400u, kFraction = 0x03ff03ffu;
  static constexpr uint32_t k128 = 0x5800u, k16384 = 0x7400u;
  static __device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16;
  }
};

// Bits 15 and 31: whether the two numbers of a word are infinite or NaN.
template <int DTYPE>
__device__ __forceinline__ uint32_t special_halves(uint32_t w) {
  return ((w & Half<DTYPE>::kExponent) + Half<DTYPE>::kLowest) & 0x80008000u;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest value of a row over the four lanes that hold it (lanes l, l + 16, l + 32, l + 48). NaN loses, as in fmaxf.
__device__ __forceinline__ float max_over_groups(float v) {
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const uint32_t u = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// The sum of what the four lanes of a row hold, in one order.
__device__ __forceinline__ float sum_over_groups(float v) {
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const uint32_t u = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// Four values of one element, of four consecutive keys (see read_kmajor_fragment in det_gemm_tile.h, also for the qualifier).
typedef const __attribute__((address_space(3))) char* value_bytes_t;
__device__ __forceinline__ u32x2_t read_values_transposed(value_bytes_t __restrict__ at) {
  typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;
  typedef __attribute__((address_space(3))) bf16x4_t* lds_bf16x4_ptr_t;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_ptr_t)at));
}
__device__ __forceinline__ u32x4_t read_chunk(value_bytes_t __restrict__ at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(at);
}

// LDS image of a tile: slabs of 64 elements, each 64 rows (keys) of 128 bytes, as the direct loads lay blocks of 8 rows down.
// Chunks of 16 bytes change places within a row so that the reads are free of bank conflicts: by the row's last three bits for
// keys (16 lanes read one chunk of 16 rows), by twice its bits 1 and 2 for values (32 lanes read 32 bytes of 8 rows, two rows
// to 256 bytes of banks).
__device__ __forceinline__ int key_swizzle(int row) { return row & 7; }
__device__ __forceinline__ int value_swizzle(int row) { return 2 * ((row >> 1) & 3); }

// One sequence's part of a launch.
struct Chunk {
  int sequence, first_token, tokens, length;
};

// What a row (of the 16 of a block, lane & 15) sees: keys [low, high).
struct Sight {
  int low, high;
};
__device__ __forceinline__ Sight sight_of(const AttentionArgs& a, const Chunk& c, int token) {
  const int64_t position = (int64_t)c.length - c.tokens + token;  // may be below 0: such a token sees nothing
  Sight s;
  s.high = a.causal ? (int)(position + 1 > 0 ? position + 1 : 0) : c.length;
  s.low = a.window > 0 && s.high > a.window ? s.high - a.window : 0;
  return s;
}

__device__ __forceinline__ int clamp_to(int64_t v, int low, int high) { return v < low ? low : v > high ? high : (int)v; }

__device__ __forceinline__ Chunk chunk_of(const AttentionArgs& a, int sequence) {
  Chunk c;
  c.sequence = sequence;
  c.first_token = clamp_to(a.cache.starts[sequence], 0, a.tokens);
  c.tokens = clamp_to(a.cache.starts[sequence + 1], c.first_token, a.tokens) - c.first_token;
  const int length = a.cache.lengths[sequence];
  c.length = length > 0 ? length : 0;
  return c;
}

// Positions that the page table has room for. A row that sees more of them sees the one behind, which is missing.
__host__ __device__ __forceinline__ int capacity_of(const rlk_paged_cache& c) {
  const int64_t keys = (int64_t)c.table_columns * c.page_size;
  return keys < kMostKeys ? (int)keys : kMostKeys;
}
__device__ __forceinline__ int capacity_of(const AttentionArgs& a) { return capacity_of(a.cache); }

// Where row tiles lie: sequence s has those from floor(starts[s] * group / rows) + s on, at least as many as it needs.
template <int ROWS>
__device__ __forceinline__ int64_t first_row_tile(const AttentionArgs& a, int s) {
  return (int64_t)clamp_to(a.cache.starts[s], 0, a.tokens) * a.group / ROWS + s;
}

// The running state of RB blocks of 16 rows of a wave. Lane l holds row l & 15 of each; of the output elements 16 d + 4 (l >> 4) + i.
template <int DTYPE, int SLABS, int RB, bool KEEP_Q = true>
struct Rows {
  typedef Half<DTYPE> H;
  static constexpr int kBlocks = 4 * SLABS;  // of 16 elements
  static constexpr int kSteps = 2 * SLABS;   // of 32 elements
  u32x4_t q[KEEP_Q ? kSteps : 1][RB];  // (or they stay in LDS)
  f32x4_t o[kBlocks][RB];
  float m[RB];
  float l[RB];  // the sum of the weights of this lane's keys
  Sight sight[RB];

  __device__ __forceinline__ void load_q(const AttentionArgs& a, int key_head, const int (&token)[RB], const int (&head)[RB], const bool (&live)[RB],
                                         int l16, int grp, char* shelf) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const char* row = a.q + (int64_t)token[rb] * a.q_token_stride + (int64_t)(key_head * a.group + head[rb]) * a.q_head_stride;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        const int element = 32 * ks + 8 * grp;
        const u32x4_t v = live[rb] && element < a.cache.width ? *reinterpret_cast<const u32x4_t*>(row + 2 * element) : u32x4_t{0, 0, 0, 0};
        if (KEEP_Q)
          q[KEEP_Q ? ks : 0][rb] = v;
        else
          *reinterpret_cast<u32x4_t*>(shelf + (rb * SLABS + (ks >> 1)) * 2048 + l16 * 128 + (((4 * (ks & 1) + grp) ^ key_swizzle(l16)) << 4)) = v;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      l[rb] = 0.f;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) o[d][rb] = f32x4_t{0, 0, 0, 0};
    }
  }

  // Scores of a tile, s[b][rb] of keys key0 + 16 b + 4 grp + i: those of keys that a row does not see go.
  __device__ __forceinline__ void mask(f32x4_t (&s)[4][RB], int key0, int grp) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const uint32_t range = sight[rb].high > sight[rb].low ? sight[rb].high - sight[rb].low : 0;
      const uint32_t from = (uint32_t)(key0 + 4 * grp - sight[rb].low);
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b][rb][i] = from + 16 * b + i < range ? s[b][rb][i] : -INFINITY;
    }
  }

  // Scores to weights; the state is taken to the new maximum.
  __device__ __forceinline__ void weigh(const AttentionArgs& a, const f32x4_t (&s)[4][RB], u32x4_t (&p)[2][RB]) {
    float before[RB];
    bool moved = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float top = s[0][rb][0];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[b][rb][i]);
      before[rb] = m[rb];
      m[rb] = fmaxf(m[rb], max_over_groups(top) * a.scale);
      moved |= m[rb] != before[rb];
    }
    if (__any(moved)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float f = m[rb] != before[rb] ? exp2_fast(before[rb] - m[rb]) : 1.f;
        l[rb] *= f;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) o[d][rb] *= f;
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float from = m[rb] == -INFINITY ? 0.f : m[rb];
      float sum[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4_t& v = s[2 * h + (e >> 1)][rb];
          const float x = exp2_fast(__builtin_fmaf(v[2 * (e & 1)], a.scale, -from)), y = exp2_fast(__builtin_fmaf(v[2 * (e & 1) + 1], a.scale, -from));
          sum[h][e] = x + y;
          p[h][rb][e] = H::pack(x, y);
        }
      l[rb] += ((sum[0][0] + sum[0][1]) + (sum[0][2] + sum[0][3])) + ((sum[1][0] + sum[1][1]) + (sum[1][2] + sum[1][3]));
    }
  }

  // A lane's place in the values' image: for element blocks 0 ... 3 of a slab.
  struct ValuePlace {
    int at[4];
    __device__ __forceinline__ void init(int l16, int grp) {
      const int row = 4 * grp + (l16 >> 2);
#pragma unroll
      for (int d = 0; d < 4; ++d) at[d] = row * 128 + (((2 * d + ((l16 >> 1) & 1)) ^ value_swizzle(row)) << 4) + (l16 & 1) * 8;
    }
  };
  static __device__ __forceinline__ u32x4_t value_fragment(value_bytes_t tile, int place, int d, int h) {
    const value_bytes_t at = tile + place + (d >> 2) * kSlabBytes + h * 4096;
    const u32x2_t x = read_values_transposed(at), y = read_values_transposed(at + 2048);
    return u32x4_t{x.x, x.y, y.x, y.y};
  }

  // Fragments are read a few products ahead of their use.
  static constexpr int kAhead = 4;
  __device__ __forceinline__ void add_values(value_bytes_t tile, const ValuePlace& place, const u32x4_t (&p)[2][RB]) {
    u32x4_t v[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) v[n] = value_fragment(tile, place.at[n & 3], n, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 2 * kBlocks; ++n) {
      const int d = n % kBlocks, h = n / kBlocks, next = n + kAhead;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) o[d][rb] = H::mfma(v[n % kAhead], p[h][rb], o[d][rb]);
      if (next < 2 * kBlocks) v[n % kAhead] = value_fragment(tile, place.at[next & 3], next % kBlocks, next / kBlocks);
      __builtin_amdgcn_sched_barrier(0);  // (or the reads move back to their use)
    }
  }

  // A tile with infinities or NaN among the values that some rows see and others do not. They leave the product (take_out), and what they
  // make of an element is added to it behind (an infinity, or NaN where both come together, from NaN, or from an infinity
  // with a weight of 0). One more product counts them: 1 for inf, 128 for -inf, 16384 for NaN, 64 at most of each. The results wait
  // in memory, and nothing here is unrolled: this is rare, and in registers it would cost the ordinary tiles theirs.
  __device__ __forceinline__ void find_special(value_bytes_t tile, const ValuePlace& place, const u32x4_t (&p)[2][RB], int key0, int grp, volatile float* effect) {
    const uint32_t one = H::kOnes & 0xffffu;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const uint32_t range = sight[rb].high > sight[rb].low ? sight[rb].high - sight[rb].low : 0;
#pragma unroll 1
      for (int d = 0; d < kBlocks; ++d) {
        f32x4_t count = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4_t v = value_fragment(tile, place.at[0] ^ ((d & 3) << 5), d, h);
          u32x4_t kinds, any, seen, lost;  // of the values; 1 where a row sees a key with a weight, and without one
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t from = (uint32_t)(key0 + 32 * h + 16 * (e >> 1) + 4 * grp + 2 * (e & 1) - sight[rb].low);
            const uint32_t sees = (from < range ? 0x8000u : 0u) | (from + 1 < range ? 0x80000000u : 0u);
            const uint32_t weighs = ((p[h][rb][e] & 0x7fff7fffu) + 0x7fff7fffu) & sees;
            seen[e] = (weighs >> 15) * one;
            lost[e] = ((sees ^ weighs) >> 15) * one;
            const uint32_t w = v[e], special = special_halves<DTYPE>(w);
            const uint32_t none = special & ((w & H::kFraction) + 0x7fff7fffu);
            kinds[e] = ((special & ~none & ~w) >> 15) * one | ((special & ~none & w) >> 15) * H::k128 | (none >> 15) * H::k16384;
            any[e] = (special >> 15) * H::k16384;
          }
          count = H::mfma(kinds, seen, count);
          count = H::mfma(any, lost, count);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t n = (uint32_t)count[i];
          const float up = (n & 127) != 0 ? INFINITY : 0.f, down = (n & (127 << 7)) != 0 ? -INFINITY : 0.f;
          effect[4 * (d * RB + rb) + i] = n >= 16384 ? NAN : up + down;
        }
      }
    }
  }
  __device__ __forceinline__ void add_special(const volatile float* effect) {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][rb][i] += effect[4 * (d * RB + rb) + i];
  }
};

// Zeros in the place of a chunk's infinities and NaN.
template <int DTYPE>
__device__ __forceinline__ void take_out_special(char* at) {
  typedef __attribute__((address_space(3))) u32x4_t* chunk_ptr_t;
  u32x4_t w = *(chunk_ptr_t)at;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] &= ~((special_halves<DTYPE>(w[e]) >> 15) * 0xffffu);
  *(chunk_ptr_t)at = w;
}

// A run joins those before it: factors for both, and the new maximum.
struct Join {
  float kept, added;
};
__device__ __forceinline__ Join join_maxima(float& all, float run) {
  const float top = fmaxf(all, run);
  Join j;
  j.kept = top == all ? 1.f : exp2_fast(all - top);
  j.added = top == run ? 1.f : exp2_fast(run - top);
  all = top;
  return j;
}
__device__ __forceinline__ float join_sums(float all, float run, const Join& j) { return __builtin_fmaf(run, j.added, all * j.kept); }

// An output element; -0 becomes +0, whose sign would depend on tiles that a row does not see.
__device__ __forceinline__ float output_of(float sum, float reciprocal) { return sum * reciprocal + 0.f; }
__device__ __forceinline__ float lse_of(float top, float sum) { return 0.6931471805599453f * (top + __builtin_amdgcn_logf(sum)); }

// Loads a wave's share of a tile, GROUPS groups of 8 keys (the WAVES-th ones), straight into LDS.
template <int SLABS>
struct TileLoader {
  const char *keys, *values;  // of the key head
  int64_t key_page, key_row, value_page, value_row;  // bytes
  int key_chunk, value_chunk;  // of this lane's 16 bytes in a slab's row

  __device__ __forceinline__ void init(const AttentionArgs& a, int key_head, int lane) {
    keys = static_cast<const char*>(a.cache.keys) + 2 * key_head * a.cache.key_head_stride;
    values = static_cast<const char*>(a.cache.values) + 2 * key_head * a.cache.value_head_stride;
    key_page = 2 * a.cache.key_page_stride, key_row = 2 * a.cache.key_row_stride;
    value_page = 2 * a.cache.value_page_stride, value_row = 2 * a.cache.value_row_stride;
    key_chunk = (lane & 7) ^ key_swizzle(lane >> 3);
    value_chunk = (lane & 7) ^ value_swizzle(lane >> 3);
  }
};

// Where a key's row lies. Its table entry is asked for a tile ahead and looked at when the tile is loaded: looked at sooner, it would
// be waited for together with every load in flight.
struct KeyPlace {
  int entry;
  __device__ __forceinline__ void ask(const AttentionArgs& a, int sequence, int key) {
    const int column = (int)divide_by((uint32_t)key, a.by_page), last = a.cache.table_columns - 1;
    const int32_t* from = last >= 0 ? a.cache.table + (int64_t)sequence * a.cache.table_row_stride + min(column, last) : a.cache.starts;
    entry = *from;
  }
};
// The start of a key's row in a cache: zeros where the tile does not need the key, NaN where its page is missing.
__device__ __forceinline__ const char* key_row_address(const AttentionArgs& a, const char* base, int64_t page_bytes, int64_t row_bytes, int entry, int key,
                                                       int low, int high) {
  const int column = (int)divide_by((uint32_t)key, a.by_page);
  const int row = key - column * a.cache.page_size;
  const bool there = (uint32_t)entry < (uint32_t)a.cache.pages && column < a.cache.table_columns;
  const bool wanted = key >= low && key < high;
  const char* const special = reinterpret_cast<const char*>(kSpecialRows[wanted]);
  return wanted && there ? base + entry * page_bytes + row * row_bytes : special;
}

// ---------------------------------------------------------------------------
// Many rows: WAVES waves of 16 RB rows each share the keys and values of their tile through LDS, two tiles deep, one barrier a
// tile. SPLIT: a workgroup takes every chunks-th run and leaves the parts in memory.
// ---------------------------------------------------------------------------
template <int DTYPE, int SLABS, int RB, int WAVES, bool SPLIT>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_tile_kernel(const AttentionArgs a) {
  constexpr bool kKeepQ = RB == 1;
  typedef Rows<DTYPE, SLABS, RB, kKeepQ> State;
  constexpr int kRows = 16 * RB * WAVES;
  constexpr int kGroups = 8 / WAVES;  // groups of 8 keys that a wave loads
  constexpr int kTileBytes = SLABS * kSlabBytes;
  // [2][keys, values], then the queries, block of 16 rows by block, unless they are in registers, then special_tile. Nothing lies in
  // front of it: 16-byte reads that start on 8 bytes took 62 cycles each instead of 8, and the kernel twice as long.
  extern __shared__ __align__(16) char lds[];
  int* const special_tile = reinterpret_cast<int*>(lds + 4 * kTileBytes + (kKeepQ ? 0 : WAVES * RB * SLABS * 2048));  // [2]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, grp = lane >> 4;

  // Heads change fastest, so that an XCD's workgroups read few of them; the tiles with the most keys come first.
  const uint32_t id = blockIdx.x;
  const uint32_t outer = divide_by(id, a.by_key_heads);
  const int key_head = (int)(id - outer * a.cache.key_heads);
  const int chunk_id = SPLIT ? (int)(outer % (uint32_t)a.chunks) : 0;
  const int tile_id = a.tiles - 1 - (int)(SPLIT ? outer / (uint32_t)a.chunks : outer);
  const int s = wave_search(a.cache.sequences + 1, tile_id, lane, [&](int i) { return first_row_tile<kRows>(a, i); });
  if (s >= a.cache.sequences) {  // behind the last sequence
    if (!SPLIT && a.zero_rest) {
      const int before = clamp_to(a.cache.starts[0], 0, a.tokens), behind = clamp_to(a.cache.starts[s], before, a.tokens);
      const int tail = tile_id - (int)first_row_tile<kRows>(a, s), tails = a.tiles - (int)first_row_tile<kRows>(a, s);
      const int each = a.cache.width / 8;
      for (int n = tail; n < before + a.tokens - behind; n += tails) {
        const int t = n < before ? n : behind + n - before;
        for (int i = tid; i < a.group * each; i += WAVES * 64) {
          const int head = key_head * a.group + i / each;
          *reinterpret_cast<u32x4_t*>(a.out + t * a.out_token_stride + head * a.out_head_stride + (i % each) * 16) = u32x4_t{0, 0, 0, 0};
          if (a.lse && i % each == 0) a.lse[(int64_t)t * a.heads + head] = -INFINITY;
        }
      }
    }
    return;
  }
  if (s < 0) return;
  const Chunk c = chunk_of(a, s);
  const int rows = c.tokens * a.group;
  const int row0 = (int)(tile_id - first_row_tile<kRows>(a, s)) * kRows;
  if (row0 >= rows) return;

  // What this workgroup's and this wave's rows see.
  const int last_row = min(row0 + kRows, rows) - 1;
  const Sight first_sight = sight_of(a, c, (int)divide_by(row0, a.by_group)), last_sight = sight_of(a, c, (int)divide_by(last_row, a.by_group));
  const int capacity = capacity_of(a);
  const int low = first_sight.low, high = min(last_sight.high, capacity + 1);
  const int wave_row0 = row0 + wave * 16 * RB, wave_row1 = min(wave_row0 + 16 * RB, rows) - 1;
  const bool wave_live = wave_row0 < rows;
  const Sight wave_first = sight_of(a, c, (int)divide_by(wave_live ? wave_row0 : row0, a.by_group));
  const Sight wave_last = sight_of(a, c, (int)divide_by(wave_live ? wave_row1 : row0, a.by_group));

  State st;
  int token[RB], head[RB];
  bool live[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = wave_row0 + 16 * rb + l16;
    live[rb] = row < rows;
    const int t = (int)divide_by(live[rb] ? row : row0, a.by_group);
    head[rb] = (live[rb] ? row : row0) - t * a.group;
    token[rb] = c.first_token + t;
    st.sight[rb] = live[rb] ? sight_of(a, c, t) : Sight{0, 0};
  }
  char* const shelf = lds + 4 * kTileBytes + wave * RB * SLABS * 2048;
  st.load_q(a, key_head, token, head, live, l16, grp, shelf);
  st.clear();
  if (tid < 2) special_tile[tid] = 0;

  TileLoader<SLABS> loader;
  loader.init(a, key_head, lane);
  typename State::ValuePlace place;
  place.init(l16, grp);
  int key_at[2];  // this lane's chunks of a key block for even and odd steps
#pragma unroll
  for (int h = 0; h < 2; ++h) key_at[h] = l16 * 128 + (((4 * h + grp) ^ key_swizzle(l16)) << 4);

  const int end_tile = (high + kTileKeys - 1) / kTileKeys;
  int run = run_of_tile(low / kTileKeys) + chunk_id;
  int t = SPLIT ? max(run_first_tile(run), low / kTileKeys) : low / kTileKeys;
  auto next_tile = [&](int tile) {
    if (!SPLIT) return tile + 1;
    const int r = run_of_tile(tile);
    return tile + 1 < run_first_tile(r + 1) ? tile + 1 : run_first_tile(r + a.chunks);
  };
  KeyPlace where[kGroups];  // of the tile that is loaded next
  auto find_pages = [&](int tile) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) where[j].ask(a, s, tile * kTileKeys + (wave + j * WAVES) * 8 + (lane >> 3));
  };
  auto load_tile = [&](int tile, int stage) {
    char* const to = lds + stage * 2 * kTileBytes;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int group_of_keys = wave + j * WAVES;
      const int key = tile * kTileKeys + group_of_keys * 8 + (lane >> 3);
      const char* k = key_row_address(a, loader.keys, loader.key_page, loader.key_row, where[j].entry, key, low, high);
      const char* v = key_row_address(a, loader.values, loader.value_page, loader.value_row, where[j].entry, key, low, high);
      const char* const none = reinterpret_cast<const char*>(kSpecialRows[0]);
#pragma unroll
      for (int slab = 0; slab < SLABS; ++slab) {
        const int kc = slab * 8 + loader.key_chunk, vc = slab * 8 + loader.value_chunk;
        const char* ks = kc * 8 < a.cache.width ? k + kc * 16 : none;
        const char* vs = vc * 8 < a.cache.width ? v + vc * 16 : none;
        __builtin_amdgcn_global_load_lds((global_ptr_t)ks, (lds_ptr_t)(to + slab * kSlabBytes + group_of_keys * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((global_ptr_t)vs, (lds_ptr_t)(to + kTileBytes + slab * kSlabBytes + group_of_keys * 1024), 16, 0, 0);
      }
    }
  };

  // Runs combined so far.
  f32x4_t all_o[SPLIT ? 1 : State::kBlocks][RB];
  float all_m[RB], all_l[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    all_m[rb] = -INFINITY, all_l[rb] = 0.f;
#pragma unroll
    for (int d = 0; d < (SPLIT ? 1 : State::kBlocks); ++d) all_o[d][rb] = f32x4_t{0, 0, 0, 0};
  }

  int stage = 0;
  if (t < end_tile) {
    find_pages(t);
    load_tile(t, 0);
    const int next = next_tile(t);
    if (next < end_tile) find_pages(next);
  }
  wg_barrier();  // special_tile is there
  while (t < end_tile) {
    const int key0 = t * kTileKeys;
    const int next = next_tile(t);
    // some rows of the workgroup see a key that others do not
    const bool mixed = min(key0 + kTileKeys, high) > first_sight.high || max(key0, low) < last_sight.low;
    __builtin_amdgcn_s_waitcnt(kWaitAll0);  // my part of the tile has landed, and I have read what I wanted of the one before
    asm volatile("" ::: "memory");
    if (mixed) {
      uint32_t special = 0;
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
#pragma unroll
        for (int slab = 0; slab < SLABS; ++slab) {
          const u32x4_t w = read_chunk((value_bytes_t)(lds + stage * 2 * kTileBytes + kTileBytes + slab * kSlabBytes + (wave + j * WAVES) * 1024 + lane * 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) special |= special_halves<DTYPE>(w[e]);
        }
      if (special != 0) special_tile[stage] = t + 1;
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    }
    wg_barrier();  // everybody's has, and the other stage is no longer read
    if (next < end_tile) {
      load_tile(next, stage ^ 1);
      const int after = next_tile(next);
      if (after < end_tile) find_pages(after);
    }
    const bool special = mixed && special_tile[stage] == t + 1;
    const bool busy = wave_live && key0 < wave_last.high && key0 + kTileKeys > wave_first.low;
    const value_bytes_t keys = (value_bytes_t)(lds + stage * 2 * kTileBytes), values = keys + kTileBytes;
    u32x4_t p[2][RB];
    volatile float effect[4 * State::kBlocks * RB];  // (in memory, see find_special)
    if (busy) {
      f32x4_t scores[4][RB];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) scores[b][rb] = f32x4_t{0, 0, 0, 0};
      constexpr int kAhead = 4;
      u32x4_t k[kAhead], q[2][RB];
      auto key_fragment = [&](int n) { return read_chunk(keys + key_at[(n >> 2) & 1] + (n >> 3) * kSlabBytes + (n & 3) * 2048); };
      auto query_fragment = [&](int ks, int rb) {
        return kKeepQ ? st.q[kKeepQ ? ks : 0][rb] : read_chunk((value_bytes_t)shelf + key_at[ks & 1] + (rb * SLABS + (ks >> 1)) * 2048);
      };
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) q[0][rb] = query_fragment(0, rb);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) k[n] = key_fragment(n);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 4 * State::kSteps; ++n) {
        const int ks = n >> 2, b = n & 3;
        if (b == 0 && ks + 1 < State::kSteps)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) q[(ks + 1) & 1][rb] = query_fragment(ks + 1, rb);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) scores[b][rb] = Half<DTYPE>::mfma(k[n % kAhead], q[ks & 1][rb], scores[b][rb]);
        if (n + kAhead < 4 * State::kSteps) k[n % kAhead] = key_fragment(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);  // (or the reads move back to their use)
      }
      if (key0 + kTileKeys > wave_first.high || key0 < wave_last.low) st.mask(scores, key0, grp);
      st.weigh(a, scores, p);
    }
    if (special) {
      if (busy) st.find_special(values, place, p, key0, grp, effect);
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
      wg_barrier();
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
#pragma unroll
        for (int slab = 0; slab < SLABS; ++slab)
          take_out_special<DTYPE>(lds + stage * 2 * kTileBytes + kTileBytes + slab * kSlabBytes + (wave + j * WAVES) * 1024 + lane * 16);
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
      wg_barrier();
    }
    if (busy) st.add_values(values, place, p);
    if (special && busy) st.add_special(effect);
    const int this_run = run_of_tile(t);
    if (next >= end_tile || run_of_tile(next) != this_run) {  // the run ends
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float sum = sum_over_groups(st.l[rb]);
        if (SPLIT) {
          if (live[rb]) {
            const int64_t at = (int64_t)this_run * a.part_rows + (int64_t)token[rb] * a.heads + key_head * a.group + head[rb];
            if (grp == 0) a.part_max[at] = st.m[rb], a.part_sum[at] = sum;
#pragma unroll
            for (int d = 0; d < State::kBlocks; ++d)
              if (16 * d + 4 * grp < a.cache.width) *reinterpret_cast<f32x4_t*>(a.part_out + at * a.cache.width + 16 * d + 4 * grp) = st.o[d][rb];
          }
        } else if (sum != 0.f) {  // (NaN is a sum too)
          const Join j = join_maxima(all_m[rb], st.m[rb]);
          all_l[rb] = join_sums(all_l[rb], sum, j);
#pragma unroll
          for (int d = 0; d < State::kBlocks; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) all_o[SPLIT ? 0 : d][rb][i] = join_sums(all_o[SPLIT ? 0 : d][rb][i], st.o[d][rb][i], j);
        }
      }
      st.clear();
    }
    t = next;
    stage ^= 1;
  }
  if (SPLIT) return;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    if (!live[rb]) continue;
    const bool sees = st.sight[rb].high > st.sight[rb].low;
    const float reciprocal = sees ? 1.f / all_l[rb] : 0.f;
    char* to = a.out + (int64_t)token[rb] * a.out_token_stride + (int64_t)(key_head * a.group + head[rb]) * a.out_head_stride;
#pragma unroll
    for (int d = 0; d < State::kBlocks; ++d) {
      const f32x4_t& o = all_o[SPLIT ? 0 : d][rb];
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = sees ? output_of(o[i], reciprocal) : 0.f;
      if (16 * d + 4 * grp < a.cache.width)
        *reinterpret_cast<u32x2_t*>(to + 2 * (16 * d + 4 * grp)) = u32x2_t{Half<DTYPE>::pack(y[0], y[1]), Half<DTYPE>::pack(y[2], y[3])};
    }
    if (a.lse && grp == 0) a.lse[(int64_t)token[rb] * a.heads + key_head * a.group + head[rb]] = sees ? lse_of(all_m[rb], all_l[rb]) : -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Few rows: a wave takes 16 rows and every chunks-th run, on its own. Keys go straight into registers (a lane reads the pieces
// of its key that the matrix instruction wants), values through the wave's own two tiles of LDS.
// ---------------------------------------------------------------------------
constexpr int kRowWaves = 2;

template <int DTYPE, int SLABS>
__global__ __launch_bounds__(kRowWaves * 64) void attention_rows_kernel(const AttentionArgs a) {
  typedef Rows<DTYPE, SLABS, 1> State;
  constexpr int kRows = 16;
  constexpr int kTileBytes = SLABS * kSlabBytes;
  extern __shared__ __align__(16) char lds[];  // [wave][2][values]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, grp = lane >> 4;
  char* const mine = lds + wave * 2 * kTileBytes;

  const uint32_t id = blockIdx.x;
  const uint32_t outer = divide_by(id, a.by_key_heads);
  const int key_head = (int)(id - outer * a.cache.key_heads);
  const int workgroups = a.chunks / kRowWaves;
  const int chunk_id = (int)(outer % (uint32_t)workgroups) * kRowWaves + wave;
  const int tile_id = (int)(outer / (uint32_t)workgroups);
  const int s = wave_search(a.cache.sequences + 1, tile_id, lane, [&](int i) { return first_row_tile<kRows>(a, i); });
  if (s < 0 || s >= a.cache.sequences) return;
  const Chunk c = chunk_of(a, s);
  const int rows = c.tokens * a.group;
  const int row0 = (int)(tile_id - first_row_tile<kRows>(a, s)) * kRows;
  if (row0 >= rows) return;
  const int last_row = min(row0 + kRows, rows) - 1;
  const Sight first_sight = sight_of(a, c, (int)divide_by(row0, a.by_group)), last_sight = sight_of(a, c, (int)divide_by(last_row, a.by_group));
  const int capacity = capacity_of(a);
  const int low = first_sight.low, high = min(last_sight.high, capacity + 1);
  const int end_tile = (high + kTileKeys - 1) / kTileKeys;
  int run = run_of_tile(low / kTileKeys) + chunk_id;
  int t = max(run_first_tile(run), low / kTileKeys);
  if (t >= end_tile) return;

  State st;
  int token[1], head[1];
  bool live[1];
  {
    const int row = row0 + l16;
    live[0] = row < rows;
    const int i = (int)divide_by(live[0] ? row : row0, a.by_group);
    head[0] = (live[0] ? row : row0) - i * a.group;
    token[0] = c.first_token + i;
    st.sight[0] = live[0] ? sight_of(a, c, i) : Sight{0, 0};
  }
  st.load_q(a, key_head, token, head, live, l16, grp, nullptr);
  st.clear();
  TileLoader<SLABS> loader;
  loader.init(a, key_head, lane);
  typename State::ValuePlace place;
  place.init(l16, grp);
  const char* const none = reinterpret_cast<const char*>(kSpecialRows[0]);

  auto next_tile = [&](int tile) {
    const int r = run_of_tile(tile);
    return tile + 1 < run_first_tile(r + 1) ? tile + 1 : run_first_tile(r + a.chunks);
  };
  KeyPlace key_where[4], value_where[8];  // of the tile that is loaded next
  auto find_pages = [&](int tile) {
#pragma unroll
    for (int b = 0; b < 4; ++b) key_where[b].ask(a, s, tile * kTileKeys + 16 * b + l16);
#pragma unroll
    for (int j = 0; j < 8; ++j) value_where[j].ask(a, s, tile * kTileKeys + 8 * j + (lane >> 3));
  };
  auto load_values = [&](int tile, int stage) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* v = key_row_address(a, loader.values, loader.value_page, loader.value_row, value_where[j].entry, tile * kTileKeys + 8 * j + (lane >> 3), low, high);
#pragma unroll
      for (int slab = 0; slab < SLABS; ++slab) {
        const int vc = slab * 8 + loader.value_chunk;
        const char* from = vc * 8 < a.cache.width ? v + vc * 16 : none;
        __builtin_amdgcn_global_load_lds((global_ptr_t)from, (lds_ptr_t)(mine + stage * kTileBytes + slab * kSlabBytes + j * 1024), 16, 0, 0);
      }
    }
  };
  u32x4_t k[State::kSteps][4];
  auto load_keys = [&](int tile) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const char* from = key_row_address(a, loader.keys, loader.key_page, loader.key_row, key_where[b].entry, tile * kTileKeys + 16 * b + l16, low, high);
#pragma unroll
      for (int ks = 0; ks < State::kSteps; ++ks) {
        const int element = 32 * ks + 8 * grp;
        k[ks][b] = *reinterpret_cast<const u32x4_t*>(element < a.cache.width ? from + 2 * element : none);
      }
    }
  };

  int stage = 0;
  find_pages(t);
  load_values(t, 0);
  asm volatile("" ::: "memory");
  load_keys(t);
  if (next_tile(t) < end_tile) find_pages(next_tile(t));
  while (t < end_tile) {
    const int key0 = t * kTileKeys;
    const int next = next_tile(t);
    f32x4_t scores[4][1];
#pragma unroll
    for (int b = 0; b < 4; ++b) scores[b][0] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < State::kSteps; ++ks)
#pragma unroll
      for (int b = 0; b < 4; ++b) scores[b][0] = Half<DTYPE>::mfma(k[ks][b], st.q[ks][0], scores[b][0]);
    __builtin_amdgcn_s_waitcnt(kWaitAll0);  // its values are here too, and those of the tile before have been read
    asm volatile("" ::: "memory");
    const bool mixed = min(key0 + kTileKeys, high) > first_sight.high || max(key0, low) < last_sight.low;
    const value_bytes_t values = (value_bytes_t)(mine + stage * kTileBytes);
    bool special = false;
    if (mixed) {
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < 8 * SLABS; ++j) {
        const u32x4_t w = read_chunk(values + j * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= special_halves<DTYPE>(w[e]);
      }
      special = __any(any != 0);
    }
    if (next < end_tile) {
      load_values(next, stage ^ 1);
      asm volatile("" ::: "memory");
      load_keys(next);
      if (next_tile(next) < end_tile) find_pages(next_tile(next));
    }
    u32x4_t p[2][1];
    volatile float effect[4 * State::kBlocks];
    if (key0 + kTileKeys > first_sight.high || key0 < last_sight.low) st.mask(scores, key0, grp);
    st.weigh(a, scores, p);
    if (special) {
      st.find_special(values, place, p, key0, grp, effect);
#pragma unroll 1
      for (int j = 0; j < 8 * SLABS; ++j) take_out_special<DTYPE>(mine + stage * kTileBytes + j * 1024 + lane * 16);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    st.add_values(values, place, p);
    if (special) st.add_special(effect);
    const int this_run = run_of_tile(t);
    if (next >= end_tile || run_of_tile(next) != this_run) {
      const float sum = sum_over_groups(st.l[0]);
      if (live[0]) {
        const int64_t at = (int64_t)this_run * a.part_rows + (int64_t)token[0] * a.heads + key_head * a.group + head[0];
        if (grp == 0) a.part_max[at] = st.m[0], a.part_sum[at] = sum;
#pragma unroll
        for (int d = 0; d < State::kBlocks; ++d)
          if (16 * d + 4 * grp < a.cache.width) *reinterpret_cast<f32x4_t*>(a.part_out + at * a.cache.width + 16 * d + 4 * grp) = st.o[d][0];
      }
      st.clear();
    }
    t = next;
    stage ^= 1;
  }
}

// ---------------------------------------------------------------------------
// The runs of a row, left in memory, combined in ascending order: a workgroup a row, a thread an element.
// ---------------------------------------------------------------------------
constexpr int kJoinRuns = 64;

template <int DTYPE>
__global__ __launch_bounds__(kMaxWidth) void attention_join_kernel(const AttentionArgs a) {
  __shared__ float run_max[kJoinRuns], run_sum[kJoinRuns];
  const int tid = threadIdx.x, lane = tid & 63, width = a.cache.width;
  const int token = blockIdx.x / a.heads, head = blockIdx.x - token * a.heads;
  const int64_t row = (int64_t)token * a.heads + head;
  char* const out = a.out + (int64_t)token * a.out_token_stride + (int64_t)head * a.out_head_stride + 2 * tid;
  const int s = wave_search(a.cache.sequences + 1, token, lane, [&](int i) { return (int64_t)a.cache.starts[i]; });
  Sight sight = {0, 0};
  bool known = false;
  if (s >= 0 && s < a.cache.sequences) {
    const Chunk c = chunk_of(a, s);
    known = token - c.first_token < c.tokens;
    if (known) sight = sight_of(a, c, token - c.first_token);
  }
  if (!known && !a.zero_rest) return;
  float top = -INFINITY, sum = 0.f, o = 0.f;
  const int capacity = capacity_of(a);
  const int high = min(sight.high, capacity + 1);
  if (sight.low < high) {
    const int first = run_of_tile(sight.low / kTileKeys), last = run_of_tile((high - 1) / kTileKeys);
    for (int r0 = first; r0 <= last; r0 += kJoinRuns) {
      const int count = min(kJoinRuns, last + 1 - r0);
      __syncthreads();
      if (tid < count) run_max[tid] = a.part_max[(r0 + tid) * a.part_rows + row], run_sum[tid] = a.part_sum[(r0 + tid) * a.part_rows + row];
      __syncthreads();
      const float* from = a.part_out + ((int64_t)r0 * a.part_rows + row) * width + (tid < width ? tid : 0);
      const int64_t step = a.part_rows * width;
      constexpr int kAhead = 8;
      for (int r = 0; r < count; r += kAhead) {
        float v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i] = r + i < count ? from[(r + i) * step] : 0.f;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (r + i < count && run_sum[r + i] != 0.f) {
            const Join j = join_maxima(top, run_max[r + i]);
            sum = join_sums(sum, run_sum[r + i], j);
            o = join_sums(o, v[i], j);
          }
      }
    }
  }
  const bool sees = sight.high > sight.low;
  const float y = sees ? output_of(o, 1.f / sum) : 0.f;
  if (tid < width) *reinterpret_cast<uint16_t*>(out) = (uint16_t)Half<DTYPE>::pack(y, 0.f);
  if (a.lse && tid == 0) a.lse[row] = sees ? lse_of(top, sum) : -INFINITY;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct AttentionPlan {
  int rows;    // of a tile
  bool split;  // runs side by side
  int chunks, tiles;
};

static int run_limit(const rlk_paged_cache& c) {
  return run_of_tile(capacity_of(c) / kTileKeys) + 1;  // (with the position behind the table)
}

static AttentionPlan attention_plan(const rlk_paged_cache& c, int64_t tokens, int heads, int config) {
  AttentionPlan p;
  const int group = heads / c.key_heads;
  const int most = c.width > 128 ? 128 : 256;  // rows of the largest tile
  const int choice = config & 0xff;
  const int64_t each = (tokens + c.sequences - 1) / c.sequences * group;  // rows of a sequence and key head
  p.rows = choice == RLK_ATTENTION_CFG_ROWS16 ? 16 : choice == RLK_ATTENTION_CFG_ROWS64 ? 64 : choice == RLK_ATTENTION_CFG_ROWS256 ? most : each <= 16 ? 16 : each <= 64 ? 64 : most;
  p.tiles = (int)(tokens * group / p.rows) + c.sequences + 1;
  const int runs = run_limit(c);
  const int64_t side_by_side = (int64_t)(p.tiles - 1) * c.key_heads;
  const int cus = device_cu_count();
  p.split = p.rows == 16 || (choice != RLK_ATTENTION_CFG_AUTO ? (config & RLK_ATTENTION_CFG_SPLIT) != 0 : side_by_side < cus && runs > 1);
  p.chunks = 1;
  if (p.split) {
    const int64_t wanted = p.rows == 16 ? (16 * cus + side_by_side - 1) / side_by_side : (2 * cus + side_by_side - 1) / side_by_side;
    p.chunks = (int)(wanted < 1 ? 1 : wanted < runs ? wanted : runs);
    if (p.rows == 16) p.chunks = (p.chunks + kRowWaves - 1) / kRowWaves * kRowWaves;
  }
  return p;
}

size_t paged_attention_workspace_bytes(const rlk_paged_cache& c, int64_t tokens, int heads, int config) {
  if (tokens == 0 || c.sequences == 0 || heads == 0) return 0;
  if (!attention_plan(c, tokens, heads, config).split) return 0;
  return (size_t)run_limit(c) * tokens * heads * (c.width + 2) * sizeof(float);
}

template <int DTYPE, int SLABS, int RB, int WAVES, bool SPLIT>
static hipError_t attention_tiles_launch(const AttentionArgs& a, hipStream_t stream) {
  constexpr int kLds = 4 * SLABS * kSlabBytes + (RB == 1 ? 0 : WAVES * RB * SLABS * 2048) + 16;
  static PerDeviceOnce once;
  const auto kernel = attention_tile_kernel<DTYPE, SLABS, RB, WAVES, SPLIT>;
  const hipError_t err = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds, once);
  if (err != hipSuccess) return err;
  kernel<<<dim3((unsigned)(a.tiles * a.chunks * a.cache.key_heads)), WAVES * 64, kLds, stream>>>(a);
  return hipGetLastError();
}
template <int DTYPE, int SLABS, bool SPLIT>
static hipError_t attention_tiles_of(const AttentionArgs& a, int rows, hipStream_t stream) {
  if (rows == 64) return attention_tiles_launch<DTYPE, SLABS, 1, 4, SPLIT>(a, stream);
  return attention_tiles_launch<DTYPE, SLABS, SLABS <= 2 ? 2 : 1, 8, SPLIT>(a, stream);
}
template <int DTYPE, int SLABS>
static hipError_t attention_launch_of(const AttentionArgs& a, const AttentionPlan& p, hipStream_t stream) {
  hipError_t err;
  if (p.rows == 16) {
    constexpr int kLds = kRowWaves * 2 * SLABS * kSlabBytes;
    static PerDeviceOnce once;
    const auto kernel = attention_rows_kernel<DTYPE, SLABS>;
    err = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds, once);
    if (err != hipSuccess) return err;
    kernel<<<dim3((unsigned)(a.tiles * (a.chunks / kRowWaves) * a.cache.key_heads)), kRowWaves * 64, kLds, stream>>>(a);
    err = hipGetLastError();
  } else {
    err = p.split ? attention_tiles_of<DTYPE, SLABS, true>(a, p.rows, stream) : attention_tiles_of<DTYPE, SLABS, false>(a, p.rows, stream);
  }
  if (err != hipSuccess || !p.split) return err;
  attention_join_kernel<DTYPE><<<dim3((unsigned)a.part_rows), (a.cache.width + 63) / 64 * 64, 0, stream>>>(a);
  return hipGetLastError();
}
template <int DTYPE>
static hipError_t attention_launch_as(const AttentionArgs& a, const AttentionPlan& p, hipStream_t stream) {
  if (a.cache.width <= 64) return attention_launch_of<DTYPE, 1>(a, p, stream);
  if (a.cache.width <= 128) return attention_launch_of<DTYPE, 2>(a, p, stream);
  return attention_launch_of<DTYPE, 4>(a, p, stream);
}

hipError_t paged_attention_launch(const rlk_paged_cache& cache, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out,
                                  int64_t out_token_stride, int64_t out_head_stride, float* lse, int64_t tokens, int heads, float scale,
                                  bool causal, int window, bool zero_rest, int config, void* workspace, hipStream_t stream) {
  const AttentionPlan p = attention_plan(cache, tokens, heads, config);
  AttentionArgs a{};
  a.cache = cache;
  a.q = static_cast<const char*>(q);
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.q_token_stride = 2 * q_token_stride, a.q_head_stride = 2 * q_head_stride;
  a.out_token_stride = 2 * out_token_stride, a.out_head_stride = 2 * out_head_stride;
  a.part_rows = tokens * heads;
  if (p.split) {
    const int64_t parts = run_limit(cache) * a.part_rows;
    a.part_out = static_cast<float*>(workspace);
    a.part_max = a.part_out + parts * cache.width;
    a.part_sum = a.part_max + parts;
  }
  a.group = heads / cache.key_heads;
  a.by_page = page_divider((uint32_t)cache.page_size);
  a.by_group = page_divider((uint32_t)a.group);
  a.by_key_heads = page_divider((uint32_t)cache.key_heads);
  a.tokens = (int)tokens;
  a.heads = heads;
  a.causal = causal, a.window = window, a.zero_rest = zero_rest;
  a.tiles = p.tiles, a.chunks = p.chunks;
  a.scale = (float)((double)scale * 1.4426950408889634074);
  return cache.dtype == RLK_DTYPE_BF16 ? attention_launch_as<RLK_DTYPE_BF16>(a, p, stream) : attention_launch_as<RLK_DTYPE_FP16>(a, p, stream);
}

}  // namespace rlk
