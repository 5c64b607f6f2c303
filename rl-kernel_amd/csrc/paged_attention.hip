// Attention of new tokens over a paged cache for gfx950: single tokens, chunks of a prompt, whole prompts.
//
// Rows. A sequence's new tokens and the heads that share a key head are rows of one matrix, token by token, so that every key and
// value that is read serves all of them. A tile is a run of such rows of one sequence and one key head.
//
// Sums. Scores come transposed, S^T = K Q^T, 32 keys by 32 rows: the matrix instruction's result then has a row's scores in two
// lanes (and its statistics need one lane swap), and its registers, rounded to 16 bits, are the operands of O^T = V^T P^T as they
// stand: of 16 keys, slot 8 g + e of half-wave g holds key 8 (e / 4) + 4 g + e % 4, and the transposing LDS read brings the values in
// that order. Each of a row's two lanes sums the weights of its own keys; they meet at the end of a run.
//   tile of 64 keys:  m' = next(m, max s),  a = 2^(m - m'),  p = 2^(s - m'),  o = a o + round(p) V,  l = a l + sum p
// with s in units of log2(e) * scale. A run of tiles starts from nothing; runs are combined in ascending order:
//   M' = next(M, m),  O = 2^(m - M') o + 2^(M - M') O  (one fused step), L likewise;  out = O / L,  lse = ln 2 (M + log2 L)
// next(m, x) is x where x is more than 8 above m, else m: weights of up to 2^8 do no harm, and rows then hardly ever change their scale, which
// takes a product for every element (with the plain maximum nearly every tile of 32 rows did).
// Which keys form a tile and which tiles a run is a function of their positions, and keys that a row does not see leave its chain as it is (a
// factor of 1, a sum with 0). So a row's bits are the same in every kernel below, however its runs are spread over the chip.
// Statistics and outputs are fp32 throughout; weights are rounded to the inputs' 16 bits for the matrix units (half a step, 2^-9 of a
// weight in bf16, which averages out over the keys), not for their sum: its logarithm is an answer in 32 bits.
//
// What a row does not see may hold anything. Scores are replaced, not added to. Keys and values that no row of a tile sees are
// read as zeros. Where some rows see a value and others do not, a zero weight would not save them from infinities and NaN in
// it: such a tile is looked through before it is used, and if it holds any they are taken out of the product and added to the
// rows that see them.
//
// What bounds it. With few rows a tile's keys and values, HBM: 4 sequences of 131071 positions 415 us, 5.2 TB/s (a large copy reaches 4.9);
// 64 of up to 8192 222 us, 4.5 TB/s. With many the two products beside the vector work of the weights (32 matrix instructions of 32
// cycles against 235 vector instructions, 33 of them exponentials, for 32 rows and a tile: matrix units busy in 47 % of a CU's cycles, vector
// units in 56 %): prompts of up to 12000 tokens 2.3 ms, 0.95 PFLOP/s (2.1 ms on zeros, where the clock does not drop). A short call is a chain of latencies: 1025 positions of one token take 15 us, of
// which 3 to 4 go by until the first keys are there, 2 for each of the four tiles of a run and 4 for joining the runs.
#include "det_gemm_solo.h"
#include "paged.h"

namespace rlk {

constexpr int kTileKeys = 64;
constexpr int kSlabBytes = kTileKeys * 128;  // 64 keys x 64 elements
constexpr int kMaxWidth = 256;
constexpr int kMostKeys = 0x7fffff00;  // of a sequence: positions behind have no place (32-bit numbers of keys and tiles ahead must not overflow)

// Runs: their lengths grow with the position, so that a short context still has enough of them for the chip and a long
// one's partial results stay few (of 8 rows a part is 1/32 of the keys and values that a run of 256 reads, 1/256 of 2048). Tiles 0 ... 63 in fours, ... 255 in eights, ... 1023 in sixteens, then 32 at a time.
constexpr int kFirstRunTiles = 4;
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
  float* part_out;  // [run of those that a row sees][token][head][width]
  float* part_max;  // [run][token][head]
  float* part_sum;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // bytes
  int64_t part_rows;  // tokens * heads
  PageDivider by_page, by_group, by_key_heads, by_chunks;
  int tokens, heads, lse_heads, group, causal, window, zero_rest, longest_first, tiles, chunks;  // (lse_heads: of a row of lse)
  float scale;  // times log2(e)
};

// Operands: lane l holds row l % 32 of the first and column l % 32 of the second, slots 8 (l / 32) ... + 7 of 16. Result: register
// i of lane l is row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32.
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
template <int DTYPE>
struct Half;
template <>
struct Half<RLK_DTYPE_BF16> {
  static constexpr uint32_t kOnes = 0x3f803f80u, kExponent = 0x7f807f80u, kLowest = 0x00800080u, kFraction = 0x007f007fu;
  static constexpr uint32_t k128 = 0x4300u, k16384 = 0x4680u;
  static __device__ __forceinline__ f32x16_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Half<RLK_DTYPE_FP16> {
  static constexpr uint32_t kOnes = 0x3c003c00u, kExponent = 0x7c007c00u, kLowest = 0x04000400u, kFraction = 0x03ff03ffu;
  static constexpr uint32_t k128 = 0x5800u, k16384 = 0x7400u;
  static __device__ __forceinline__ f32x16_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
    typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
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

// The maximum that weights are taken from, once a value x has come up.
constexpr float kSlack = 8.f;
__device__ __forceinline__ float next_top(float top, float x) { return x > top + kSlack ? x : top; }

// NaN wins, and next_top() leaves the maximum as it is: such a row is NaN by its weights. (fmaxf, where it loses, takes an instruction more for
// each first operand: 31 a tile, not 19; a chunk of 1000 tokens over 65500 0.5 to 1.4 % longer.)
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }
// The largest value of a row over the two lanes that hold it (l and l + 32), and the sum.
__device__ __forceinline__ float max_over_halves(float v) {
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
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
// Chunks of 16 bytes change places within a row so that the reads are free of bank conflicts (counted: none in decode shapes, 0.02 cycles
// an LDS instruction in prompts): by three bits of the row for
// keys (lanes read one chunk of 32 rows, 16 of them at a time, two rows to 256 bytes of banks: bits 1 to 3 tell them apart whichever
// 16), by bits 1 and 2 for values (32 lanes read 64 bytes of four rows or 32 bytes of eight).
__device__ __forceinline__ int key_swizzle(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int value_swizzle(int row) { return 4 * ((row >> 1) & 1) + 2 * ((row >> 2) & 1); }

// One sequence's part of a launch.
struct Chunk {
  int sequence, first_token, tokens, length;
};

// What a row sees: keys [low, high).
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

// Positions that the page table has room for. A row that sees any behind them is NaN: without a window it sees the first of those, which is
// loaded as NaN, but a window may begin behind it, where nothing is loaded, so the end of a row asks for its last position.
__host__ __device__ __forceinline__ int capacity_of(const rlk_paged_cache& c) {
  const int64_t keys = (int64_t)c.table_columns * c.page_size;
  return keys < kMostKeys ? (int)keys : kMostKeys;
}
__device__ __forceinline__ int capacity_of(const AttentionArgs& a) { return capacity_of(a.cache); }

// Row tiles: the first one of every sequence (a workgroup knows it without a search, and of sequences of single tokens there are no others), then
// the others, of sequence s at floor(starts[s] * group / rows) and behind, at least as many as it needs.
template <int ROWS>
__device__ __forceinline__ int64_t other_row_tiles(const AttentionArgs& a, int s) {
  return (int64_t)clamp_to(a.cache.starts[s], 0, a.tokens) * a.group / ROWS;
}

// The running state of 32 rows of a wave. Lane l holds row l & 31; of the output, register i of block d is element
// 32 d + 8 (i / 4) + 4 (l / 32) + i % 4.
template <int DTYPE, int SLABS>
struct Rows {
  typedef Half<DTYPE> H;
  static constexpr int kBlocks = 2 * SLABS;  // of 32 elements
  static constexpr int kSteps = 4 * SLABS;   // of 16 elements
  f32x16_t o[kBlocks];
  float m;
  float l;  // the sum of the weights of this lane's keys
  Sight sight;

  __device__ __forceinline__ void clear_output() {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  }
  // Scores of a tile, s[b][i] of keys key0 + 32 b + 8 (i / 4) + 4 half + i % 4: those of keys that a row does not see go.
  __device__ __forceinline__ void mask(f32x16_t (&s)[2], int key0) {
    const int half = solo_lane() >> 5;
    const uint32_t range = sight.high > sight.low ? sight.high - sight.low : 0;
    const uint32_t from = (uint32_t)(key0 + 4 * half - sight.low);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = from + 32 * b + 8 * (i >> 2) + (i & 3) < range ? s[b][i] : -INFINITY;
  }
  // (see find_special)
  __device__ __forceinline__ void add_special(const volatile float* effect) {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] += effect[16 * d + i];
  }
};

// Scores to weights, in pieces that stand between matrix instructions: the maximum of eight scores each, the new maximum and what the
// state is scaled by, the weights of four scores each.
template <int DTYPE>
struct Weighing {
  static constexpr int kPieces = 13;
  float top[4], from, factor, sum[4];
  bool moved;
  template <int SLABS>
  __device__ __forceinline__ void piece(int n, const AttentionArgs& a, Rows<DTYPE, SLABS>& st, const f32x16_t (&s)[2], u32x4_t (&p)[4]) {
    if (n < 4) {
      const int b = n >> 1, first = 8 * (n & 1);
      float x = s[b][first];
#pragma unroll
      for (int i = 1; i < 8; ++i) x = larger(x, s[b][first + i]);
      asm volatile("" : "+v"(x));  // (here and below: computed in its piece, not where it is used)
      top[n] = x;
    } else if (n == 4) {
      const float before = st.m;
      st.m = next_top(before, max_over_halves(larger(larger(top[0], top[1]), larger(top[2], top[3]))) * a.scale);
      moved = st.m != before;
      factor = moved ? exp2_fast(before - st.m) : 1.f;
      from = st.m == -INFINITY ? 0.f : st.m;
    } else {
      const int j = n - 5, b = j >> 2, first = 4 * (j & 3);
      float x[4] = {s[b][first], s[b][first + 1], s[b][first + 2], s[b][first + 3]};
      asm volatile("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));  // (nor before its piece)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = exp2_fast(__builtin_fmaf(x[i], a.scale, -from));
      uint32_t pair = Half<DTYPE>::pack(x[0], x[1]), other = Half<DTYPE>::pack(x[2], x[3]);
      float four = (x[0] + x[1]) + (x[2] + x[3]);
      asm volatile("" : "+v"(pair), "+v"(other), "+v"(four));
      p[j >> 1][2 * (j & 1)] = pair;
      p[j >> 1][2 * (j & 1) + 1] = other;
      sum[j >> 1] = (j & 1) ? sum[j >> 1] + four : four;
      if (n == kPieces - 1) st.l = __builtin_fmaf(st.l, factor, (sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
  }
};

// A run joins those before it: factors for both, and the new maximum.
struct Join {
  float kept, added;
};
__device__ __forceinline__ Join join_maxima(float& all, float run) {
  const float top = next_top(all, run);
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

// One of the two caches, of a key head; distances in bytes.
struct CacheSide {
  const char* base;
  uint32_t page, row;
  __device__ __forceinline__ void init(const void* cache, int64_t head, int64_t page_stride, int64_t row_stride) {
    base = static_cast<const char*>(cache) + 2 * head;
    page = (uint32_t)(2 * page_stride), row = (uint32_t)(2 * row_stride);
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
struct KeyRow {
  uint32_t page, row;
  const char* special;  // instead: zeros where the tile does not need the key, NaN where its page is missing
  __device__ __forceinline__ void find(const AttentionArgs& a, int entry, int key, int low, int high) {
    const int column = (int)divide_by((uint32_t)key, a.by_page);
    const bool there = (uint32_t)entry < (uint32_t)a.cache.pages && column < a.cache.table_columns;
    const bool wanted = key >= low && key < high;
    special = wanted && there ? nullptr : reinterpret_cast<const char*>(kSpecialRows[wanted]);
    page = wanted && there ? entry : 0;
    row = key - column * a.cache.page_size;
  }
  __device__ __forceinline__ const char* in(const CacheSide& c) const {
    const char* at = c.base + (uint64_t)page * c.page + (uint64_t)row * c.row;
    return special != nullptr ? special : at;
  }
};

// 16 bytes of each lane straight into LDS, at a distance from a wave's base; zeros for kSoloOutside.
__device__ __forceinline__ void load_block(char* base, uint32_t offset, char* to) {
  const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(base, 0, kSoloRange, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (lds_ptr_t)to, 16, offset, 0, 0, 0);
}
// Eight keys of one page straight into LDS, at the address of the first (odd where the page is missing), each lane 16 bytes of every slab
// of its key's row: `offset` from there where all of them are needed, else what a lane has to work out (from its number as if it had just
// been read, so that nothing is kept for that through the turns that do not need it). SWIZZLE: of the image.
template <int SLABS, class Swizzle>
__device__ __forceinline__ void load_group(uint32_t low_word, uint32_t high_word, const uint32_t (&offset)[SLABS], bool whole, int first_key, int low,
                                           int high, uint32_t row_bytes, int width, Swizzle swizzle, char* to) {
  uint32_t at[SLABS];
#pragma unroll
  for (int slab = 0; slab < SLABS; ++slab) at[slab] = offset[slab];
  if ((low_word & 1) != 0 || !whole) {
    const int lane = solo_lane(), key = first_key + (lane >> 3), chunk = (lane & 7) ^ swizzle(first_key + (lane >> 3));
#pragma unroll
    for (int slab = 0; slab < SLABS; ++slab) {
      at[slab] = ((low_word & 1) == 0 ? (lane >> 3) * row_bytes : 0) + chunk * 16 + slab * 128;
      if (key < low || key >= high || (slab * 8 + chunk) * 8 >= width) at[slab] = kSoloOutside;
    }
  }
#pragma unroll
  for (int slab = 0; slab < SLABS; ++slab) load_block(reinterpret_cast<char*>((uint64_t)high_word << 32 | (low_word & ~1u)), at[slab], to + slab * kSlabBytes);
}
// The same for keys of any pages.
template <int SLABS>
__device__ __forceinline__ void load_rows(const AttentionArgs& a, const CacheSide& side, const KeyPlace& where, int chunk, int key, int low, int high,
                                          char* to) {
  const char* const none = reinterpret_cast<const char*>(kSpecialRows[0]);
  KeyRow row;
  row.find(a, where.entry, key, low, high);
  const char* const from = row.in(side) + chunk * 16;
#pragma unroll
  for (int slab = 0; slab < SLABS; ++slab) {
    const char* const at = (slab * 8 + chunk) * 8 < a.cache.width ? from + slab * 128 : none;
    __builtin_amdgcn_global_load_lds((global_ptr_t)at, (lds_ptr_t)(to + slab * kSlabBytes), 16, 0, 0);
  }
}

// A tile with infinities or NaN among the values that some rows see and others do not. They have left the tile in LDS (take_out_special), and
// what they make of an element is added to it behind the product: an infinity, or NaN where both come together, from NaN, or from
// an infinity with a weight of 0. One more product counts them: 1 for inf, 128 for -inf, 16384 for NaN, 64 at most of each. The values are
// read from the cache again, the results wait in memory, and nothing here is unrolled: this is rare, and in registers it would cost the
// ordinary tiles theirs.
template <int DTYPE, class State>
__device__ __forceinline__ void find_special(const AttentionArgs& a, const State& st, const CacheSide& values, int sequence, const u32x4_t (&p)[4],
                                             int key0, int low, int high, int lane, volatile float* effect) {
  typedef Half<DTYPE> H;
  const uint32_t one = H::kOnes & 0xffffu;
  const uint32_t range = st.sight.high > st.sight.low ? st.sight.high - st.sight.low : 0;
#pragma unroll 1
  for (int d = 0; d < State::kBlocks; ++d) {
    f32x16_t count;
#pragma unroll
    for (int i = 0; i < 16; ++i) count[i] = 0.f;
#pragma unroll 1
    for (int f = 0; f < 4; ++f) {
      u32x4_t kinds, any, seen, lost;  // of the values; 1 where a row sees a key with a weight, and without one
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int first = key0 + 16 * f + 8 * (e >> 1) + 4 * (lane >> 5) + 2 * (e & 1);
        uint32_t w = 0;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          KeyPlace where;
          where.ask(a, sequence, first + i);
          KeyRow row;
          row.find(a, where.entry, first + i, low, high);
          const int element = 32 * d + (lane & 31);
          if (element < a.cache.width) w |= (uint32_t)reinterpret_cast<const uint16_t*>(row.in(values))[element] << (16 * i);
        }
        const uint32_t from = (uint32_t)(first - st.sight.low);
        const uint32_t sees = (from < range ? 0x8000u : 0u) | (from + 1 < range ? 0x80000000u : 0u);
        const uint32_t bits = f == 0 ? p[0][e] : f == 1 ? p[1][e] : f == 2 ? p[2][e] : p[3][e];
        const uint32_t weighs = ((bits & 0x7fff7fffu) + 0x7fff7fffu) & sees;
        seen[e] = (weighs >> 15) * one;
        lost[e] = ((sees ^ weighs) >> 15) * one;
        const uint32_t special = special_halves<DTYPE>(w);
        const uint32_t none = special & ((w & H::kFraction) + 0x7fff7fffu);
        kinds[e] = ((special & ~none & ~w) >> 15) * one | ((special & ~none & w) >> 15) * H::k128 | (none >> 15) * H::k16384;
        any[e] = (special >> 15) * H::k16384;
      }
      count = H::mfma(kinds, seen, count);
      count = H::mfma(any, lost, count);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t n = (uint32_t)count[i];
      const float up = (n & 127) != 0 ? INFINITY : 0.f, down = (n & (127 << 7)) != 0 ? -INFINITY : 0.f;
      effect[16 * d + i] = n >= 16384 ? NAN : up + down;
    }
  }
}
// Zeros in the place of a chunk's infinities and NaN; whether there were any.
template <int DTYPE>
__device__ __forceinline__ bool take_out_special(char* at) {
  typedef __attribute__((address_space(3))) u32x4_t* chunk_ptr_t;
  u32x4_t w = *(chunk_ptr_t)at;
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t special = special_halves<DTYPE>(w[e]);
    w[e] &= ~((special >> 15) * 0xffffu);
    any |= special;
  }
  if (any != 0) *(chunk_ptr_t)at = w;
  return any != 0;
}

// ---------------------------------------------------------------------------
// WAVES waves of 32 rows each (2, 4 or 8) share the keys and values of their tile through LDS, two tiles of each deep, one barrier a tile. SPLIT:
// a workgroup takes some of the runs and leaves the parts in memory. GROUPED: eight keys that a load instruction brings lie in one page
// (page sizes that 8 divides), so that a wave-uniform base and constant lane offsets address them, a buffer load's range makes
// zeros of the keys that a tile does not need, and the compiler counts LDS reads one by one (beside a direct load with lane
// addresses, which it takes for one that might have gone to LDS, it waits for all of them at every step: prompts of 12000 tokens
// 2.9 ms). Other page sizes get tiles of 128 rows whatever their number, so that there are fewer kernels to build.
//
// In turn i a wave multiplies its queries with tile i's keys, and then tile i - 1's weights with its values; between these
// products stands, piece by piece, what turns tile i's scores into weights, because a wave's vector instructions run beside its own
// matrix instructions (and exponentials, 16 cycles each, are a third of the time of both products) but two waves a SIMD are too
// few to fill one with the other's (half a turn apart they took as long as side by side). Half of a tile's weights beside the next
// tile's first product took longer (2.38 ms for 2.35, with one wave a SIMD 1.66 for 1.57), as did more loads ahead: four stages and waits
// for one tile of three gave the same times with 64 rows and 1.60 ms for 1.55 with 128. Tile i + 1's keys and tile i's values are asked for at the start of turn i and have landed at
// its end; the places they go to were last read in turn i - 1.
// ---------------------------------------------------------------------------
template <int DTYPE, int SLABS, int WAVES, bool SPLIT, bool GROUPED>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(WAVES == 8 ? 2 : 1, WAVES == 8 ? 2 : 1))) void attention_tile_kernel(
    const AttentionArgs a) {
  typedef Rows<DTYPE, SLABS> State;
  typedef Half<DTYPE> H;
  constexpr int kRows = 32 * WAVES;
  constexpr bool kKeepQ = SLABS > 2 || WAVES <= 2;  // queries stay in registers; else in LDS (with four waves both took as long)
  constexpr int kGroups = 8 / WAVES;  // groups of 8 keys that a wave loads
  constexpr int kSpan = 64 / kGroups;  // tiles whose addresses the lanes of a wave have
  constexpr int kTileBytes = SLABS * kSlabBytes;
  constexpr int kShelfBytes = kKeepQ ? 0 : SLABS * 4096;  // of a wave
  // [2][keys, values], then the queries, wave by wave, then special_tile. Nothing lies in front of it: 16-byte reads that
  // start on 8 bytes took 62 cycles each instead of 8.
  extern __shared__ __align__(16) char lds[];
  int* const special_tile = reinterpret_cast<int*>(lds + 4 * kTileBytes + WAVES * kShelfBytes);  // [2]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;

  // Heads change fastest, so that an XCD's workgroups read few of them; of a sequence's other tiles those with the most keys come first.
  const uint32_t id = blockIdx.x;
  const uint32_t outer = divide_by(id, a.by_key_heads);
  const int key_head = (int)(id - outer * a.cache.key_heads);
  const int tile_id = (int)(SPLIT ? divide_by(outer, a.by_chunks) : outer);
  const int chunk_id = SPLIT ? (int)outer - tile_id * a.chunks : 0;
  int s = tile_id, row0 = 0;
  if (tile_id < a.cache.sequences && a.longest_first) {  // of 64 sequences: this one's place is its length's
    const int first = tile_id & ~63, count = min(64, a.cache.sequences - first);
    const int mine = lane < count ? a.cache.lengths[first + lane] : 0;
    int rank = 0;
    for (int i = 0; i < count; ++i) {
      const int other = __builtin_amdgcn_readlane(mine, i);
      rank += other > mine || (other == mine && i < lane);
    }
    s = first + __ffsll(__ballot(lane < count && rank == (tile_id & 63))) - 1;
  }
  if (tile_id >= a.cache.sequences) {
    const int others = a.tiles - a.cache.sequences, i = tile_id - a.cache.sequences;
    const int other = i + 1 < others ? others - 2 - i : others - 1;  // (that one is hardly ever needed)
    s = wave_search(a.cache.sequences + 1, other, lane, [&](int i) { return other_row_tiles<kRows>(a, i); });
    if (s < 0) return;
    const int first = (int)other_row_tiles<kRows>(a, s);
    if (other < first) return;  // (starts that do not ascend: what the search finds need not lie in front; row0 and tails below would be negative)
    if (s >= a.cache.sequences) {  // behind the last sequence
      if (!SPLIT && a.zero_rest) {
        const int before = clamp_to(a.cache.starts[0], 0, a.tokens), behind = clamp_to(a.cache.starts[s], before, a.tokens);
        const int tails = others - first;
        const int each = a.cache.width / 8;
        for (int n = other - first; n < before + a.tokens - behind; n += tails) {
          const int t = n < before ? n : behind + n - before;
          for (int i = tid; i < a.group * each; i += WAVES * 64) {
            const int head = key_head * a.group + i / each;
            *reinterpret_cast<u32x4_t*>(a.out + t * a.out_token_stride + head * a.out_head_stride + (i % each) * 16) = u32x4_t{0, 0, 0, 0};
            if (a.lse && i % each == 0) a.lse[(int64_t)t * a.lse_heads + head] = -INFINITY;
          }
        }
      }
      return;
    }
    row0 = (1 + other - first) * kRows;
  }
  const Chunk c = chunk_of(a, s);
  const int rows = c.tokens * a.group;
  if (row0 >= rows) return;

  // What this workgroup's and this wave's rows see.
  const int last_row = min(row0 + kRows, rows) - 1;
  const Sight first_sight = sight_of(a, c, (int)divide_by(row0, a.by_group)), last_sight = sight_of(a, c, (int)divide_by(last_row, a.by_group));
  const int capacity = capacity_of(a);
  const int low = first_sight.low, high = min(last_sight.high, capacity + 1);
  const int wave_row0 = row0 + wave * 32, wave_row1 = min(wave_row0 + 32, rows) - 1;
  const bool wave_live = wave_row0 < rows;
  const Sight wave_first = sight_of(a, c, (int)divide_by(wave_live ? wave_row0 : row0, a.by_group));
  const Sight wave_last = sight_of(a, c, (int)divide_by(wave_live ? wave_row1 : row0, a.by_group));

  struct RowPlace {
    int token, head;
    bool live;
  };
  auto row_place = [&]() __attribute__((always_inline)) {
    const int row = wave_row0 + (lane & 31);
    RowPlace r;
    r.live = row < rows;
    const int t = (int)divide_by(r.live ? row : row0, a.by_group);
    r.head = key_head * a.group + (r.live ? row : row0) - t * a.group;
    r.token = c.first_token + t;
    return r;
  };
  State st;
  char* const shelf = lds + 4 * kTileBytes + wave * kShelfBytes;
  u32x4_t kept_q[kKeepQ ? State::kSteps : 1];
  {
    const RowPlace r = row_place();
    st.sight = r.live ? sight_of(a, c, r.token - c.first_token) : Sight{0, 0};
    const char* const row = a.q + (int64_t)r.token * a.q_token_stride + (int64_t)r.head * a.q_head_stride;
#pragma unroll
    for (int ks = 0; ks < State::kSteps; ++ks) {
      const int element = 16 * ks + 8 * half;
      const bool wanted = r.live && element < a.cache.width;
      u32x4_t v = *reinterpret_cast<const u32x4_t*>(row + (wanted ? 2 * element : 0));
      if (!wanted) v = u32x4_t{0, 0, 0, 0};
      if (kKeepQ)
        kept_q[kKeepQ ? ks : 0] = v;
      else
        *reinterpret_cast<u32x4_t*>(shelf + (ks >> 2) * 4096 + (lane & 31) * 128 + (((2 * (ks & 3) + half) ^ key_swizzle(lane)) << 4)) = v;
    }
  }
  if (tid < 2) special_tile[tid] = 0;

  CacheSide key_side, value_side;
  key_side.init(a.cache.keys, key_head * a.cache.key_head_stride, a.cache.key_page_stride, a.cache.key_row_stride);
  value_side.init(a.cache.values, key_head * a.cache.value_head_stride, a.cache.value_page_stride, a.cache.value_row_stride);
  // Of a loading lane.
  const int key_chunk = (lane & 7) ^ key_swizzle(8 * (wave & 1) + (lane >> 3));  // (a wave's groups of eight keys are all even or all odd)
  const int value_chunk = (lane & 7) ^ value_swizzle(lane >> 3);
  // This lane's places in the images: of 16 elements of its key (or query) for every step of a slab, of its elements' values for even
  // and odd blocks of 32.
  int key_at[4], value_at[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) key_at[i] = (lane & 31) * 128 + (((2 * i + half) ^ key_swizzle(lane)) << 4);
  {
    const int row = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) value_at[i] = row * 128 + (((4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle(row)) << 4) + (lane & 1) * 8;
  }

  // This workgroup's tiles: those of runs that start in its part.
  int t = low / kTileKeys, end_tile = (high + kTileKeys - 1) / kTileKeys;
  if (SPLIT) {
    // The first run that starts at a part's border or later: even lanes for this part, odd ones for the next (in one go, without branches).
    const int first = t, count = end_tile - first, each = (int)divide_by((uint32_t)max(count, 0), a.by_chunks);
    const int part = chunk_id + (lane & 1), tile = first + each * part + min(part, max(count, 0) - each * a.chunks);
    const int run = run_of_tile(tile), run_start = run_first_tile(run), next_start = run_first_tile(run + 1);
    const int border = tile <= first ? first : run_start >= tile ? tile : next_start;
    t = __builtin_amdgcn_readlane(border, 0);
    end_tile = min(end_tile, __builtin_amdgcn_readlane(border, 1));
  }
  if (t >= end_tile && SPLIT) return;
  auto keys_of = [&](int stage) __attribute__((always_inline)) { return lds + stage * 2 * kTileBytes; };
  auto values_of = [&](int stage) __attribute__((always_inline)) { return lds + stage * 2 * kTileBytes + kTileBytes; };

  // GROUPED: lane kGroups i + j has the addresses of group j of tile from + i, odd ones where the page is missing, of keys and of values; the
  // next ones' table entries are on their way. They change hands at the start of a turn, when nothing is in flight.
  uint32_t key_low = 0, key_high = 0, value_low = 0, value_high = 0, later_low = 0, later_high = 0;
  int key_from = t, value_from = t;
  KeyPlace lane_where;
  auto key_of_lane = [&](int tile) __attribute__((always_inline)) { return (tile + lane / kGroups) * kTileKeys + (wave + (lane % kGroups) * WAVES) * 8; };
  auto find_addresses = [&](int tile) __attribute__((always_inline)) {
    const int key = key_of_lane(tile), column = (int)divide_by((uint32_t)key, a.by_page);
    const bool there = (uint32_t)lane_where.entry < (uint32_t)a.cache.pages && column < a.cache.table_columns;
    const uint64_t page = (uint32_t)lane_where.entry, row = (uint32_t)(key - column * a.cache.page_size);
    const uint64_t missing = reinterpret_cast<uint64_t>(kSpecialRows[1]) + 1;
    const uint64_t k = there ? reinterpret_cast<uint64_t>(key_side.base) + page * key_side.page + row * key_side.row : missing;
    const uint64_t v = there ? reinterpret_cast<uint64_t>(value_side.base) + page * value_side.page + row * value_side.row : missing;
    key_low = (uint32_t)k, key_high = (uint32_t)(k >> 32);
    later_low = (uint32_t)v, later_high = (uint32_t)(v >> 32);
    key_from = tile;
    lane_where.ask(a, s, key_of_lane(tile + kSpan));
  };
  // Else: the table's entries of the tile whose keys have been asked for, and of the one behind.
  KeyPlace here[kGroups], ahead[kGroups];
  auto find_entries = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      here[j] = ahead[j];
      ahead[j].ask(a, s, tile * kTileKeys + (wave + j * WAVES) * 8 + (lane >> 3));
    }
  };
  uint32_t key_offset[SLABS], value_offset[SLABS];
#pragma unroll
  for (int slab = 0; slab < SLABS; ++slab) {
    key_offset[slab] = (slab * 8 + key_chunk) * 8 < a.cache.width ? (lane >> 3) * key_side.row + key_chunk * 16 + slab * 128 : kSoloOutside;
    value_offset[slab] = (slab * 8 + value_chunk) * 8 < a.cache.width ? (lane >> 3) * value_side.row + value_chunk * 16 + slab * 128 : kSoloOutside;
  }
  const int whole_from = (low + kTileKeys - 1) / kTileKeys, whole_to = high / kTileKeys;  // tiles all of whose keys are needed
  auto load_keys = [&](const KeyPlace (&where)[kGroups], int tile, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int i = (tile - key_from) * kGroups + j, first_key = tile * kTileKeys + (wave + j * WAVES) * 8;
      char* const to = keys_of(stage) + (wave + j * WAVES) * 1024;
      if (GROUPED)
        load_group<SLABS>(__builtin_amdgcn_readlane(key_low, i), __builtin_amdgcn_readlane(key_high, i), key_offset,
                          tile >= whole_from && tile < whole_to, first_key, low, high, key_side.row, a.cache.width, key_swizzle, to);
      else
        load_rows<SLABS>(a, key_side, where[j], (lane & 7) ^ key_swizzle(first_key + (lane >> 3)), first_key + (lane >> 3), low, high, to);
    }
  };
  auto load_values = [&](int tile, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const int i = (tile - value_from) * kGroups + j, first_key = tile * kTileKeys + (wave + j * WAVES) * 8;
      char* const to = values_of(stage) + (wave + j * WAVES) * 1024;
      if (GROUPED)
        load_group<SLABS>(__builtin_amdgcn_readlane(value_low, i), __builtin_amdgcn_readlane(value_high, i), value_offset,
                          tile >= whole_from && tile < whole_to, first_key, low, high, value_side.row, a.cache.width, value_swizzle, to);
      else
        load_rows<SLABS>(a, value_side, here[j], (lane & 7) ^ value_swizzle(lane >> 3), first_key + (lane >> 3), low, high, to);
    }
  };
  // What turn `tile` asks for: its values, the next one's keys.
  auto ask_for = [&](int tile, int stage) __attribute__((always_inline)) {
    if (GROUPED) {
      if (tile - value_from >= kSpan) {
        value_low = later_low, value_high = later_high;
        value_from = tile;
      }
      if (tile + 1 - key_from >= kSpan) find_addresses(tile + 1);
    }
    load_values(tile, stage);
    if (tile + 1 < end_tile) load_keys(ahead, tile + 1, stage ^ 1);
    if (!GROUPED) find_entries(tile + 2 < end_tile ? tile + 2 : tile);
  };
  // Some rows of the workgroup see a key of the tile that others do not.
  const int mixed_from = first_sight.high < high ? first_sight.high / kTileKeys : 0x7fffffff;
  const int mixed_to = low < last_sight.low ? (last_sight.low + kTileKeys - 1) / kTileKeys : 0;
  auto mixed = [&](int tile) __attribute__((always_inline)) { return tile >= mixed_from || tile < mixed_to; };
  // The end of a turn: what I asked for has landed. Values that not everybody sees are looked through.
  auto landed = [&](int tile, int stage, bool plain) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(kWaitAll0);
    asm volatile("" ::: "memory");
    if (!plain && mixed(tile)) {
      bool special = false;
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
#pragma unroll
        for (int slab = 0; slab < SLABS; ++slab) special |= take_out_special<DTYPE>(values_of(stage) + slab * kSlabBytes + (wave + j * WAVES) * 1024 + lane * 16);
      if (special) special_tile[stage] = tile + 1;
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    }
    wg_barrier();
  };

  // Runs combined so far.
  f32x16_t all_o[SPLIT ? 1 : State::kBlocks];
  float all_m = -INFINITY, all_l = 0.f;
#pragma unroll
  for (int d = 0; d < (SPLIT ? 1 : State::kBlocks); ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) all_o[d][i] = 0.f;
  // A run ends, with the maximum and this lane's sum.
  auto end_run = [&](int run, float its_m, float its_l) __attribute__((always_inline)) {
    const float sum = sum_over_halves(its_l);
    if (SPLIT) {
      const RowPlace r = row_place();
      const int its_first = run_of_tile(st.sight.low / kTileKeys), its_last = run_of_tile((min(st.sight.high, capacity + 1) - 1) / kTileKeys);
      if (r.live && run >= its_first && run <= its_last) {
        const int64_t at = (int64_t)(run - its_first) * a.part_rows + (int64_t)r.token * a.heads + r.head;
        if (half == 0) a.part_max[at] = its_m, a.part_sum[at] = sum;
#pragma unroll
        for (int d = 0; d < State::kBlocks; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int element = 32 * d + 2 * i + 4 * half;
            if (element < a.cache.width)
              *reinterpret_cast<f32x4_t*>(a.part_out + at * a.cache.width + element) = f32x4_t{st.o[d][i], st.o[d][i + 1], st.o[d][i + 2], st.o[d][i + 3]};
          }
      }
    } else if (sum != 0.f) {  // (NaN is a sum too)
      const Join j = join_maxima(all_m, its_m);
      all_l = join_sums(all_l, sum, j);
      if (__any(j.kept != 1.f)) {
#pragma unroll
        for (int d = 0; d < State::kBlocks; ++d) all_o[SPLIT ? 0 : d] *= j.kept;
      }
#pragma unroll
      for (int d = 0; d < State::kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) all_o[SPLIT ? 0 : d][i] = __builtin_fmaf(st.o[d][i], j.added, all_o[SPLIT ? 0 : d][i]);
    }
    st.clear_output();
  };

  if (t < end_tile) {
    if (GROUPED) {
      lane_where.ask(a, s, key_of_lane(t));
      find_addresses(t);
      value_low = later_low, value_high = later_high;
    } else {
      find_entries(t);
      find_entries(t + 1 < end_tile ? t + 1 : t);
    }
    load_keys(here, t, 0);
    // The first turn multiplies weights of 0 with what lies where its values would: it must be numbers.
    for (int i = tid * 16; i < kTileBytes; i += WAVES * 64 * 16) *reinterpret_cast<u32x4_t*>(values_of(1) + i) = u32x4_t{0, 0, 0, 0};
    __builtin_amdgcn_s_waitcnt(kWaitAll0);
    wg_barrier();
  }
  int stage = 0, before = -1;  // the tile whose weights wait for its values
  if (!wave_live) {  // loads its share, no more
    for (; t < end_tile; ++t, stage ^= 1) {
      ask_for(t, stage);
      landed(t, stage, false);
    }
    return;
  }
  const int masked_from = wave_first.high / kTileKeys, masked_to = (wave_last.low + kTileKeys - 1) / kTileKeys;
  int run_end = t < end_tile ? run_first_tile(run_of_tile(t) + 1) : 0;
  st.clear_output();
  st.m = -INFINITY;
  st.l = 0.f;
  u32x4_t p[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) p[f] = u32x4_t{0, 0, 0, 0};
  // The products read their fragments a few ahead of their use.
  constexpr int kAhead = 4, kValueFragments = 4 * State::kBlocks, kKeyFragments = 2 * State::kSteps;
  auto value_fragment = [&](int n, int its_stage) __attribute__((always_inline)) {  // 16 keys n / kBlocks, block n % kBlocks
    const int d = n % State::kBlocks, f = n / State::kBlocks;
    const value_bytes_t at = (value_bytes_t)values_of(its_stage) + value_at[d & 1] + (d >> 1) * kSlabBytes + f * 2048;
    const u32x2_t x = read_values_transposed(at), y = read_values_transposed(at + 1024);
    return u32x4_t{x.x, x.y, y.x, y.y};
  };
  auto key_fragment = [&](int n) __attribute__((always_inline)) {  // step n / 2, 32 keys n % 2
    return read_chunk((value_bytes_t)keys_of(stage) + key_at[(n >> 1) & 3] + (n >> 3) * kSlabBytes + (n & 1) * 4096);
  };
  auto query_fragment = [&](int ks) __attribute__((always_inline)) { return kKeepQ ? kept_q[kKeepQ ? ks : 0] : read_chunk((value_bytes_t)shelf + key_at[ks & 3] + (ks >> 2) * 4096); };

  // One turn. PLAIN: every row sees every key of the tile, and the last tile's values hold nothing special and do not end a run.
  auto turn = [&](auto plain, float& its_m, float& its_l) __attribute__((always_inline)) {
    constexpr bool PLAIN = decltype(plain)::value != 0;
    ask_for(t, stage);
    f32x16_t scores[2];
    u32x4_t ring[kAhead], q[2];
    q[0] = query_fragment(0);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = key_fragment(n);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) scores[b][i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kKeyFragments; ++n) {
      const int ks = n >> 1, b = n & 1, next = n + kAhead;
      if (b == 0 && ks + 1 < State::kSteps) q[(ks + 1) & 1] = query_fragment(ks + 1);
      scores[b] = H::mfma(ring[n % kAhead], q[ks & 1], scores[b]);
      if (next < kKeyFragments)
        ring[n % kAhead] = key_fragment(next);
      else
        ring[n % kAhead] = value_fragment(next - kKeyFragments, stage ^ 1);
      __builtin_amdgcn_sched_barrier(0);  // (or the reads move back to their use)
    }
    if (!PLAIN) {
      if (t >= masked_from || t < masked_to) st.mask(scores, t * kTileKeys);
      // A run that has ended waits with its statistics for its last values.
      its_m = st.m, its_l = st.l;
      if (t == run_end) st.m = -INFINITY, st.l = 0.f;
    }
    Weighing<DTYPE> weighing;
    u32x4_t next_p[4];
#pragma unroll
    for (int n = 0; n < kValueFragments; ++n) {
      const int d = n % State::kBlocks, f = n / State::kBlocks, next = n + kAhead;
      st.o[d] = H::mfma(ring[n % kAhead], p[f], st.o[d]);
      if (next < kValueFragments) ring[n % kAhead] = value_fragment(next, stage ^ 1);
#pragma unroll
      for (int j = 0; j < Weighing<DTYPE>::kPieces; ++j)
        if (j * kValueFragments / Weighing<DTYPE>::kPieces == n) weighing.template piece<SLABS>(j, a, st, scores, next_p);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) p[f] = next_p[f];
    landed(t, stage, PLAIN);
    before = t, ++t, stage ^= 1;
    return weighing.factor;
  };
  while (t < end_tile) {
    // A turn with everything that may come up, then plain ones as long as nothing does: what changes the outputs besides the
    // products stands outside of their loop, where it would have them copied from register to register in every turn.
    const bool run_starts = t == run_end, first_turn = before < 0;
    float its_m, its_l;
    volatile float effect[16 * State::kBlocks];  // (in memory, see find_special)
    const bool special = before >= 0 && mixed(before) && special_tile[stage ^ 1] == before + 1;
    if (special) find_special<DTYPE, State>(a, st, value_side, s, p, before * kTileKeys, low, high, lane, effect);
    float factor = turn(IntTag<0>{}, its_m, its_l);
    if (special) st.add_special(effect);
    if (run_starts) {
      const int run = run_of_tile(before);
      end_run(run - 1, its_m, its_l);
      run_end = run_first_tile(run + 1);
    }
    if (run_starts || first_turn) factor = 1.f;  // (nothing is there to be scaled)
    const int plain_to = min(min(run_end, end_tile), min(masked_from, mixed_from)), plain_from = max(masked_to, mixed_to + 1);
    while (t >= plain_from && t < plain_to && !__any(factor != 1.f)) factor = turn(IntTag<1>{}, its_m, its_l);
    if (__any(factor != 1.f)) {
#pragma unroll
      for (int d = 0; d < State::kBlocks; ++d) st.o[d] *= factor;
    }
  }
  if (before >= 0) {  // the last tile's values
    volatile float effect[16 * State::kBlocks];
    const bool special = mixed(before) && special_tile[stage ^ 1] == before + 1;
    if (special) find_special<DTYPE, State>(a, st, value_side, s, p, before * kTileKeys, low, high, lane, effect);
#pragma unroll
    for (int n = 0; n < kValueFragments; ++n) {
      const int d = n % State::kBlocks, f = n / State::kBlocks;
      st.o[d] = H::mfma(value_fragment(n, stage ^ 1), p[f], st.o[d]);
    }
    if (special) st.add_special(effect);
    end_run(run_of_tile(before), st.m, st.l);
  }
  if (SPLIT) return;
  const RowPlace r = row_place();
  if (!r.live) return;
  const bool any = st.sight.high > st.sight.low, behind = st.sight.high > capacity;
  const float reciprocal = behind ? NAN : any ? 1.f / all_l : 0.f;
  char* const to = a.out + (int64_t)r.token * a.out_token_stride + (int64_t)r.head * a.out_head_stride;
#pragma unroll
  for (int d = 0; d < State::kBlocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const f32x16_t& o = all_o[SPLIT ? 0 : d];
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = any ? output_of(o[i + e], reciprocal) : 0.f;
      const int element = 32 * d + 2 * i + 4 * half;
      if (element < a.cache.width) *reinterpret_cast<u32x2_t*>(to + 2 * element) = u32x2_t{H::pack(y[0], y[1]), H::pack(y[2], y[3])};
    }
  if (a.lse && half == 0) a.lse[(int64_t)r.token * a.lse_heads + r.head] = behind ? NAN : any ? lse_of(all_m, all_l) : -INFINITY;
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
    known = token >= c.first_token && token - c.first_token < c.tokens;
    if (known) sight = sight_of(a, c, token - c.first_token);
  }
  if (!known && !a.zero_rest) return;
  float top = -INFINITY, sum = 0.f, o = 0.f;
  const int capacity = capacity_of(a);
  const int high = min(sight.high, capacity + 1);
  if (sight.low < high) {
    const int first = run_of_tile(sight.low / kTileKeys), last = run_of_tile((high - 1) / kTileKeys);
    for (int r0 = 0; r0 <= last - first; r0 += kJoinRuns) {
      const int count = min(kJoinRuns, last - first + 1 - r0);
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
  const bool sees = sight.high > sight.low, behind = sight.high > capacity;
  const float y = behind ? NAN : sees ? output_of(o, 1.f / sum) : 0.f;
  if (tid < width) *reinterpret_cast<uint16_t*>(out) = (uint16_t)Half<DTYPE>::pack(y, 0.f);
  if (a.lse && tid == 0) a.lse[(int64_t)token * a.lse_heads + head] = behind ? NAN : sees ? lse_of(top, sum) : -INFINITY;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct AttentionPlan {
  int rows;    // of a tile
  bool split;  // runs side by side
  bool longest_first;  // of the sequences
  int chunks, tiles;
  int key_heads;  // of a launch
};

// The most runs that a row sees: those of the table (with the position behind it), or of a window's tiles, which touch most runs where
// these are shortest and the first tile is the last one of a run.
static int run_limit(const rlk_paged_cache& c, int window) {
  const int all = run_of_tile(capacity_of(c) / kTileKeys) + 1;
  if (window == 0) return all;
  const int tiles = (int)(((int64_t)window + kTileKeys - 2) / kTileKeys) + 1, of_window = run_of_tile(kFirstRunTiles - 1 + tiles - 1) + 1;
  return of_window < all ? of_window : all;
}
static size_t parts_bytes(const rlk_paged_cache& c, int64_t tokens, int heads, int window) {
  return (size_t)run_limit(c, window) * tokens * heads * (c.width + 2) * sizeof(float);
}
// Parts take no more memory than this: a call that has more goes through its key heads in several launches, each of which fills the chip, and
// where a single key head has more, all runs go one after the other. In one launch / several / one after the other, us (32 heads, 8 key heads of
// 128, a table of 2^20 positions): 512 tokens over 2^20 10600 with 4.8 GB / 12000 with 0.6 / 20700, over 131072 1550 / 1810 / 2650; with a table
// of 131072, 100 sequences of 8 tokens 11640 with 1.6 GB / 10370 / 8830, 127 of 16 over 30000 3890 with 4.1 GB / 3180 / 2400.
constexpr size_t kMostParts = (size_t)1 << 30;

static bool pages_of_groups(const rlk_paged_cache& c) {
  const int64_t most = kSoloRange / 16;  // elements between rows: eight of them stay within a buffer's range
  return c.page_size % 8 == 0 && c.key_row_stride < most && c.value_row_stride < most;
}

// Tiles. A call is sized by what it may need: its tokens, spread evenly over the sequences, and the table's positions (or the window's).
// Measured, us, heads of 128, 8 key heads:
//   64 rows, runs one after the other / side by side: one token over 700 positions 25.6 / 16.1, 16 sequences over up to 1000 34 / 20, 64 of up to
//     8192 259 / 223, but 256 of up to 4000 384 / 452 (parts cost traffic), 32 with a window of 1024 47 / 49. Two workgroups share a CU.
//     A kernel of a single wave was slower everywhere (42 / 34 / 142 where two take 34 / 26 / 112): two share the loads.
//   rows 256 or 128, one after the other / side by side at 256: a chunk of 1000 over 4096 125, 107 / 169, over 65500 1724, 1570 / 1717,
//     of 256 over 1000 40, 34 / 40, over 16000 433, 351 / 161, 4 of 100 over up to 8192 230, 188 / 115, of 2000 over 4096 138, 166 / 302.
//   longest sequences first / as they come, where workgroups outnumber the chip: 64 of up to 8192 223 / 246, 128 368 / 462, with fewer
//     the ranks cost half a microsecond (16 of up to 1000 20.0 / 19.1). Twice as many parts for 64 rows: 236 / 244 for the first.
static AttentionPlan attention_plan(const rlk_paged_cache& c, int64_t tokens, int heads, int window, int config) {
  AttentionPlan p;
  const int group = heads / c.key_heads;
  const int most = c.width > 128 ? 128 : 256;  // rows of the largest tile
  const int choice = config & 0xff;
  const int64_t each = (tokens + c.sequences - 1) / c.sequences * group;  // rows of a sequence and key head
  const int64_t cus = device_cu_count();
  const int runs = run_limit(c, 0);
  p.key_heads = c.key_heads;
  auto side_by_side = [&](int rows) { return (int64_t)c.sequences * ((each + rows - 1) / rows) * p.key_heads; };
  const int64_t seen = window > 0 ? window + tokens / c.sequences : kMostKeys;
  const int64_t depth = (seen < capacity_of(c) ? seen : capacity_of(c)) / kTileKeys + 1;  // tiles that a row tile goes through
  if (choice != RLK_ATTENTION_CFG_AUTO) {
    p.rows = 64 << (choice - RLK_ATTENTION_CFG_ROWS64);
    p.split = (config & RLK_ATTENTION_CFG_SPLIT) != 0;
  } else {
    p.rows = each <= 64 ? 64 : each <= 128 ? 128 : most;
    if (p.rows == 256 && side_by_side(256) < cus && (4 * side_by_side(128) >= 3 * cus || depth < 32)) p.rows = 128;
    const int64_t units = side_by_side(p.rows);
    p.split = p.rows == 64 ? (units < cus && depth > 8) || (units < 4 * cus && depth >= 64) : 4 * units < 3 * cus && depth >= 32;
  }
  if (p.rows > most || !pages_of_groups(c)) p.rows = 128;
  const size_t of_key_head = parts_bytes(c, tokens, group, window);
  if (p.split && of_key_head * c.key_heads > kMostParts) {
    if (of_key_head > kMostParts && choice == RLK_ATTENTION_CFG_AUTO) {
      p.split = false;
    } else {
      const int at_once = of_key_head > kMostParts ? 1 : (int)(kMostParts / of_key_head), launches = (c.key_heads + at_once - 1) / at_once;
      p.key_heads = (c.key_heads + launches - 1) / launches;
    }
  }
  p.tiles = (int)(tokens * group / p.rows) + c.sequences + 1;
  p.chunks = 1;
  if (p.split) {
    const int64_t units = side_by_side(p.rows), wanted = ((p.rows == 64 ? 4 : 2) * cus + units - 1) / units, of_runs = depth / 4 + 1 < runs ? depth / 4 + 1 : runs;
    p.chunks = (int)(wanted < of_runs ? wanted : of_runs);
  }
  p.longest_first = c.sequences > 1 && side_by_side(p.rows) * p.chunks > (p.rows == 64 ? 2 : 1) * cus;
  return p;
}

size_t paged_attention_workspace_bytes(const rlk_paged_cache& c, int64_t tokens, int heads, int window, int config) {
  if (tokens == 0 || c.sequences == 0 || heads == 0) return 0;
  const AttentionPlan p = attention_plan(c, tokens, heads, window, config);
  return p.split ? parts_bytes(c, tokens, heads / c.key_heads * p.key_heads, window) : 0;
}

template <int DTYPE, int SLABS, int WAVES, bool SPLIT, bool GROUPED>
static hipError_t attention_tiles_launch(const AttentionArgs& a, hipStream_t stream) {
  constexpr int kLds = 4 * SLABS * kSlabBytes + (SLABS > 2 || WAVES <= 2 ? 0 : WAVES * SLABS * 4096) + 16;
  static PerDeviceOnce once;
  const auto kernel = attention_tile_kernel<DTYPE, SLABS, WAVES, SPLIT, GROUPED>;
  const hipError_t err = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds, once);
  if (err != hipSuccess) return err;
  const int64_t groups = (int64_t)a.tiles * a.chunks * a.cache.key_heads;
  if (groups * WAVES * 64 >= (int64_t)1 << 32) return hipErrorInvalidConfiguration;
  kernel<<<dim3((unsigned)groups), WAVES * 64, kLds, stream>>>(a);
  return hipGetLastError();
}
template <int DTYPE, int SLABS, bool SPLIT, bool GROUPED>
static hipError_t attention_tiles_of(const AttentionArgs& a, const AttentionPlan& p, hipStream_t stream) {
  if constexpr (GROUPED)
    if (p.rows == 64) return attention_tiles_launch<DTYPE, SLABS, 2, SPLIT, GROUPED>(a, stream);
  if constexpr (GROUPED && SLABS <= 2)
    if (p.rows == 256) return attention_tiles_launch<DTYPE, SLABS, 8, SPLIT, GROUPED>(a, stream);
  return attention_tiles_launch<DTYPE, SLABS, 4, SPLIT, GROUPED>(a, stream);
}
template <int DTYPE, int SLABS>
static hipError_t attention_launch_of(const AttentionArgs& a, const AttentionPlan& p, hipStream_t stream) {
  const bool grouped = pages_of_groups(a.cache);
  const hipError_t err = p.split ? (grouped ? attention_tiles_of<DTYPE, SLABS, true, true>(a, p, stream) : attention_tiles_of<DTYPE, SLABS, true, false>(a, p, stream))
                                 : (grouped ? attention_tiles_of<DTYPE, SLABS, false, true>(a, p, stream) : attention_tiles_of<DTYPE, SLABS, false, false>(a, p, stream));
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
  const AttentionPlan p = attention_plan(cache, tokens, heads, window, config);
  AttentionArgs a{};
  a.cache = cache;
  a.q_token_stride = 2 * q_token_stride, a.q_head_stride = 2 * q_head_stride;
  a.out_token_stride = 2 * out_token_stride, a.out_head_stride = 2 * out_head_stride;
  a.group = heads / cache.key_heads;
  a.by_page = page_divider((uint32_t)cache.page_size);
  a.by_group = page_divider((uint32_t)a.group);
  a.tokens = (int)tokens;
  a.lse_heads = heads;
  a.causal = causal, a.window = window, a.zero_rest = zero_rest;
  a.tiles = p.tiles, a.by_chunks = page_divider((uint32_t)p.chunks);
  a.chunks = p.chunks, a.longest_first = p.longest_first;
  a.scale = (float)((double)scale * 1.4426950408889634074);
  for (int first = 0; first < cache.key_heads; first += p.key_heads) {
    const int count = cache.key_heads - first < p.key_heads ? cache.key_heads - first : p.key_heads;
    a.cache.keys = static_cast<char*>(cache.keys) + 2 * first * cache.key_head_stride;
    a.cache.values = static_cast<char*>(cache.values) + 2 * first * cache.value_head_stride;
    a.cache.key_heads = count;
    a.q = static_cast<const char*>(q) + first * a.group * a.q_head_stride;
    a.out = static_cast<char*>(out) + first * a.group * a.out_head_stride;
    a.lse = lse != nullptr ? lse + first * a.group : nullptr;
    a.heads = count * a.group;
    a.by_key_heads = page_divider((uint32_t)count);
    a.part_rows = tokens * a.heads;
    if (p.split) {
      const int64_t parts = run_limit(cache, window) * a.part_rows;
      a.part_out = static_cast<float*>(workspace);
      a.part_max = a.part_out + parts * cache.width;
      a.part_sum = a.part_max + parts;
    }
    const hipError_t err = cache.dtype == RLK_DTYPE_BF16 ? attention_launch_as<RLK_DTYPE_BF16>(a, p, stream) : attention_launch_as<RLK_DTYPE_FP16>(a, p, stream);
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace rlk
