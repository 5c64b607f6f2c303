// Rotary positions for gfx950, of queries and keys in one launch, on their own or on the way into a paged cache.
//
// A pair (a, b) of a head's elements at position p becomes m (a cos t - b sin t, b cos t + a sin t), t = p f with the pair's frequency
// f in radians a position. p f has far more turns than an fp32 product could hold (position 10^6 at one radian is 1.6 10^5 turns, an
// ulp of it 4 degrees), so t is taken in turns in 64 bits, whole turns are dropped there, and only the rest, half a turn at most, is
// rounded to fp32 for the sine and cosine.
//
// HBM-bound: every element is read once and written once. A token's sines and cosines are the same for all its heads: a
// workgroup has one token, computes them once into LDS (one 64-bit product and one sincospi for each pair) and then goes through the
// heads, a 16-byte piece of a thread at a time (both halves of eight pairs where they lie apart). Four tokens a workgroup computed the
// same in fewer, longer workgroups: 8192 tokens of 40 heads of 128 with their gradient 70 us, with one each 66 (5.1 TB/s, above a
// large copy's 4.9); 4095 tokens into a paged cache 36 and 28.5 (3.5 TB/s: its sequence, page and place are three loads one after the other
// before the first store).
#include "paged.h"

namespace rlk {

constexpr int kRotaryThreads = 256;
constexpr int64_t kRotaryGroups = 1 << 23;  // workgroups of a launch at most (a grid has fewer than 2^32 threads)

template <int ELEM>
struct RotaryElem;
template <>
struct RotaryElem<RLK_DTYPE_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float widen(uint16_t v) { return bf16_bits_to_float(v); }
  static __device__ __forceinline__ uint16_t narrow(float v) { return to_bf16_bits(v); }
};
template <>
struct RotaryElem<RLK_DTYPE_FP16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float widen(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
template <>
struct RotaryElem<RLK_DTYPE_FP32> {
  typedef float type;
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
};

// 16 bytes of a row.
template <class T>
struct RowPiece {
  static constexpr int kCount = 16 / sizeof(T);
  T v[kCount];
  __device__ __forceinline__ void load(const T* from) { *reinterpret_cast<u32x4_t*>(v) = *reinterpret_cast<const u32x4_t*>(from); }
  __device__ __forceinline__ void store(T* to) const { *reinterpret_cast<u32x4_t*>(to) = *reinterpret_cast<const u32x4_t*>(v); }
};

enum RowTarget { kToRows, kToKeys, kToValues };

struct RotaryPart {
  rlk_head_rows rows;
  int target;      // RowTarget
  int first_head;  // of all parts' heads together
};
struct RotaryArgs {
  RotaryPart part[3];
  int parts, heads;  // of all parts
  rlk_rotary rotary;
  rlk_paged_cache cache;  // of an append
  PageDivider by_page, by_items, by_inner;
  int64_t tokens, inner, first;  // (of this launch)
  int width, items;  // pieces (or single pairs and elements) of a head
  float sign;
};

// What a workgroup knows of its token.
struct TokenPlace {
  int64_t key_base, value_base;  // of its cache row, -1 where it has none
  int64_t position;
  int known;  // whether a sequence has it
};

template <int ELEM, bool WHOLE, bool APPEND>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
  typedef RotaryElem<ELEM> E;
  typedef typename E::type T;
  extern __shared__ float2 turn[];  // [pairs] cosine and sine, scaled
  const int tid = threadIdx.x, pairs = a.rotary.pairs;
  const int64_t t = a.first + blockIdx.x;

  TokenPlace place = {-1, -1, 0, 0};
  if (APPEND) {  // every wave for itself
    const int s = wave_search(a.cache.sequences + 1, t, tid & 63, [&](int i) { return (int64_t)a.cache.starts[i]; });
    if (s >= 0 && s < a.cache.sequences && t >= a.cache.starts[s] && t < a.cache.starts[s + 1]) {  // (starts need not ascend)
      place.known = 1;
      place.position = (int64_t)a.cache.lengths[s] - a.cache.starts[s + 1] + t;
      if (place.position >= 0 && place.position < 0x7fffffff) {
        const uint32_t column = divide_by((uint32_t)place.position, a.by_page);
        const int page = page_at(a.cache, s, (int)column);
        if (page >= 0) {
          const int64_t row = place.position - (int64_t)column * a.cache.page_size;
          place.key_base = page * a.cache.key_page_stride + row * a.cache.key_row_stride;
          place.value_base = page * a.cache.value_page_stride + row * a.cache.value_row_stride;
        }
      }
    }
  }
  for (int i = tid; i < pairs; i += kRotaryThreads) {
    int64_t position;
    if (a.rotary.positions == nullptr)
      position = place.position;
    else if (a.rotary.positions_are_64)
      position = static_cast<const int64_t*>(a.rotary.positions)[t];
    else
      position = static_cast<const int32_t*>(a.rotary.positions)[t];
    constexpr double kTurnsPerRadian = 0.15915494309189533577;
    double turns = (double)position * (a.rotary.frequencies[i] * kTurnsPerRadian);
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    turn[i] = make_float2(c * a.rotary.magnitude, s * a.rotary.magnitude * a.sign);
  }
  __syncthreads();

  const int64_t outer = (int64_t)(a.inner == a.tokens ? 0 : divide_by((uint32_t)t, a.by_inner)), inner = t - outer * a.inner;
  for (int i = tid; i < a.heads * a.items; i += kRotaryThreads) {
    const int any_head = (int)divide_by((uint32_t)i, a.by_items);
    const int item = i - any_head * a.items;
    int which = 0;
    if (a.parts > 1 && any_head >= a.part[1].first_head) which = 1;
    if (APPEND && a.parts > 2 && any_head >= a.part[2].first_head) which = 2;
    const RotaryPart& part = a.part[which];
    const int head = any_head - part.first_head;
    const T* x = static_cast<const T*>(part.rows.x) + outer * part.rows.x_outer_stride + inner * part.rows.x_token_stride + head * part.rows.x_head_stride;
    T* y;
    bool turns = pairs > 0, zero = false;
    if (!APPEND || part.target == kToRows) {
      y = static_cast<T*>(part.rows.y) + outer * part.rows.y_outer_stride + inner * part.rows.y_token_stride + head * part.rows.y_head_stride;
      zero = APPEND && !place.known;
    } else if (part.target == kToKeys) {
      if (place.key_base < 0) continue;
      y = static_cast<T*>(a.cache.keys) + place.key_base + head * a.cache.key_head_stride;
    } else {
      if (place.key_base < 0) continue;
      y = static_cast<T*>(a.cache.values) + place.value_base + head * a.cache.value_head_stride;
      turns = false;
    }
    const float2* const by = turn;
    if (WHOLE) {
      typedef RowPiece<T> Piece;
      constexpr int kCount = Piece::kCount;
      const int half_items = pairs / kCount;  // (with pairs apart)
      Piece p, r;
      if (a.rotary.interleaved || item >= half_items) {  // one piece: pairs side by side, or a copy
        const int at = a.rotary.interleaved ? item * kCount : (item + half_items) * kCount;
        p.load(x + at);
        if (turns && at < 2 * pairs) {
#pragma unroll
          for (int e = 0; e < kCount; e += 2) {
            const float2 cs = by[(at + e) >> 1];
            const float u = E::widen(p.v[e]), v = E::widen(p.v[e + 1]);
            p.v[e] = E::narrow(__builtin_fmaf(u, cs.x, -(v * cs.y)));
            p.v[e + 1] = E::narrow(__builtin_fmaf(v, cs.x, u * cs.y));
          }
        }
        if (zero) p = Piece{};
        p.store(y + at);
      } else {  // a piece of each half
        const int at = item * kCount;
        p.load(x + at);
        r.load(x + pairs + at);
        if (turns) {
#pragma unroll
          for (int e = 0; e < kCount; ++e) {
            const float2 cs = by[at + e];
            const float u = E::widen(p.v[e]), v = E::widen(r.v[e]);
            p.v[e] = E::narrow(__builtin_fmaf(u, cs.x, -(v * cs.y)));
            r.v[e] = E::narrow(__builtin_fmaf(v, cs.x, u * cs.y));
          }
        }
        if (zero) p = Piece{}, r = Piece{};
        p.store(y + at);
        r.store(y + pairs + at);
      }
    } else if (item < pairs) {
      const int first = a.rotary.interleaved ? 2 * item : item, second = a.rotary.interleaved ? 2 * item + 1 : item + pairs;
      T p = x[first], r = x[second];
      if (turns) {
        const float2 cs = by[item];
        const float u = E::widen(p), v = E::widen(r);
        p = E::narrow(__builtin_fmaf(u, cs.x, -(v * cs.y)));
        r = E::narrow(__builtin_fmaf(v, cs.x, u * cs.y));
      }
      y[first] = zero ? T(0) : p;
      y[second] = zero ? T(0) : r;
    } else {
      y[item + pairs] = zero ? T(0) : x[item + pairs];
    }
  }
}

// Whether every head of the tensor starts on 16 bytes.
static bool whole_pieces(const void* base, int64_t outer, int64_t token, int64_t head, int count) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && outer % count == 0 && token % count == 0 && head % count == 0;
}

template <int ELEM>
static hipError_t rotary_launch_as(RotaryArgs& a, bool append, hipStream_t stream) {
  constexpr int kCount = RowPiece<typename RotaryElem<ELEM>::type>::kCount;
  const int pairs = a.rotary.pairs;
  bool whole = a.width % kCount == 0 && (a.rotary.interleaved ? 2 * pairs : pairs) % kCount == 0;
  for (int i = 0; i < a.parts; ++i) {
    const rlk_head_rows& r = a.part[i].rows;
    const bool split = a.inner != a.tokens;  // (else the outer stride is not used)
    whole = whole && whole_pieces(r.x, split ? r.x_outer_stride : 0, r.x_token_stride, r.x_head_stride, kCount);
    if (a.part[i].target == kToRows) whole = whole && whole_pieces(r.y, split ? r.y_outer_stride : 0, r.y_token_stride, r.y_head_stride, kCount);
  }
  if (append)
    whole = whole && whole_pieces(a.cache.keys, a.cache.key_page_stride, a.cache.key_row_stride, a.cache.key_head_stride, kCount) &&
            whole_pieces(a.cache.values, a.cache.value_page_stride, a.cache.value_row_stride, a.cache.value_head_stride, kCount);
  a.items = whole ? (a.rotary.interleaved ? a.width : a.width - pairs) / kCount : a.width - pairs;
  a.by_items = page_divider(a.items);
  const size_t lds = sizeof(float2) * (pairs > 0 ? pairs : 1);
  for (a.first = 0; a.first < a.tokens; a.first += kRotaryGroups) {
    const dim3 grid((unsigned)(a.tokens - a.first < kRotaryGroups ? a.tokens - a.first : kRotaryGroups));
    if (append && whole)
      rotary_kernel<ELEM, true, true><<<grid, kRotaryThreads, lds, stream>>>(a);
    else if (append)
      rotary_kernel<ELEM, false, true><<<grid, kRotaryThreads, lds, stream>>>(a);
    else if (whole)
      rotary_kernel<ELEM, true, false><<<grid, kRotaryThreads, lds, stream>>>(a);
    else
      rotary_kernel<ELEM, false, false><<<grid, kRotaryThreads, lds, stream>>>(a);
  }
  return hipGetLastError();
}

static hipError_t rotary_launch_any(RotaryArgs& a, int dtype, bool append, hipStream_t stream) {
  switch (dtype) {
    case RLK_DTYPE_BF16: return rotary_launch_as<RLK_DTYPE_BF16>(a, append, stream);
    case RLK_DTYPE_FP16: return rotary_launch_as<RLK_DTYPE_FP16>(a, append, stream);
    default: return rotary_launch_as<RLK_DTYPE_FP32>(a, append, stream);
  }
}

hipError_t rotary_launch(const rlk_rotary& rotary, const rlk_head_rows& q, const rlk_head_rows* k, int64_t tokens, int64_t inner, int width,
                         int dtype, bool inverse, hipStream_t stream) {
  RotaryArgs a{};
  a.part[0] = {q, kToRows, 0};
  if (k != nullptr) a.part[1] = {*k, kToRows, q.heads};
  a.parts = k != nullptr ? 2 : 1;
  a.heads = q.heads + (k != nullptr ? k->heads : 0);
  a.rotary = rotary;
  a.tokens = tokens;
  a.inner = inner;
  a.by_inner = page_divider((uint32_t)inner);
  a.width = width;
  a.sign = inverse ? -1.f : 1.f;
  return rotary_launch_any(a, dtype, false, stream);
}

hipError_t paged_append_launch(const rlk_paged_cache& cache, const rlk_rotary* rotary, const rlk_head_rows* q, const rlk_head_rows& k,
                               const rlk_head_rows& v, int64_t tokens, hipStream_t stream) {
  RotaryArgs a{};
  int heads = 0;
  if (q != nullptr) {
    a.part[a.parts++] = {*q, kToRows, 0};
    heads = q->heads;
  }
  a.part[a.parts++] = {k, kToKeys, heads};
  a.part[a.parts++] = {v, kToValues, heads + cache.key_heads};
  a.heads = heads + 2 * cache.key_heads;
  if (rotary != nullptr) a.rotary = *rotary;
  a.cache = cache;
  a.by_page = page_divider((uint32_t)cache.page_size);
  a.tokens = a.inner = tokens;
  a.width = cache.width;
  a.sign = 1.f;
  return rotary_launch_any(a, cache.dtype, true, stream);
}

}  // namespace rlk
