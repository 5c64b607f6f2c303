// Loads of materialised logits of any element type, and lane exchanges, shared by the kernels that reduce over them or write their gradient.
#pragma once

#include "linear_logp_common.h"
#include "rlk_host.h"

namespace rlk {

// What the forward leaves of the logits in the 256 MB memory-side cache, for a backward that starts at the columns the
// forward ended with: of larger logits the first workgroups read past the caches, or their lines would push out one another
// and those that are still to be used (the backward, whose reads are the last ones, does the same, see
// logits_backward_launch). Forward + backward, bf16, everything cached / 128 / 192 / 232 MiB: 2048 x 151936 356.5 / 364.2 /
// 349.6 / 347.0 us, 1000 x 151936 168.2 / 179.6 / 170.7 / 166.2, 4096 x 32000 149.8 / 159.7 / 154.9 / 149.6, 20000 x 32000
// 798.6 / 765.5 / 759.8 / 757.9, fp32 2048 x 65536 322.4 / 322.6 / 313.4 / 309.7; the forward alone 129.5 -> 126.4 us at
// 2048 x 151936, 305 -> 294 at 20000 x 32000, equal below.
constexpr int64_t kCachedLogitsBytes = (int64_t)232 << 20;

template <int ELEM>
struct LogitElem;

template <>
struct LogitElem<RLK_DTYPE_BF16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t from_float(float f) {
    return (uint16_t)(pack_bf16x2(f, 0.f) & 0xffffu);
  }
};
template <>
struct LogitElem<RLK_DTYPE_FP16> {
  using type = _Float16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from_float(float f) { return (_Float16)f; }
};
template <>
struct LogitElem<RLK_DTYPE_FP32> {
  using type = float;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float f) { return f; }
};

// Columns [g * VEC, g * VEC + VEC) of a row as floats; `aligned` says the row base is 16-byte
// aligned, `cols` bounds the row (a vector that would run past it is read element by element).
// NT: the load leaves nothing in the caches.
template <bool NT, class V>
__device__ __forceinline__ V load_vector(const V* p) {
  if constexpr (NT) {
    return __builtin_nontemporal_load(p);
  } else {
    return *p;
  }
}

template <int ELEM, bool NT>
__device__ __forceinline__ void load_logit_vector(const typename LogitElem<ELEM>::type* row, int col, int cols,
                                                  bool aligned, float (&out)[LogitElem<ELEM>::kVec]) {
  using L = LogitElem<ELEM>;
  using E = typename L::type;
  constexpr int kBytes = L::kVec * (int)sizeof(E);
  if (aligned && col + L::kVec <= cols) {
    E vals[L::kVec];
    const u32x4_t* src = reinterpret_cast<const u32x4_t*>(row + col);
    u32x4_t raw[kBytes / 16];
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) raw[i] = load_vector<NT>(src + i);
    __builtin_memcpy(vals, raw, kBytes);
#pragma unroll
    for (int i = 0; i < L::kVec; ++i) out[i] = L::to_float(vals[i]);
  } else {
#pragma unroll
    for (int i = 0; i < L::kVec; ++i) out[i] = (col + i < cols) ? L::to_float(row[col + i]) : 0.f;
  }
}

// The eight values of vector g of a row, widened to fp32. ALIGNED: every row is made of whole,
// 16-byte aligned vectors (decided once on the host), so a vector is one or two 16-byte loads from a
// uniform row base plus a 32-bit lane offset; otherwise element by element, columns past the row as 0.
template <int ELEM, bool ALIGNED>
struct RawVector;

template <bool ALIGNED>
struct RawVector<RLK_DTYPE_BF16, ALIGNED> {
  u32x4_t w;
  template <bool NT>
  __device__ __forceinline__ void load(const uint16_t* row, int g, int cols) {
    if constexpr (ALIGNED) {
      w = load_vector<NT>(reinterpret_cast<const u32x4_t*>(reinterpret_cast<const char*>(row) + (uint32_t)g * 16u));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = g * 8 + 2 * i;
        const uint32_t lo = c < cols ? row[c] : 0u, hi = c + 1 < cols ? row[c + 1] : 0u;
        w[i] = lo | (hi << 16);
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = __uint_as_float(w[i] << 16);
      y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

template <bool ALIGNED>
struct RawVector<RLK_DTYPE_FP16, ALIGNED> {
  _Float16 h[8];
  template <bool NT>
  __device__ __forceinline__ void load(const _Float16* row, int g, int cols) {
    if constexpr (ALIGNED) {
      const u32x4_t w = load_vector<NT>(reinterpret_cast<const u32x4_t*>(reinterpret_cast<const char*>(row) + (uint32_t)g * 16u));
      __builtin_memcpy(h, &w, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = g * 8 + i < cols ? row[g * 8 + i] : (_Float16)0.f;
    }
  }
  __device__ __forceinline__ void unpack(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)h[i];
  }
};

template <bool ALIGNED>
struct RawVector<RLK_DTYPE_FP32, ALIGNED> {
  f32x4_t lo, hi;
  template <bool NT>
  __device__ __forceinline__ void load(const float* row, int g, int cols) {
    if constexpr (ALIGNED) {
      const char* p = reinterpret_cast<const char*>(row) + (uint32_t)g * 32u;
      lo = load_vector<NT>(reinterpret_cast<const f32x4_t*>(p));
      hi = load_vector<NT>(reinterpret_cast<const f32x4_t*>(p) + 1);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = g * 8 + i < cols ? row[g * 8 + i] : 0.f;
        hi[i] = g * 8 + 4 + i < cols ? row[g * 8 + 4 + i] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = lo[i];
      y[4 + i] = hi[i];
    }
  }
};

typedef u32x4_t u32x4_at2_t __attribute__((aligned(2)));
typedef u32x4_t u32x4_at4_t __attribute__((aligned(4)));
template <int BYTES>
struct UnalignedPart {
  using type = u32x4_at2_t;
};
template <>
struct UnalignedPart<4> {
  using type = u32x4_at4_t;
};

// The first of the eight columns that a load at `col` of a row of `cols` columns brings (RowVector::load_window).
__device__ __forceinline__ int window_of(int col, int cols) {
  const int last = cols > 8 ? cols - 8 : 0;
  return col < last ? col : last;
}

// Eight logits of a row. Rows may start at any element: the loads ask for the element's alignment only.
template <int ELEM>
struct RowVector {
  using E = typename LogitElem<ELEM>::type;
  static constexpr int kParts = (int)sizeof(E) / 2;
  using Part = typename UnalignedPart<(int)sizeof(E)>::type;
  u32x4_t w[kParts];

  template <bool NT>
  __device__ __forceinline__ void load(const E* p) {
    const Part* src = reinterpret_cast<const Part*>(p);
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      if constexpr (NT) {
        w[i] = __builtin_nontemporal_load(src + i);
      } else {
        w[i] = src[i];
      }
    }
  }
  // vector g of a row of `cols` columns, those behind it 0
  template <bool NT>
  __device__ __forceinline__ void load_edge(const E* row, int g, int cols) {
    if ((int64_t)g * 8 + 8 <= cols) {
      load<NT>(row + (int64_t)g * 8);
    } else {
      E vals[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) vals[i] = (int64_t)g * 8 + i < cols ? row[(int64_t)g * 8 + i] : E(0);
      __builtin_memcpy(w, vals, sizeof(w));
    }
  }
  // Columns [col, col + 8): a uniform row and a lane's offset of 32 bits (rows have up to 2^28 columns).
  template <bool NT>
  __device__ __forceinline__ void load_at(const E* row, uint32_t col) {
    load<NT>(reinterpret_cast<const E*>(reinterpret_cast<const char*>(row) + col * (uint32_t)sizeof(E)));
  }
  // Columns [window_of(col, cols), + 8): a vector that would run past the row is read from further left, so that it is one wide
  // load as well. (Element by element it was the better half of a kernel's code, all of it fetched once by a call of one row.)
  template <bool NT>
  __device__ __forceinline__ void load_window(const E* row, int col, int cols) {
    if (cols >= 8) {
      load_at<NT>(row, (uint32_t)(col < cols - 8 ? col : cols - 8));
    } else if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = reinterpret_cast<const uint32_t*>(row)[i < cols ? i : cols - 1];
    } else {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[0][i] = bits[2 * i < cols ? 2 * i : cols - 1] | (uint32_t)bits[2 * i + 1 < cols ? 2 * i + 1 : cols - 1] << 16;
    }
  }
  // (word by word: held as an array of halves the eight would take a register each while they wait)
  __device__ __forceinline__ void unpack(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (ELEM == RLK_DTYPE_FP32) y[i] = __uint_as_float(w[i / 4][i % 4]);
      else if constexpr (ELEM == RLK_DTYPE_BF16) y[i] = __uint_as_float(i % 2 ? w[0][i / 2] & 0xffff0000u : w[0][i / 2] << 16);
      else y[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[0][i / 2] >> (16 * (i % 2))));
    }
  }
  // (fp16: the fp32 value is fixed first. Left alone the compiler rounds some last products straight to fp16, some not.)
  __device__ __forceinline__ void pack(const float (&y)[8]) {
    E vals[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = y[i];
      if constexpr (ELEM == RLK_DTYPE_FP16) asm volatile("" : "+v"(v));
      vals[i] = LogitElem<ELEM>::from_float(v);
    }
    __builtin_memcpy(w, vals, sizeof(w));
  }
  template <bool NT>
  __device__ __forceinline__ void store(E* p) const {
    Part* dst = reinterpret_cast<Part*>(p);
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      if constexpr (NT) {
        __builtin_nontemporal_store(w[i], dst + i);
      } else {
        dst[i] = w[i];
      }
    }
  }
  // to columns [col, col + 8) of a row, those from `cols` on left as they are
  template <bool NT>
  __device__ __forceinline__ void store_edge(E* row, int64_t col, int64_t cols) const {
    if (col + 8 <= cols) {
      store<NT>(row + col);
    } else {
      E vals[8];
      __builtin_memcpy(vals, w, sizeof(w));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < cols) row[col + i] = vals[i];
    }
  }
};

// max(a, b, c) in one instruction. (fmaxf on values that come out of integer shifts costs an extra
// canonicalising instruction per operand; v_max3_f32 needs none. For the non-NaN values of this contract it
// returns what nested fmaxf returns.)
__device__ __forceinline__ float max3_f32(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Value of lane (l ^ OFFSET) for OFFSET 1, 2 (DPP quad permutes) and 4, 8 (ds_swizzle xor mode).
template <int OFFSET>
__device__ __forceinline__ float xor_lane(float v) {
  const int bits = __float_as_int(v);
  int out;
  if constexpr (OFFSET == 1) {
    out = __builtin_amdgcn_update_dpp(bits, bits, 0xB1, 0xf, 0xf, false);  // quad_perm [1, 0, 3, 2]
  } else if constexpr (OFFSET == 2) {
    out = __builtin_amdgcn_update_dpp(bits, bits, 0x4E, 0xf, 0xf, false);  // quad_perm [2, 3, 0, 1]
  } else {
    out = __builtin_amdgcn_ds_swizzle(bits, (OFFSET << 10) | 0x1f);  // and 0x1f, or 0, xor OFFSET
  }
  return __int_as_float(out);
}

template <bool V>
struct BoolConstant {
  static constexpr bool value = V;
};

constexpr int kTileLanes = 16;                    // lanes that share a tile
constexpr int kTilesPerWave = kWave / kTileLanes;  // 4

}  // namespace rlk
