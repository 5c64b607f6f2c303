// What appending to a paged cache and attending over it share: finding a token's sequence and a position's page.
#pragma once

#include "rlk_device.h"
#include "rlk_host.h"

namespace rlk {

// n / d for n < 2^31 by a product.
struct PageDivider {
  uint32_t factor, shift, d;
};
inline PageDivider page_divider(uint32_t d) {
  uint32_t shift = 0;
  while (((uint64_t)1 << shift) < d) ++shift;
  const uint64_t factor = (((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1;
  return {(uint32_t)factor, shift, d};
}
__device__ __forceinline__ uint32_t divide_by(uint32_t n, const PageDivider& by) { return (__umulhi(n, by.factor) + n) >> by.shift; }

// The largest s in [0, count) with at(s) <= value, or -1; at() ascends. The 64 lanes of a wave look at 64 places at a time, so that up
// to 64 sequences take one load and 4096 two. Whatever at() returns, only places below count are looked at and every round leaves
// fewer than the one before.
template <class At>
__device__ __forceinline__ int wave_search(int count, int64_t value, int lane, const At& at) {
  int low = 0, left = count;
  for (bool first = true; first || left > 1; first = false) {
    const int step = (left + 63) >> 6;
    const int64_t place = (int64_t)lane * step;
    const bool below = place < left && at(low + (int)place) <= value;
    const int hits = __popcll(__ballot(below));
    if (hits == 0) return first ? -1 : low;
    low += (hits - 1) * step;
    const int rest = left - (hits - 1) * step;
    left = rest < step ? rest : step;
  }
  return low;
}

// The page of a position, or -1 where it is missing.
__device__ __forceinline__ int page_at(const rlk_paged_cache& c, int sequence, int column) {
  if (column >= c.table_columns) return -1;
  const int page = c.table[(int64_t)sequence * c.table_row_stride + column];
  return page >= 0 && page < c.pages ? page : -1;
}

}  // namespace rlk
