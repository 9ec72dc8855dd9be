// Device-side building blocks of the paged-cache kernels.
#pragma once

#include "tla_device.cuh"
#include "tla_internal.h"

namespace tla {

// First element of a (page, kv head, slot) row of the pool. (A bounds-check
// build reports a row outside the pool and hands out row 0.)
__device__ __forceinline__ int64_t pool_row(const PagedArgs& p, int page, int kvh, int slot) {
  if (!TLA_IN_BOUNDS(page, p.page_count, p.a.error) || !TLA_IN_BOUNDS(kvh, p.a.Hk, p.a.error) ||
      !TLA_IN_BOUNDS(slot, 1 << p.page_shift, p.a.error))
    return 0;
  return page * p.page_stride + kvh * p.head_stride + slot * p.slot_stride;
}

// First element of a (page, kv head)'s bounds: [low, high][D].
__device__ __forceinline__ int64_t bounds_row(const PagedArgs& p, int page, int kvh, int D) {
  if (!TLA_IN_BOUNDS(page, p.page_count, p.a.error) || !TLA_IN_BOUNDS(kvh, p.a.Hk, p.a.error)) return 0;
  return (static_cast<int64_t>(page) * p.a.Hk + kvh) * 2 * D;
}

// The page that holds logical page `index` of sequence b, or -1 (reported)
// when the table's entry is not a page of the pool. index < p.width.
__device__ __forceinline__ int pool_page(const PagedArgs& p, int b, int index) {
  const int page = p.table[static_cast<int64_t>(b) * p.width + index];
  if (static_cast<unsigned>(page) < static_cast<unsigned>(p.page_count)) return page;
  report_error(p.a.error, TLA_ERR_PAGE);
  return -1;
}

// Tokens [lo, hi] that a sequence at `pos` attends to (math.ts:208's window);
// empty (lo > hi) for a row without a sequence or a position past the capacity.
__device__ __forceinline__ bool paged_range(const PagedArgs& p, int pos, int* lo, int* hi) {
  const bool held = pos >= 0 && pos < p.capacity;
  *lo = held && p.a.sliding > 0 ? max(0, pos - p.a.sliding + 1) : 0;
  *hi = held ? pos : -1;
  return held;
}

// Entries of a page list that count: the strictly rising prefix of pages that
// the sequence has. Called by a whole warp; lane 0 reports a faulty list.
__device__ __forceinline__ int list_length(const PagedArgs& p, const int32_t* list, int count, int last_page,
                                           int lane) {
  int n = 0;
  for (int base = 0; base < count; base += 32) {
    const int i = base + lane;
    const int e = i < count ? list[i] : -1;
    const int before = i > 0 && i < count ? list[i - 1] : -1;
    const bool good = e >= 0 && e > before && e <= last_page;
    const unsigned bad = __ballot_sync(0xffffffffu, !good);
    if (bad != 0) {
      const int stop = __ffs(bad) - 1;
      if (lane == stop && e >= 0) report_error(p.a.error, TLA_ERR_PAGE);
      return n + stop;
    }
    n += 32;
  }
  return count;
}

}  // namespace tla
