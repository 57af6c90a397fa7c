// Where the rows of a page pool are, and how the tiles of an attention call are
// dealt to its workgroups: plain integer functions, the same on the host (where
// their bounds are tested) and on the device.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define SI_HD __host__ __device__ __forceinline__
#else
#define SI_HD static inline
#endif

// Row of (page, head, offset) in the pool's [pages, heads, page_size] rows, -1 for
// a page outside the pool. Pools have fewer than 2^31 rows.
SI_HD int32_t si_page_row(int64_t page, int64_t pages, int32_t head, int32_t heads, int32_t offset,
                          int32_t page_size) {
  if (page < 0 || page >= pages) return -1;
  return (int32_t)((page * heads + head) * page_size + offset);
}

// Row of a slot (page * page_size + offset) of one head, -1 for a slot outside.
SI_HD int32_t si_slot_row(int64_t slot, int64_t pages, int32_t head, int32_t heads, int32_t page_size) {
  if (slot < 0 || slot >= pages * page_size) return -1;
  const uint32_t s = (uint32_t)slot, p = s / (uint32_t)page_size;
  return si_page_row(p, pages, head, heads, (int32_t)(s - p * (uint32_t)page_size), page_size);
}

// Positions [lo, hi) that take part: the last `window` (0: all) of `length`, which
// is cut to what a page table of `capacity` positions can hold.
SI_HD int32_t si_span_hi(int32_t length, int64_t capacity) {
  const int64_t n = length < 0 ? 0 : length;
  return (int32_t)(n < capacity ? n : capacity);
}
SI_HD int32_t si_span_lo(int32_t hi, int32_t window) {
  return window > 0 && hi > window ? hi - window : 0;
}
SI_HD int32_t si_span_tiles(int32_t lo, int32_t hi, int32_t tile) {
  return (int32_t)(((int64_t)hi - lo + tile - 1) / tile);
}

// Workgroups that share `total` tiles: each has one at least.
SI_HD int64_t si_part_count(int64_t total, int64_t most) { return total < most ? total : most; }
// Tiles [begin(w), begin(w + 1)) of `total` go to workgroup w of `parts`.
SI_HD int64_t si_part_begin(int64_t w, int64_t total, int64_t parts) { return w * total / parts; }
// The workgroup that has tile f.
SI_HD int64_t si_part_of(int64_t f, int64_t total, int64_t parts) {
  return ((f + 1) * parts - 1) / total;
}
// A workgroup leaves at most two unfinished items: the one its range begins inside
// of (slot 2w), and another that goes on in the next workgroup (slot 2w + 1).
SI_HD int64_t si_part_slot(int64_t w, int begins_inside) { return 2 * w + (begins_inside ? 0 : 1); }
