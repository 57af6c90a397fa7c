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
SI_HD int32_t si_page_row(int32_t page, int32_t pages, int32_t head, int32_t heads, int32_t offset,
                          int32_t page_size) {
  if ((uint32_t)page >= (uint32_t)pages) return -1;
  return (page * heads + head) * page_size + offset;
}

// Row of a slot (page * page_size + offset) of one head, -1 for a slot outside.
SI_HD int32_t si_slot_row(int64_t slot, int32_t pages, int32_t head, int32_t heads, int32_t page_size) {
  if (slot < 0 || slot >= (int64_t)pages * page_size) return -1;
  const uint32_t s = (uint32_t)slot, p = s / (uint32_t)page_size;
  return si_page_row((int32_t)p, pages, head, heads, (int32_t)(s - p * (uint32_t)page_size), page_size);
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
// Tiles start at a multiple of eight, so that eight positions from there lie in one
// page where the page size is one too; the positions before lo are masked.
SI_HD int32_t si_span_origin(int32_t lo) { return lo & ~7; }
SI_HD int32_t si_span_tiles(int32_t lo, int32_t hi, int32_t tile) {
  return hi > lo ? (int32_t)(((int64_t)hi - si_span_origin(lo) + tile - 1) / tile) : 0;
}

// t / d for 0 <= t < 2^31 by a multiplication (the round-up method: with 2^shift the
// power of two from d on, m = floor(2^32 (2^shift - d) / d) + 1).
typedef struct {
  uint32_t m, shift;
} si_divisor;
static inline si_divisor si_make_divisor(uint32_t d) {
  si_divisor r = {0, 0};
  while (((uint64_t)1 << r.shift) < d) ++r.shift;
  r.m = (uint32_t)(((((uint64_t)1 << r.shift) - d) << 32) / d + 1);
  return r;
}
SI_HD uint32_t si_divide(uint32_t t, si_divisor d) {
  return ((uint32_t)(((uint64_t)t * d.m) >> 32) + t) >> d.shift;
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
