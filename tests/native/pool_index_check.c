/*
 * Checks the integer functions that place the page pool's rows and deal an
 * attention call's tiles (shadow-infer_amd/csrc/si_pool_index.h):
 *
 *  1. rows of slots and of table entries are in [0, pages * heads * page_size) or -1,
 *     distinct slots have distinct rows, and pages or slots outside give -1;
 *  2. spans: [lo, hi) within [0, capacity], at most `window` long, tiles cover it from a
 *     multiple of eight; divisions by a multiplication are exact below 2^31;
 *  3. dealing, walked as the kernel walks it: every tile of every item is taken once,
 *     every block has at least one tile, an item that one block takes whole leaves no
 *     partial, no partial slot is written twice or past 2 * most, and the join of an
 *     item reads exactly the slots its blocks wrote.
 * Prints the number of cases; exit status 0 iff all hold.
 */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../shadow-infer_amd/csrc/si_pool_index.h"

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)

static uint64_t rng_state = 12345;
static uint64_t rnd(uint64_t n) {
  uint64_t z = (rng_state += 0x9E3779B97F4A7C15ull);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (z ^ (z >> 31)) % n;
}

static void rows(void) {
  const int32_t pages = 1 + (int32_t)rnd(9);
  const int heads = 1 + (int)rnd(5), P = 1 + (int)rnd(20);
  const int64_t n = (int64_t)pages * heads * P;
  char* seen = calloc((size_t)n, 1);
  for (int h = 0; h < heads; ++h)
    for (int64_t s = -3; s < pages * P + 3; ++s) {
      const int32_t r = si_slot_row(s, pages, h, heads, P);
      if (s < 0 || s >= pages * P) { CHECK(r == -1); continue; }
      CHECK(r >= 0 && r < n && !seen[r]);
      seen[r] = 1;
      CHECK(r == si_page_row((int32_t)(s / P), pages, h, heads, (int32_t)(s % P), P));
    }
  free(seen);
  CHECK(si_page_row(-2147483647 - 1, pages, 0, heads, 0, P) < 0 && si_page_row(2147483647, pages, 0, heads, 0, P) < 0);
  for (int32_t p = -2; p < pages + 2; ++p)
    CHECK((si_page_row(p, pages, 0, heads, 0, P) >= 0) == (p >= 0 && p < pages));
}

static void large_rows(void) {  /* 2^31 - 1 rows at most: the last one */
  CHECK(si_page_row(16777215, 16777216, 7, 8, 14, 15) == (int32_t)(16777215LL * 120 + 7 * 15 + 14));
  CHECK(si_slot_row(16777216LL * 15 - 1, 16777216, 7, 8, 15) == 2013265919);
  CHECK(si_slot_row((int64_t)1 << 40, 16777216, 0, 8, 15) == -1);
}

static void spans(void) {
  const int64_t cap = rnd(2000);
  const int32_t len = (int32_t)rnd(3000) - 200, win = (int32_t)rnd(3) ? (int32_t)rnd(500) : 0;
  const int32_t hi = si_span_hi(len, cap), lo = si_span_lo(hi, win), n = si_span_tiles(lo, hi, 128);
  CHECK(lo >= 0 && lo <= hi && hi <= cap && (len < 0 ? hi == 0 : hi <= len));
  CHECK(hi == (len < 0 ? 0 : len < cap ? len : cap));
  CHECK(win ? hi - lo == (hi < win ? hi : win) : lo == 0);
  const int32_t from = si_span_origin(lo);
  CHECK(from % 8 == 0 && from <= lo && from > lo - 8 && (hi == lo) == (n == 0));
  if (n) CHECK(from + (int64_t)n * 128 >= hi && from + (int64_t)(n - 1) * 128 < hi);
  const int32_t big = si_span_hi(2147483647, 2147483647LL - 128);
  CHECK(si_span_tiles(0, big, 128) == 16777215 && big == 2147483519);
}

static void divisions(void) {
  const uint32_t d = rnd(40) ? (uint32_t)(1 + rnd(5000)) : (uint32_t)(1 + rnd(2147483647));
  const si_divisor v = si_make_divisor(d);
  for (int i = 0; i < 200; ++i) {
    uint32_t t = (uint32_t)rnd(2147483648u);
    if (i % 4 == 1) t = (uint32_t)(t / d * d);                    /* a multiple */
    if (i % 4 == 2) t = t >= d ? t / d * d - 1 : 0;              /* just below one */
    if (i == 3) t = 2147483647u;
    CHECK(si_divide(t, v) == t / d);
  }
}

static void dealing(int most) {
  enum { B = 40, PER = 12 };
  int32_t n[B];
  int64_t total = 0, start[B];
  const int batch = 1 + (int)rnd(B), per = 1 + (int)rnd(PER), big = 1 + (int)rnd(300);
  for (int b = 0; b < batch; ++b) {
    n[b] = rnd(4) ? (int32_t)rnd(big) : 0;
    start[b] = total;
    total += (int64_t)n[b] * per;
  }
  const int64_t parts = si_part_count(total, most);
  if (total == 0) return;
  char* taken = calloc((size_t)total, 1);
  int64_t* slot_item = malloc(sizeof(int64_t) * 2 * most);
  for (int i = 0; i < 2 * most; ++i) slot_item[i] = -1;
  char* whole_item = calloc((size_t)batch * per, 1);
  for (int64_t w = 0; w < parts; ++w) {
    int64_t f = si_part_begin(w, total, parts);
    const int64_t end = si_part_begin(w + 1, total, parts);
    CHECK(f < end && end <= total);
    int b = 0;
    while (f >= start[b] + (int64_t)n[b] * per) ++b;
    int item = (int)((f - start[b]) / n[b]);
    int32_t ta = (int32_t)((f - start[b]) % n[b]);
    for (;;) {
      CHECK(b < batch && n[b] > 0);
      const int32_t tb = ta + (end - f) < n[b] ? (int32_t)(ta + (end - f)) : n[b];
      for (int32_t t = ta; t < tb; ++t) {
        const int64_t g = start[b] + (int64_t)item * n[b] + t;
        CHECK(!taken[g] && si_part_of(g, total, parts) == w);
        taken[g] = 1;
      }
      if (ta == 0 && tb == n[b]) {
        whole_item[b * per + item] = 1;
      } else {
        const int64_t s = si_part_slot(w, ta > 0);
        CHECK(s >= 0 && s < 2 * most && slot_item[s] < 0);
        slot_item[s] = (int64_t)b * per + item;
      }
      f += tb - ta;
      if (f >= end) break;
      ta = 0;
      if (++item == per) {
        item = 0;
        do { ++b; CHECK(b < batch); } while (n[b] == 0);
      }
    }
  }
  for (int64_t g = 0; g < total; ++g) CHECK(taken[g]);
  for (int b = 0; b < batch; ++b)
    for (int item = 0; item < per && n[b]; ++item) {
      const int64_t f0 = start[b] + (int64_t)item * n[b];
      const int64_t w0 = si_part_of(f0, total, parts), w1 = si_part_of(f0 + n[b] - 1, total, parts);
      CHECK((w0 == w1) == whole_item[b * per + item]);
      if (w0 == w1) continue;
      for (int64_t w = w0; w <= w1; ++w) {
        const int64_t s = si_part_slot(w, si_part_begin(w, total, parts) > f0);
        CHECK(slot_item[s] == (int64_t)b * per + item);
        slot_item[s] = -1;
      }
    }
  for (int i = 0; i < 2 * most; ++i) CHECK(slot_item[i] < 0);
  free(taken); free(slot_item); free(whole_item);
}

int main(void) {
  long cases = 0;
  large_rows();
  for (int i = 0; i < 2000; ++i, ++cases) rows();
  for (int i = 0; i < 20000; ++i, ++cases) spans();
  for (int i = 0; i < 20000; ++i, ++cases) divisions();
  const int most[4] = {1, 7, 64, 512};
  for (int i = 0; i < 800; ++i, ++cases) dealing(most[i % 4]);
  printf("cases %ld\n", cases);
  return 0;
}
