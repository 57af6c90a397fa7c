// Attention of one new token of each sequence over a page pool.
//
//   s_t = scale <q, k_t>,  o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  m = max_t s_t
//
// for positions t of [lo, hi): the sequence's cached tokens, or the last `window`
// of them. Position t lies in page table[b][t / page_size]; the positions of a page
// outside the pool take no part. Every cached byte of the sequence's heads is read
// once, so HBM bounds long caches; the launches and one chain of loads short ones.
//
// Work. An item is (sequence, kv head, block of 16 query heads of its group); its
// positions are cut into tiles of 128, 32 for each of a block's four waves. All
// tiles of all items, in a row, are dealt evenly to a fixed number of workgroups
// (si_pool_index.h), whatever the lengths are: a workgroup finishes the items that
// lie inside its range, and leaves the maximum, sum and unnormalised output of the
// at most two that go over its edges in the workspace, where paged_join merges them.
// The lengths are read on the device, so a captured graph replays with new ones. Items
// of few tiles are finished by a block each instead, in one launch (dealt()).
//
// Measured, 32 query heads of 128, bf16: 131072 positions of 8 kv heads, int8 58 us (4.7
// TB/s of cache, 7.7 us more for the join), int4 54, bf16 106 (5.1 TB/s); 16 sequences of
// 8192 over 32 kv heads, int8 201 (5.15 TB/s); 64 uneven sequences up to 4096, int4 73: 32
// positions cost a wave about 580 VALU instructions, which keep a SIMD busy 80% of the
// time that its waves live. 100 positions: 6.5.
#include "si_pool_args.h"
#include "si_pool_index.h"
#include "si_kv_common.h"

namespace si {
namespace {

constexpr int kRows = 16;        // query heads of an item
constexpr int kWaveTokens = 32;
constexpr int kTile = 4 * kWaveTokens;  // of a dealt launch
constexpr int kCUs = 256;
constexpr int kMostParts = 4 * kCUs;  // workgroups of a dealt launch at most
constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;

// Weights of fp32's range are 2^-24 at most, so that the sum over 2^24 positions of the
// largest values does not overflow.
constexpr float kSpare = 24.0f;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const void* q;
  int64_t qs[2];            // elements between sequences and heads
  int qdt;
  const int32_t* table;
  int64_t ts;               // entries between sequences
  const int32_t* lens;
  int64_t capacity;         // positions of a table row
  int B, Hk, group, rb;     // rb: row blocks of a group
  int P, window, D, g;
  si_divisor by_page;       // divides by P
  int pages;
  float scale, scale_lo;    // times log2(e), and what fp32 leaves of that
  const void* pool[4];      // k, v, scale_k, scale_v
  int sdt;
  void* out;                // [B, Hk * group, D], q's type
  float* lse;               // [B, Hk * group] or NULL
  int most;                 // workgroups of a dealt launch
  float* parts;             // [2 * most][part_rows][D], then [2 * most][part_rows][2]
  int part_rows;
};

// Storage kinds of a pool.
enum { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3, kI4 = 4 };

// Tiles of sequence b's items, and the first of its positions.
__device__ __forceinline__ int span_tiles(const AttnArgs& a, int b, int32_t* lo, int32_t* hi, int tile = kTile) {
  *hi = si_span_hi(a.lens[b], a.capacity);
  *lo = si_span_lo(*hi, a.window);
  return si_span_tiles(*lo, *hi, tile);
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Memory that no kernel writes while this one runs, read through scalar loads.
__device__ __forceinline__ const __attribute__((address_space(4))) int32_t* scalar(const int32_t* p) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// v, computed again where it is used: what is derived from it is not kept in
// registers over a loop it does not change in.
__device__ __forceinline__ int afresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Sum over the block of v, and over the threads before this one.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int64_t* before) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int64_t s = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int64_t base = 0, total = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) base += lds[w];
    total += lds[w];
  }
  __syncthreads();
  *before = base + s - v;
  return uniform(total);
}

// A wave's running softmax over its positions: lane (c, kq) = (lane % 16, lane / 16)
// has query row c's maximum (the same in all four kq) and sum over the positions of
// its kq, and the output's values d = (4 kq + i) J + j in o[j][i], all relative to
// 2^m.
template <int J>
struct Running {
  float m, l;
  f32x4 o[J];
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The larger of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ __forceinline__ float max_over_kq(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float w = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(w), __float_as_uint(w), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// ---------------------------------------------------------------------------
// A wave's part of an item. A tile's scores are K times q transposed,
// [position][query row] (A holds 16 positions, B 16 query rows): a lane has the
// scores of its own query row at positions s * 16 + 4 kq + i. The weights are then
// in place as the second product's operand when its k runs over those positions,
// and the output is V transposed times the weights, [d][query row]. Nothing passes
// between lanes but the row maxima.
//
// FP32 (fp32 queries or fp32 rows): v_mfma_f32_16x16x4_f32 on values widened to fp32.
//
// Otherwise v_mfma_f32_16x16x32 on 16-bit operands, eight k per lane. What keeps
// this as exact as fp32 weights would be:
//  * int8 and int4 codes are exact in fp16 (0x6400 | u is 1024 + u); a row's int8
//    scale multiplies its score, and its value's scale the weight, in fp32;
//  * an int4 group's scale is split as 2^e (e from the row's largest group, in fp32
//    like an int8 scale) times s' < 2. n s' has 3 + 8 bits for a bf16 scale, so it is
//    exact in fp16; fp16 and fp32 scales are carried as two such parts (NS = 2);
//  * query rows are scaled by a power of two so that their largest value is in
//    [2^14, 2^15): bf16's 8 bits are then exact in fp16 over 2^32. fp16 queries over
//    bf16 rows are two bf16 parts (NQ = 2), again exact;
//  * weights w = exp(s - m) sv are two 16-bit parts, hi and what hi leaves. Their
//    reference m is the maximum of s + log2(sv), so the largest is 2^14 in fp16 whatever
//    the rows' scales are (2^-24 in bf16), and the parts hold a weight to 2^-22 (fp16,
//    down to 2^-38 of the largest) or 2^-16 (bf16).
// The k order within a chunk of eight is free as long as both operands have the
// same: int4's nibbles come out as 1 5 0 4 3 7 2 6.
//
// HBM bounds it: a wave has the next tile's keys in flight during the softmax and
// the second product, and its values during the first; rows and scales of a tile go
// through LDS.
// ---------------------------------------------------------------------------
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ uint32_t as_u32(h2 h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ h2 pair(float x) { return h2{(_Float16)x, (_Float16)x}; }

// Two nibbles of a word, at bits 0 and 16 (HIGH: 4 and 20), as fp16 values n - 8. The
// constants are kept in registers, where one v_and_or_b32 can take both.
template <bool HIGH>
__device__ __forceinline__ h2 nibbles(uint32_t u) {
  uint32_t mask = HIGH ? 0x00f000f0u : 0x000f000fu, base = 0x64006400u;
  asm("" : "+s"(mask));
  asm("" : "+v"(base));
  const h2 x = as_h2((u & mask) | base);  // 1024 + n, or 1024 + 16 n
  return HIGH ? __builtin_elementwise_fma(x, pair(0.0625f), pair(-72.0f)) : x - pair(1032.0f);
}

template <int WORDS>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (WORDS == 0) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);  // four int4 codes
  } else if constexpr (WORDS % 4 == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const u4 x = *reinterpret_cast<const u4*>(p + 4 * i);
      w[i] = x[0]; w[i + 1] = x[1]; w[i + 2] = x[2]; w[i + 3] = x[3];
    }
  } else if constexpr (WORDS == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    static_assert(WORDS == 1, "half a word, a word, two, or whole 16 bytes");
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// N stored values as fp32 (int4: without their scale).
template <int KIND, int N>
__device__ __forceinline__ void widen(const uint32_t* w, float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (KIND == kF32) x[i] = __uint_as_float(w[i]);
    else if constexpr (KIND == kBF16) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else if constexpr (KIND == kF16) x[i] = f16_bits_to_f32(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
    else if constexpr (KIND == kI8) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i & 3)));
    else x[i] = (float)((int)(w[i / 8] >> (8 * ((i & 7) / 2) + (i & 1 ? 0 : 4)) & 0xfu) - 8);  // high nibble first
  }
}

// EXACT: D == DP, and wider loads of K. EIGHTS: eight positions from a multiple of
// eight on lie in one page, so a tile's rows are four runs whose first ones are
// scalars; otherwise each lane finds one position's row and they go through LDS.
template <int KIND, int DP_, bool EXACT, bool EIGHTS, bool FP32, int NQ, int NS>
struct Engine {
  static constexpr int kKind = KIND;
  static constexpr int DP = DP_, J = DP / 16, M = DP / 32;
  // Blocks of a CU, for the registers' bound and the dealing. Two against three, us:
  // int4 88 / 77 (64 uneven sequences) and 58.7 / 54 (131072 positions); int8 64.4 / 65.8
  // and 197.5 / 203.8 (16 x 8192) at 128 wide, but 28.1 / 27.3 at 64, 54.8 / 50.6 at 80 and
  // 97.4 / 92.1 with fp32 queries; bf16 106.4 / 108.7. fp32 rows, one against two: 90 / 125.
  static constexpr int kBlocks = KIND == kF32 ? 1 : KIND == kI8 || (KIND == kI4 && !FP32) ? 3 : 2;
  static constexpr bool kBf = !FP32 && KIND == kBF16;
  static constexpr bool kScaled = KIND == kI8 || KIND == kI4;
  static constexpr int kG = FP32 ? 16 : 8;  // int4 groups of a row at most
  static constexpr float kRoom = FP32 || kBf ? -kSpare : 14.0f;  // weights are up to 2^kRoom
  // bits of a value; words of K per lane and 16 positions, of V per lane and position
  static constexpr int kBits = KIND == kI4 ? 4 : KIND == kI8 ? 8 : KIND == kF32 ? 32 : 16;
  static constexpr int kKW = DP / 4 * kBits / 32, kVW = J * kBits / 32;  // 0: half a word
  static constexpr int kVW1 = kVW ? kVW : 1;
  static constexpr int kUnit = 8 * kBits / 32;  // words of eight values

  // A wave's LDS: rows [32], then per position K's factor, V's and its logarithm, and int4's
  // scales as [32][kG] for K and [kG][32] for V, s' in NS fp16 parts each or
  // fp32.
  static constexpr int kLdsScale = 32 * 4;
  static constexpr int kLdsParts = kLdsScale + (kScaled ? 3 * 32 * 4 : 0);
  static constexpr int kLds = kLdsParts + (KIND == kI4 ? 2 * 32 * kG * (FP32 ? 4 : 2 * NS) : 0);

  uint32_t k[2][kKW], v[2][4][kVW1];  // a tile's rows
  uint32_t sc[KIND == kI4 ? (FP32 ? 16 : NS == 1 ? 4 : 8) : 1];
  int32_t row;    // of position lane % 32 (-1: takes no part)
  uint32_t live, next_live;  // bit 4 s + i: position s * 16 + 4 kq + i takes part
  bool full, next_full;      // all positions of the tile do
  int32_t t0, end;  // the wave's position, and where its tiles end
  // The next tile's table entries and the offsets in their pages: of position lane % 32,
  // or of the four eights. Then the first rows of the eights that are being loaded.
  int32_t page[EIGHTS ? 4 : 1], offset[EIGHTS ? 4 : 1], run[EIGHTS ? 4 : 1];

  Running<J> st;
  u4 q[NQ][M];
  float qf[FP32 ? M * 8 : 1];
  float qscale;  // what scores are multiplied by: scale * log2(e) / the row's power of two

  // The first d of chunk m.
  __device__ __forceinline__ static int chunk_d(int m, int kq) {
    if constexpr (EXACT && KIND == kI8) return (m >> 1) * 64 + kq * 16 + (m & 1) * 8;
    if constexpr (EXACT && KIND == kI4) return kq * (DP / 4) + m * 8;
    return (m * 4 + kq) * 8;
  }

  // The item's query rows, from the block's LDS.
  __device__ __forceinline__ void begin(const AttnArgs& a, const float (*rows)[DP + 4]) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    float x[M][8];
    float top = 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(&rows[c][chunk_d(m, kq)]);
      const f32x4 w = *reinterpret_cast<const f32x4*>(&rows[c][chunk_d(m, kq) + 4]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        constexpr int order[8] = {1, 5, 0, 4, 3, 7, 2, 6};
        const int n = KIND == kI4 && !FP32 ? order[e] : e;
        x[m][e] = n < 4 ? u[n & 3] : w[n & 3];
        top = fmaxf(top, fabsf(x[m][e]));
      }
    }
    qscale = a.scale;
    if constexpr (FP32) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[m * 8 + e] = x[m][e];
    } else if constexpr (!kBf) {
      top = max_over_kq(top);
      int up = 0;  // a power of two for the row
      if (top > 0.0f && top < INFINITY) up = 15 - __builtin_amdgcn_frexp_expf(top);
      qscale = __builtin_amdgcn_ldexpf(a.scale, -up);
#pragma unroll
      for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          q[0][m][e / 2] = as_u32(h2{(_Float16)__builtin_amdgcn_ldexpf(x[m][e], up),
                                     (_Float16)__builtin_amdgcn_ldexpf(x[m][e + 1], up)});
      }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t hi = f32x2_to_bf16x2_bits(x[m][e], x[m][e + 1]);
          q[0][m][e / 2] = hi;
          if constexpr (NQ == 2)
            q[1][m][e / 2] = f32x2_to_bf16x2_bits(x[m][e] - __uint_as_float(hi << 16),
                                                  x[m][e + 1] - __uint_as_float(hi & 0xffff0000u));
        }
      }
    }
  }

  // The page table entries of the tile at t.
  __device__ __forceinline__ void find_pages(const AttnArgs& a, int b, int32_t t, int32_t hi) {
    if constexpr (EIGHTS) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t u = t + 8 * g, p = si_divide(u, a.by_page);
        page[g] = (int32_t)u < hi ? scalar(a.table)[b * a.ts + p] : -1;
        offset[g] = (int32_t)(u - p * (uint32_t)a.P);
      }
    } else {
      const uint32_t u = t + (threadIdx.x & 31), p = si_divide(u, a.by_page);
      page[0] = (int32_t)u < hi ? a.table[b * a.ts + p] : -1;
      offset[0] = (int32_t)(u - p * (uint32_t)a.P);
    }
  }

  // The tile's rows, from its table entries.
  __device__ __forceinline__ void find_rows(const AttnArgs& a, int32_t* lds_rows, int hk, int32_t lo, int32_t hi) {
    const int lane = threadIdx.x & 63, kq = lane >> 4;
    const int32_t t = t0 + (lane & 31);
    if constexpr (EIGHTS) {
      bool all = t0 >= lo && t0 + kWaveTokens <= hi;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        run[g] = si_page_row(page[g], a.pages, hk, a.Hk, offset[g], a.P);
        all = all && run[g] >= 0;
      }
      if constexpr (kScaled) {
        // (copies: a choice between members would put them all into memory)
        int32_t r[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) r[g] = afresh(run[g]);
        const int32_t lower = lane & 8 ? r[1] : r[0], upper = lane & 8 ? r[3] : r[2], first = lane & 16 ? upper : lower;
        row = first >= 0 && t >= lo && t < hi ? first + (lane & 7) : -1;
      }
      next_full = all;
      next_live = 0xffu;
      if (!all) {
        next_live = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t u = t0 + s * 16 + kq * 4 + i;
            const bool there = kq & 2 ? run[2 * s + 1] >= 0 : run[2 * s] >= 0;
            if (there && u >= lo && u < hi) next_live |= 1u << (4 * s + i);
          }
        }
      }
    } else {
      row = t >= lo && t < hi
                ? si_page_row(page[0], a.pages, hk, a.Hk, offset[0], a.P) : -1;
      if (lane < 32) lds_rows[lane] = row;
      wave_sync();
      next_live = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int4 r4 = *reinterpret_cast<const int4*>(lds_rows + s * 16 + kq * 4);
        const int32_t r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r[i] >= 0) next_live |= 1u << (4 * s + i);
      }
      next_full = __all(next_live == 0xffu);
    }
  }

  static constexpr int kRowBytes = EXACT ? DP * kBits / 8 : 0;
  __device__ __forceinline__ static int64_t row_bytes(const AttnArgs& a) {
    return EXACT ? (int64_t)kRowBytes : (int64_t)a.D * kBits / 8;
  }
  // Bytes of run g from a tensor's start, for rows of n bytes; row 0 where there is none.
  __device__ __forceinline__ int64_t run_at(int g, int64_t n) const { return (int64_t)(run[g] < 0 ? 0 : run[g]) * n; }

  // Starts the loads of the keys and scales of the tile at t0. Positions that do not
  // take part read row 0, or one of the eight rows from their run's first on.
  __device__ __forceinline__ void start_keys(const AttnArgs& a, int32_t* lds_rows, int hk, int32_t lo, int32_t hi) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    find_rows(a, lds_rows, hk, lo, hi);
    const char* kp = reinterpret_cast<const char*>(a.pool[0]);
    const int64_t n = row_bytes(a);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p;
      if constexpr (EIGHTS) {
        p = (c < 8 ? kp + run_at(2 * s, n) : kp + run_at(2 * s + 1, n)) + (c & 7) * (int)n;
      } else {
        const int32_t r = lds_rows[s * 16 + c];
        p = kp + (r < 0 ? 0 : r) * n;
      }
      if constexpr (EXACT) {
        // 16 bytes a load: 64 bytes of a row by its four lanes
        if constexpr (kBits >= 16) {
#pragma unroll
          for (int m = 0; m < M; ++m) load_words<kUnit>(p + chunk_d(m, kq) * kBits / 8, k[s] + kUnit * m);
        } else if constexpr (kBits == 8) {
#pragma unroll
          for (int m = 0; m < M; m += 2) load_words<4>(p + chunk_d(m, kq), k[s] + 2 * m);
        } else {
          load_words<kKW>(p + chunk_d(0, kq) / 2, k[s]);
        }
      } else {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int d = chunk_d(m, kq);
          if (d < a.D) {
            load_words<kUnit>(p + d * kBits / 8, k[s] + kUnit * m);
          } else {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) k[s][kUnit * m + i] = KIND == kI4 ? 0x88888888u : 0u;
          }
        }
      }
    }
    if constexpr (kScaled) {  // K's scales in the lower lanes, V's in the upper
      const int64_t r = row < 0 ? 0 : row;
      const void* sp = a.pool[lane < 32 ? 2 : 3];
      if constexpr (KIND == kI8) {
        sc[0] = a.sdt == SI_DT_F32 ? reinterpret_cast<const uint32_t*>(sp)[r]
                                   : reinterpret_cast<const uint16_t*>(sp)[r];
      } else {
        const int G = a.D / a.g;
        if constexpr (!FP32 && NS == 1) {  // bf16
          if (G == 8) {
            load_words<4>(reinterpret_cast<const char*>(sp) + r * 16, sc);
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(sp) + r * G + 2 * w;
              const uint32_t lo16 = 2 * w < G ? h[0] : 0, hi16 = 2 * w + 1 < G ? h[1] : 0;
              sc[w] = lo16 | (hi16 << 16);
            }
          }
        } else {
#pragma unroll
          for (int w = 0; w < kG; ++w) sc[w] = w < G ? __float_as_uint(load_any(sp, a.sdt, r * G + w)) : 0;
        }
      }
    }
  }

  // Starts the loads of its values.
  __device__ __forceinline__ void start_values(const AttnArgs& a, const int32_t* lds_rows) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    const char* vp = reinterpret_cast<const char*>(a.pool[1]);
    const int64_t n = row_bytes(a);
    live = next_live;
    full = next_full;
    const bool in = EXACT || c * J < a.D;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p[4];
      if constexpr (EIGHTS) {
        p[0] = (kq & 2 ? vp + run_at(2 * s + 1, n) : vp + run_at(2 * s, n)) + (kq & 1) * 4 * (int)n + c * J * kBits / 8;
#pragma unroll
        for (int i = 1; i < 4; ++i) p[i] = p[0] + i * n;
      } else {
        const int4 r4 = *reinterpret_cast<const int4*>(lds_rows + s * 16 + kq * 4);
        const int32_t r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = vp + (r[i] < 0 ? 0 : r[i]) * n + c * J * kBits / 8;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (in) {
          load_words<kVW>(p[i], v[s][i]);
        } else {
#pragma unroll
          for (int w = 0; w < kVW1; ++w) v[s][i][w] = KIND == kI4 ? 0x88888888u : 0u;
        }
      }
    }
  }

  // The factors of the lane's own positions s * 16 + 4 kq + i (j: 0 K, 1 V): an int8 row's
  // scale, 2^e of an int4 row's, 0 for a position that takes no part. j 2: log2 of V's.
  __device__ __forceinline__ static f32x4 factors(const char* lds, int j, int s) {
    const int kq = (threadIdx.x & 63) >> 4;
    return *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + kLdsScale) + 32 * j + s * 16 + kq * 4);
  }

  // The tile's scales into the wave's LDS.
  __device__ __forceinline__ void place_scales(const AttnArgs& a, char* lds) const {
    const int lane = threadIdx.x & 63, t = lane & 31;
    float* factor = reinterpret_cast<float*>(lds + kLdsScale);  // [3][32]
    float f = 1.0f;
    if constexpr (KIND == kI8) {
      f = a.sdt == SI_DT_F32 ? __uint_as_float(sc[0])
          : a.sdt == SI_DT_BF16 ? bf16_bits_to_f32(sc[0]) : f16_bits_to_f32(sc[0]);
      if (row < 0) f = 0.0f;
    } else {
      float s[kG], top = 0.0f;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const uint32_t word = row < 0 ? 0u : sc[!FP32 && NS == 1 ? g / 2 : g];
        s[g] = __uint_as_float(FP32 || NS == 2 ? word : g & 1 ? word & 0xffff0000u : word << 16);
        top = fmaxf(top, s[g]);
      }
      if constexpr (FP32) {
        float* part = reinterpret_cast<float*>(lds + kLdsParts) + (lane < 32 ? 0 : 32 * kG);
#pragma unroll
        for (int g = 0; g < kG; ++g) part[lane < 32 ? t * kG + g : g * 32 + t] = s[g];
      } else {
        // s' = s / 2^e < 2; a row of infinities keeps e within fp32
        const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
        f = __builtin_amdgcn_ldexpf(1.0f, e);
        _Float16* part = reinterpret_cast<_Float16*>(lds + kLdsParts) + (lane < 32 ? 0 : NS * 32 * kG);
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const float r = __builtin_amdgcn_ldexpf(s[g], -e);
          const int at = lane < 32 ? t * kG + g : g * 32 + t;
          if constexpr (NS == 1) {
            part[at] = (_Float16)r;
          } else {
            const float hi = bf16_bits_to_f32(f32_to_bf16_bits(r));
            part[at] = (_Float16)hi;
            part[32 * kG + at] = (_Float16)(hi < INFINITY ? r - hi : 0.0f);
          }
        }
      }
    }
    factor[lane] = f;
    // (a factor below 2^-80 or not a number: its weight needs no more room than this)
    if (!FP32 && lane >= 32) factor[32 + lane] = f < INFINITY ? fmaxf(__builtin_amdgcn_logf(f), -80.0f) : -80.0f;
    wave_sync();
  }

  // Chunk m of K, positions s * 16 + c, as the first product's 16-bit operand.
  __device__ __forceinline__ u4 k_operand(int s, int m, h2 scale) const {
    if constexpr (kBits == 16) return u4{k[s][4 * m], k[s][4 * m + 1], k[s][4 * m + 2], k[s][4 * m + 3]};
    u4 r;
    if constexpr (KIND == kI8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t u = k[s][2 * m + i] ^ 0x80808080u;
        r[2 * i] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - pair(1152.0f));
        r[2 * i + 1] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - pair(1152.0f));
      }
    } else {
      const uint32_t u = k[s][m], w = u >> 8;
      r[0] = as_u32(nibbles<false>(u) * scale);
      r[1] = as_u32(nibbles<true>(u) * scale);
      r[2] = as_u32(nibbles<false>(w) * scale);
      r[3] = as_u32(nibbles<true>(w) * scale);
    }
    return r;
  }

  // Values kJG * i .. of two positions, paired: out[j] = (x's value, y's value).
  static constexpr int kJG = KIND == kI8 ? 4 : 2;
  __device__ __forceinline__ static void v_pairs(const uint32_t* x, const uint32_t* y, int i, uint32_t* out) {
    if constexpr (kBits == 16) {
      out[0] = __builtin_amdgcn_perm(y[i], x[i], 0x05040100u);
      out[1] = __builtin_amdgcn_perm(y[i], x[i], 0x07060302u);
    } else if constexpr (KIND == kI8) {
      const uint32_t lo = __builtin_amdgcn_perm(y[i], x[i], 0x05010400u) ^ 0x80808080u;
      const uint32_t hi = __builtin_amdgcn_perm(y[i], x[i], 0x07030602u) ^ 0x80808080u;
      out[0] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - pair(1152.0f));
      out[1] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - pair(1152.0f));
      out[2] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - pair(1152.0f));
      out[3] = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - pair(1152.0f));
    } else {  // byte i: values 2i (high nibble) and 2i + 1
      const uint32_t u = __builtin_amdgcn_perm(y[0], x[0], 0x0c040c00u + 0x00010001u * i);
      out[0] = as_u32(nibbles<true>(u));
      out[1] = as_u32(nibbles<false>(u));
    }
  }

  __device__ __forceinline__ static f32x4 mma(u4 x, u4 y, f32x4 z) {
    if constexpr (kBf)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), z, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), z, 0, 0, 0);
  }

  // The scores of the tile, without their factors.
  __device__ __forceinline__ void scores(const AttnArgs& a, char* lds, f32x4* acc) const {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    if constexpr (kScaled) place_scales(a, lds);
    acc[0] = acc[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int d = chunk_d(m, kq);
        const int g = KIND == kI4 && (EXACT || d < a.D) ? d / a.g : 0;
        if constexpr (FP32) {
          float x[8];
          widen<KIND, 8>(k[s] + kUnit * m, x);
          if constexpr (KIND == kI4) {
            const float f = reinterpret_cast<const float*>(lds + kLdsParts)[(s * 16 + c) * kG + g];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            acc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[m * 8 + e], acc[s], 0, 0, 0);
        } else {
#pragma unroll
          for (int p = 0; p < (KIND == kI4 ? NS : 1); ++p) {
            h2 ks = {};
            if constexpr (KIND == kI4) {
              const _Float16 f = reinterpret_cast<const _Float16*>(lds + kLdsParts)[(p * 32 + s * 16 + c) * kG + g];
              ks = h2{f, f};
            }
            const u4 ko = k_operand(s, m, ks);
#pragma unroll
            for (int n = 0; n < NQ; ++n) acc[s] = mma(ko, q[n][m], acc[s]);
          }
        }
      }
    }
  }

  // Its weights and their products with the values.
  __device__ __forceinline__ void values(const AttnArgs& a, const char* lds, const f32x4* acc) {
    float w[8], y[8], bound[8], top = st.m;
    f32x4 vf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 kf = {1.0f, 1.0f, 1.0f, 1.0f}, lg = {0.0f, 0.0f, 0.0f, 0.0f};
      vf[s] = kf;
      if constexpr (kScaled) {
        kf = factors(lds, 0, s);
        vf[s] = factors(lds, 1, s);
        if constexpr (!FP32) lg = factors(lds, 2, s);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = acc[s][i];
        if constexpr (FP32) {
          // the factor in two parts, so that the score is rounded once
          float f = a.scale, f_lo = a.scale_lo;
          if constexpr (KIND == kI8) {
            f = a.scale * kf[i];
            f_lo = __builtin_fmaf(a.scale, kf[i], -f) + a.scale_lo * kf[i];
          }
          x = __builtin_fmaf(x, f, x * f_lo);
        } else {
          x *= qscale;
          if constexpr (kScaled) x *= kf[i];
        }
        y[4 * s + i] = x;
        bound[4 * s + i] = lg[i];
      }
    }
    if (!full) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(live >> i & 1)) y[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, y[i] + bound[i]);
    top = max_over_kq(top);
    if (__any(top > st.m)) {
      const float keep = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - top);
      st.l *= keep;
#pragma unroll
      for (int j = 0; j < J; ++j) st.o[j] *= keep;
      st.m = top;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m - kRoom;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(y[4 * s + i] - ref);
        st.l += e;
        w[4 * s + i] = kScaled ? e * vf[s][i] : e;
      }
    }
    if constexpr (FP32) products32(a, lds, w);
    else products16(a, lds, w);
  }

  __device__ __forceinline__ void products32(const AttnArgs& a, const char* lds, const float* w) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    f32x4 vs[2] = {};
    if constexpr (KIND == kI4) {
      const int g = EXACT || c * J < a.D ? c * J / a.g : 0;
      const float* part = reinterpret_cast<const float*>(lds + kLdsParts) + 32 * kG + g * 32 + kq * 4;
      vs[0] = *reinterpret_cast<const f32x4*>(part);
      vs[1] = *reinterpret_cast<const f32x4*>(part + 16);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[J];
        widen<KIND, J>(v[s][i], x);
        // rows that take no part count as zeros, whatever they hold
        const bool dead = !kScaled && !full && !(live >> (4 * s + i) & 1);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if constexpr (KIND == kI4) x[j] *= vs[s][i];
          if (dead) x[j] = 0.0f;
          st.o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], w[4 * s + i], st.o[j], 0, 0, 0);
        }
      }
    }
  }

  __device__ __forceinline__ void products16(const AttnArgs& a, const char* lds, const float* w) {
    const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
    u4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = w[2 * i], y = w[2 * i + 1];
      // The bits that lo completes are the operand's own: left to itself the compiler
      // takes them from e * sv rounded once, which differs where the product's fp32
      // rounding lies halfway between two fp16 values.
      uint32_t h = kBf ? f32x2_to_bf16x2_bits(x, y) : as_u32(h2{(_Float16)x, (_Float16)y});
      asm("" : "+v"(h));
      hi[i] = h;
      if constexpr (kBf)
        lo[i] = f32x2_to_bf16x2_bits(x - __uint_as_float(h << 16), y - __uint_as_float(h & 0xffff0000u));
      else
        lo[i] = as_u32(h2{(_Float16)(x - (float)as_h2(h).x), (_Float16)(y - (float)as_h2(h).y)});
    }
    uint2 vs[NS][2];
    if constexpr (KIND == kI4) {
      const int g = EXACT || c * J < a.D ? c * J / a.g : 0;
      const _Float16* part = reinterpret_cast<const _Float16*>(lds + kLdsParts) + NS * 32 * kG + g * 32 + kq * 4;
#pragma unroll
      for (int p = 0; p < NS; ++p)
#pragma unroll
        for (int s = 0; s < 2; ++s) vs[p][s] = *reinterpret_cast<const uint2*>(part + p * 32 * kG + s * 16);
    }
#pragma unroll
    for (int i = 0; i < J / kJG; ++i) {
      uint32_t vv[4][kJG];  // [pair of positions][value]
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        v_pairs(v[t >> 1][2 * (t & 1)], v[t >> 1][2 * (t & 1) + 1], i, vv[t]);
        if constexpr (!kScaled) {
          // rows that take no part count as zeros, whatever they hold
          if (!full) {
            const uint32_t mask = (live >> (2 * t) & 1 ? 0xffffu : 0u) | (live >> (2 * t + 1) & 1 ? 0xffff0000u : 0u);
#pragma unroll
            for (int j = 0; j < kJG; ++j) vv[t][j] &= mask;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kJG; ++j) {
        f32x4& o = st.o[i * kJG + j];
        if constexpr (KIND == kI4) {
#pragma unroll
          for (int p = 0; p < NS; ++p) {
            const u4 vo = {as_u32(as_h2(vv[0][j]) * as_h2(vs[p][0].x)), as_u32(as_h2(vv[1][j]) * as_h2(vs[p][0].y)),
                           as_u32(as_h2(vv[2][j]) * as_h2(vs[p][1].x)), as_u32(as_h2(vv[3][j]) * as_h2(vs[p][1].y))};
            o = mma(vo, hi, o);
            o = mma(vo, lo, o);
          }
        } else {
          const u4 vo = {vv[0][j], vv[1][j], vv[2][j], vv[3][j]};
          o = mma(vo, hi, o);
          o = mma(vo, lo, o);
        }
      }
    }
  }

  // The loads of the wave's first tile of the block's [ta, tb), tiles of STEP positions.
  template <int STEP>
  __device__ __forceinline__ void start(const AttnArgs& a, char* lds, int b, int hk, int32_t lo, int32_t hi,
                                        int32_t ta, int32_t tb) {
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) st.o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int32_t from = si_span_origin(lo);
    t0 = from + ta * STEP + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kWaveTokens;
    end = tb * (int64_t)STEP + from < hi ? from + tb * STEP : hi;
    if (t0 >= end) return;
    int32_t* rows = reinterpret_cast<int32_t*>(lds);
    find_pages(a, b, t0, hi);
    start_keys(a, rows, hk, lo, hi);
    start_values(a, rows);
    find_pages(a, b, t0 + STEP, hi);
  }

  // All its tiles. A tile's keys are loaded over the last one's once its scores are
  // done, its values once its products are.
  template <int STEP>
  __device__ __forceinline__ void walk(const AttnArgs& a, char* lds, int b, int hk, int32_t lo, int32_t hi) {
    if (t0 >= end) return;
    int32_t* rows = reinterpret_cast<int32_t*>(lds);
    f32x4 acc[2];
    while (true) {
      scores(a, lds, acc);
      t0 += STEP;
      const bool more = t0 < end;
      if (more) {
        start_keys(a, rows, hk, lo, hi);
        find_pages(a, b, t0 + STEP, hi);
      }
      values(a, lds, acc);
      if (!more) break;
      start_values(a, rows);
    }
    st.m -= kRoom;  // the sums are of weights scaled by 2^kRoom
  }
};

// The maximum and sum of partial row i (slot * part_rows + row) at 2 i.
__device__ __forceinline__ float* part_sums(const AttnArgs& a) {
  return a.parts + (int64_t)2 * a.most * a.part_rows * a.D;
}

// DEALT: tiles dealt evenly to a.most blocks of four waves, partial results in a.parts.
// Otherwise block = item, which its W waves finish.
template <class E, bool DEALT, int W>
__global__ __launch_bounds__(64 * W, W == 4 ? E::kBlocks : 1) void paged_attn(AttnArgs a) {
  static_assert(W == 4 || (W == 8 && !DEALT), "four waves, or eight over a whole item");
  constexpr int DP = E::DP, kThreads = 64 * W, QN = kRows * DP / kThreads, kStep = W * kWaveTokens;
  constexpr int J = DP / 16;
  // the waves' outputs; before, the query rows (in the first) and the waves' own memory
  constexpr int kOut = kRows * (DP + 4) * (int)sizeof(float);
  __shared__ __attribute__((aligned(16))) char lds[kOut + ((W - 1) * kOut > W * E::kLds ? (W - 1) * kOut : W * E::kLds)];
  float (*lds_o)[kRows][DP + 4] = reinterpret_cast<float (*)[kRows][DP + 4]>(lds);
  __shared__ float lds_m[W][kRows], lds_l[W][kRows];
  __shared__ int64_t lds_scan[8];
  const int tid = threadIdx.x;
  const int per = a.Hk * a.rb;  // items of a sequence
  char* mine = lds + kOut + (tid >> 6) * E::kLds;

  // this block's tiles [f, end) in the row of all tiles, and where f lies
  int64_t f = 0, end = 0;
  int b = 0, item = 0;
  int32_t ta = 0, lo, hi;
  if (DEALT) {
    int64_t tiles = 0;
    if (tid == 0) lds_scan[4] = -1;
    const int chunk = (a.B + 255) / 256;
    const int b0 = tid * chunk, b1 = b0 + chunk < a.B ? b0 + chunk : a.B;
    for (int i = b0; i < b1; ++i) tiles += (int64_t)span_tiles(a, i, &lo, &hi) * per;
    int64_t before;
    const int64_t total = block_scan(tiles, lds_scan, &before);
    const int64_t parts = si_part_count(total, a.most);
    if (blockIdx.x >= parts) return;
    f = si_part_begin(blockIdx.x, total, parts);
    end = si_part_begin(blockIdx.x + 1, total, parts);
    if (f >= before && f < before + tiles) {
      int64_t at = before;
      for (int i = b0; i < b1; ++i) {
        const int n = span_tiles(a, i, &lo, &hi);
        if (f < at + (int64_t)n * per) {
          lds_scan[4] = i;
          lds_scan[5] = (f - at) / n;
          lds_scan[6] = (f - at) % n;
          break;
        }
        at += (int64_t)n * per;
      }
    }
    __syncthreads();
    b = (int)uniform(lds_scan[4]);
    item = (int)uniform(lds_scan[5]);
    ta = (int32_t)uniform(lds_scan[6]);
    if (b < 0) return;  // only if the lengths change while the kernel runs
  } else {
    b = blockIdx.x / per;
    item = blockIdx.x - b * per;
  }

  while (true) {
    const int n = span_tiles(a, b, &lo, &hi, kStep);
    const int32_t tb = !DEALT ? n : (int32_t)(ta + (end - f) < n ? ta + (end - f) : n);
    const int hk = item / a.rb, rb = item - hk * a.rb;
    const int rows = a.group - rb * kRows < kRows ? a.group - rb * kRows : kRows;
    const int64_t head0 = (int64_t)hk * a.group + rb * kRows;

    // the item's query rows in fp32 with zeros behind them, and the first rows' loads
    float q[QN];
    const int t0 = afresh(tid);
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const int x = t0 + kThreads * i, r = x / DP, d = x - r * DP;
      q[i] = r < rows && d < a.D ? load_any(a.q, a.qdt, b * a.qs[0] + (head0 + r) * a.qs[1] + d) : 0.0f;
    }
    E e;
    e.template start<kStep>(a, mine, b, hk, lo, hi, ta, tb);
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const int x = t0 + kThreads * i;
      lds_o[0][x / DP][x % DP] = q[i];
    }
    __syncthreads();
    e.begin(a, lds_o[0]);
    e.template walk<kStep>(a, mine, b, hk, lo, hi);

    // the waves' results together
    const int t1 = afresh(tid), lane = t1 & 63, wave = t1 >> 6, c = lane & 15, kq = lane >> 4;
    Running<J>& st = e.st;
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
    __syncthreads();  // the query rows and the waves' own memory are free
    if (kq == 0) {
      lds_m[wave][c] = st.m;
      lds_l[wave][c] = st.l;
    }
    if (c < rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) lds_o[wave][c][(kq * 4 + i) * J + j] = st.o[j][i];
    }
    __syncthreads();
    const bool whole = ta == 0 && tb == n;
    const int64_t slot = DEALT ? si_part_slot(blockIdx.x, ta > 0) : 0;
    for (int x = t1; x < rows * DP; x += kThreads) {
      const int r = x / DP, d = x - r * DP;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, lds_m[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, val = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float k = __builtin_amdgcn_exp2f(lds_m[w][r] - ref);
        sum += lds_l[w][r] * k;
        val += lds_o[w][r][d] * k;
      }
      if (d >= a.D) continue;
      if (whole) {
        const int64_t o = (int64_t)b * a.Hk * a.group + head0 + r;
        store_any(a.out, a.qdt, o * a.D + d, sum == 0.0f ? 0.0f : val / sum);
        if (d == 0 && a.lse) a.lse[o] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
      } else {
        const int64_t at = slot * a.part_rows + r;
        a.parts[at * a.D + d] = val;
        if (d == 0) *reinterpret_cast<float2*>(part_sums(a) + 2 * at) = make_float2(top, sum);
      }
    }
    if (!DEALT) return;
    f += tb - ta;
    if (f >= end) return;
    __syncthreads();  // the results have been read
    ta = 0;
    if (++item == per) {
      item = 0;
      do {  // f < end: a sequence with tiles follows (unless the lengths change meanwhile)
        if (++b >= a.B) return;
      } while (span_tiles(a, b, &lo, &hi) == 0);
    }
  }
}

// Joins the partial results of items that several blocks worked on, and gives the
// items without positions their zeros. Block (x, y): row y of item x. The maxima
// and sums of all parts come first, in one round of loads; then D / 4 threads take
// four values each of every (1024 / D)-th part.
__global__ __launch_bounds__(256) void paged_join(AttnArgs a) {
  __shared__ float weight[kMostParts];
  __shared__ f32x4 lds_o[256];
  __shared__ float red[8];
  const int tid = threadIdx.x;
  const int per = a.Hk * a.rb;
  const int b = blockIdx.x / per, item = blockIdx.x - b * per;
  const int hk = item / a.rb, rb = item - hk * a.rb;
  const int r = blockIdx.y;
  if (r >= a.group - rb * kRows) return;
  // all tiles, and those before sequence b: every wave adds them up for itself
  int64_t total = 0, before = 0;
  int32_t lo, hi;
  for (int i = tid & 63; i < a.B; i += 64) {
    const int64_t t = (int64_t)span_tiles(a, i, &lo, &hi) * per;
    total += t;
    if (i < b) before += t;
  }
  for (int x = 1; x < 64; x <<= 1) {
    total += __shfl_xor(total, x, 64);
    before += __shfl_xor(before, x, 64);
  }
  const int n = span_tiles(a, b, &lo, &hi);
  const int64_t head = (int64_t)hk * a.group + rb * kRows + r;
  const int64_t o = (int64_t)b * a.Hk * a.group + head;
  if (n == 0) {
    if (tid < a.D) store_any(a.out, a.qdt, o * a.D + tid, 0.0f);
    if (tid == 0 && a.lse) a.lse[o] = -INFINITY;
    return;
  }
  const int64_t f0 = before + (int64_t)item * n, parts = si_part_count(total, a.most);
  const int64_t w0 = si_part_of(f0, total, parts);
  const int count = (int)(si_part_of(f0 + n - 1, total, parts) - w0) + 1;
  if (count == 1) return;  // its block finished it
  // of every part: its slot is 2 w but for the first, whose block began with the item or before
  const bool inside = si_part_begin(w0, total, parts) > f0;
  auto row = [&](int i) { return si_part_slot(w0 + i, i > 0 || inside) * a.part_rows + r; };
  float m[kMostParts / 256], l[kMostParts / 256], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMostParts / 256; ++i) {
    const int w = tid + 256 * i;
    m[i] = -INFINITY;
    l[i] = 0.0f;
    if (w < count) {
      const float2 x = *reinterpret_cast<const float2*>(part_sums(a) + 2 * row(w));
      m[i] = x.x;
      l[i] = x.y;
    }
    top = fmaxf(top, m[i]);
  }
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kMostParts / 256; ++i) {
    const float k = __builtin_amdgcn_exp2f(m[i] - ref);
    weight[tid + 256 * i] = k;
    sum += l[i] * k;
  }
  for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
  __syncthreads();
  sum = (red[4] + red[5]) + (red[6] + red[7]);
  const int width = a.D / 4, lanes = 256 / width;  // lanes: parts at a time
  const int d4 = tid % width, g = tid / width;
  f32x4 val = {0.0f, 0.0f, 0.0f, 0.0f};
  if (g < lanes) {
#pragma unroll 4
    for (int w = g; w < count; w += lanes)
      val += *reinterpret_cast<const f32x4*>(a.parts + row(w) * a.D + 4 * d4) * weight[w];
  }
  lds_o[tid] = val;
  __syncthreads();
  if (tid < width) {
    for (int i = 1; i < lanes; ++i) val += lds_o[tid + i * width];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      store_any(a.out, a.qdt, o * a.D + 4 * tid + j, sum == 0.0f ? 0.0f : val[j] / sum);
    if (tid == 0 && a.lse) a.lse[o] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
}

// Any head size and group: block = (sequence, query head), a thread a position of
// the scores, then a thread a value (two at most: D <= 512) of the output.
__global__ __launch_bounds__(256) void paged_attn_any(AttnArgs a, int kind) {
  __shared__ float q[512], p[256];
  __shared__ int32_t rows[256];
  __shared__ float red[8];
  const int heads = a.Hk * a.group, tid = threadIdx.x;
  const int b = blockIdx.x / heads, h = blockIdx.x - b * heads, hk = h / a.group;
  int32_t lo, hi;
  span_tiles(a, b, &lo, &hi);
  for (int d = tid; d < a.D; d += 256) q[d] = load_any(a.q, a.qdt, b * a.qs[0] + h * a.qs[1] + d);
  auto value = [&](int j, int32_t row, int d) -> float {
    const int64_t el = (int64_t)row * a.D + d;
    if (kind == kI8) return (float)reinterpret_cast<const int8_t*>(a.pool[j])[el] * load_any(a.pool[2 + j], a.sdt, row);
    if (kind == kI4) {
      const uint32_t w = reinterpret_cast<const uint8_t*>(a.pool[j])[(int64_t)row * ((a.D + 1) / 2) + d / 2];
      const int nib = (d & 1) ? (int)(w & 0xfu) : (int)(w >> 4);
      return (float)(nib - 8) * load_any(a.pool[2 + j], a.sdt, (int64_t)row * (a.D / a.g) + d / a.g);
    }
    return load_any(a.pool[j], kind == kF32 ? SI_DT_F32 : kind == kF16 ? SI_DT_F16 : SI_DT_BF16, el);
  };
  float top = -INFINITY, sum = 0.0f, o[2] = {0.0f, 0.0f};
  for (int32_t t0 = lo; t0 < hi; t0 += 256) {
    __syncthreads();  // q is there; the previous positions have been used
    const int32_t t = t0 + tid;
    int32_t row = -1;
    if (t < hi) {
      const uint32_t pg = (uint32_t)t / (uint32_t)a.P;
      row = si_page_row(a.table[b * a.ts + pg], a.pages, hk, a.Hk, t - (int32_t)pg * a.P, a.P);
    }
    float s = -INFINITY;
    if (row >= 0) {
      s = 0.0f;
      for (int d = 0; d < a.D; ++d) s = __builtin_fmaf(value(0, row, d), q[d], s);
      s *= a.scale;
    }
    float m = s;
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    const float up = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), top);
    const float ref = up == -INFINITY ? 0.0f : up + kSpare;
    const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up);
    top = up;
    const float w = __builtin_amdgcn_exp2f(s - ref);
    p[tid] = w;
    rows[tid] = row;
    float l = w;
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x, 64);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
    __syncthreads();
    sum = sum * keep + (red[4] + red[5]) + (red[6] + red[7]);
    const int count = hi - t0 < 256 ? hi - t0 : 256;
    for (int e = 0; e < 2; ++e) {
      const int d = tid + e * 256;
      if (d >= a.D) break;
      float x = o[e] * keep;
      for (int i = 0; i < count; ++i)
        if (rows[i] >= 0) x = __builtin_fmaf(p[i], value(1, rows[i], d), x);
      o[e] = x;
    }
  }
  const int64_t out = (int64_t)b * heads + h;
  for (int e = 0; e < 2; ++e) {
    const int d = tid + e * 256;
    if (d < a.D) store_any(a.out, a.qdt, out * a.D + d, sum == 0.0f ? 0.0f : o[e] / sum);
  }
  if (tid == 0 && a.lse) a.lse[out] = sum == 0.0f ? -INFINITY : (top + kSpare + log2f(sum)) * kLn2;
}

// Whether items' tiles are dealt (and joined), by the most tiles one can have: whole
// items take about 2 us for 256 positions (eight waves), dealt ones a second launch and
// its chain. Measured with 32 query and 8 kv heads over int8 rows, whole against dealt,
// us: 1 sequence (8 items) of 600 positions 10.5 / 13.4, 800 12.5 / 13.3, 1000 14.4 /
// 13.3; 8 of 1000 15.9 / 16.7, 1600 21.1 / 19.2; 24 of 1600 22.3 / 29.9, 2400 30.1 / 33.4;
// 64 of 2400 64.7 / 64.8.
bool dealt(int64_t items, int64_t capacity, int64_t window) {
  const int64_t most = window > 0 && window < capacity ? window : capacity;
  const int64_t limit = 6 + items / 16;
  return most > (limit < 20 ? limit : 20) * kTile;
}

template <class E>
int launch(AttnArgs a, bool deal, hipStream_t st) {
  const int64_t items = (int64_t)a.B * a.Hk * a.rb;
  if (deal) {
    a.most = E::kBlocks * kCUs;
    paged_attn<E, true, 4><<<a.most, 256, 0, st>>>(a);
    const int rows = a.group < kRows ? a.group : kRows;
    paged_join<<<dim3((unsigned)items, (unsigned)rows), 256, 0, st>>>(a);
  } else if (items <= kCUs && a.capacity > kTile && (a.window == 0 || a.window > kTile)) {
    // eight waves where there is work for them and a CU has one item at most: 1000 positions of 24 x 8 items 16.9
    // us for 21.1 with four, of 64 x 8 items 34.2 for 30.1
    paged_attn<E, false, 8><<<(unsigned)items, 512, 0, st>>>(a);
  } else {
    paged_attn<E, false, 4><<<(unsigned)items, 256, 0, st>>>(a);
  }
  return check_launch("si_paged_attn");
}

template <int KIND, bool EIGHTS, bool FP32, int NQ, int NS>
int launch_size(const AttnArgs& a, bool deal, hipStream_t st) {
  if (a.D == 64) return launch<Engine<KIND, 64, true, EIGHTS, FP32, NQ, NS>>(a, deal, st);
  if (a.D == 128) return launch<Engine<KIND, 128, true, EIGHTS, FP32, NQ, NS>>(a, deal, st);
  return a.D < 64 ? launch<Engine<KIND, 64, false, EIGHTS, FP32, NQ, NS>>(a, deal, st)
                  : launch<Engine<KIND, 128, false, EIGHTS, FP32, NQ, NS>>(a, deal, st);
}

template <int KIND, bool FP32, int NQ, int NS>
int launch_pages(const AttnArgs& a, bool deal, hipStream_t st) {
  return a.P % 8 == 0 ? launch_size<KIND, true, FP32, NQ, NS>(a, deal, st)
                      : launch_size<KIND, false, FP32, NQ, NS>(a, deal, st);
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" size_t si_paged_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t heads, int64_t D,
                                                int64_t capacity, int64_t window) {
  if (heads <= 0 || Hq % heads != 0 || D <= 0 || D > 128 || D % 8 != 0) return 0;
  const int64_t group = Hq / heads, rows = group < kRows ? group : kRows;
  if (!dealt(B * heads * ceil_div(group, kRows), capacity, window)) return 0;
  return (size_t)(2 * kMostParts * rows * (D + 2)) * sizeof(float);
}

extern "C" int si_paged_attn(const si_page_pool* pool, const void* q, int q_dtype, int64_t B, int64_t Hq,
                             int64_t q_stride_b, int64_t q_stride_h, const int32_t* table,
                             int64_t table_stride, int64_t table_width, const int32_t* lengths,
                             int64_t window, double scale, void* out, float* lse, void* workspace,
                             size_t workspace_bytes, si_stream_t stream) {
  clear_error();
  const int rc = check_pool("si_paged_attn", pool);
  if (rc != SI_OK) return rc;
  const si_page_pool& p = *pool;
  SI_CHECK_ARG(dtype_ok(q_dtype), "si_paged_attn: unsupported dtype %d", q_dtype);
  SI_CHECK_ARG(B >= 0 && Hq > 0 && Hq < 65536 && Hq % p.heads == 0 && B < ((int64_t)1 << 31) / Hq,
               "si_paged_attn: bad shape");
  SI_CHECK_ARG(table_width >= 0 && table_width <= (((int64_t)1 << 31) - 1 - 2 * kTile) / p.page_size,
               "si_paged_attn: page tables reach fewer than 2^31 positions");
  SI_CHECK_ARG(window >= 0 && window < ((int64_t)1 << 31), "si_paged_attn: bad window");
  if (B == 0) return SI_OK;
  SI_CHECK_ARG(q && (table || table_width == 0) && lengths && out, "si_paged_attn: NULL argument");
  AttnArgs a = {};
  a.q = q;
  a.qs[0] = q_stride_b;
  a.qs[1] = q_stride_h;
  a.qdt = q_dtype;
  a.table = table;
  a.ts = table_stride;
  a.lens = lengths;
  a.capacity = table_width * p.page_size;
  a.B = (int)B;
  a.Hk = (int)p.heads;
  a.group = (int)(Hq / p.heads);
  a.rb = (int)ceil_div(a.group, kRows);
  a.P = (int)p.page_size;
  a.by_page = si_make_divisor((uint32_t)p.page_size);
  a.window = (int)window;
  a.D = (int)p.D;
  a.g = (int)p.group;
  a.pages = (int)p.pages;
  a.scale = (float)(scale * kLog2e);
  a.scale_lo = (float)(scale * kLog2e - a.scale);
  a.pool[0] = p.k;
  a.pool[1] = p.v;
  a.pool[2] = p.scale_k;
  a.pool[3] = p.scale_v;
  a.sdt = (int)p.dtype;
  a.out = out;
  a.lse = lse;
  a.part_rows = a.group < kRows ? a.group : kRows;
  const int kind = p.precision == SI_PREC_FP32 ? (p.dtype == SI_DT_F32 ? kF32 : p.dtype == SI_DT_F16 ? kF16 : kBF16)
                   : p.precision == SI_PREC_FP16 ? kF16 : p.precision == SI_PREC_INT8 ? kI8 : kI4;
  hipStream_t st = as_stream(stream);
  // chunks of eight values of a row, in one int4 group
  const bool tiles = a.D <= 128 && a.D % 8 == 0 && (kind != kI4 || a.g % 8 == 0);
  if (!tiles) {
    paged_attn_any<<<(unsigned)(B * Hq), 256, 0, st>>>(a, kind);
    return check_launch("si_paged_attn/any");
  }
  const bool deal = dealt(B * p.heads * a.rb, a.capacity, window);
  if (deal) {
    const size_t need = si_paged_attn_workspace_bytes(B, Hq, p.heads, a.D, a.capacity, window);
    SI_CHECK_ARG(workspace && workspace_bytes >= need, "si_paged_attn: workspace of %zu bytes needed, got %zu",
                 need, workspace ? workspace_bytes : (size_t)0);
    SI_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "si_paged_attn: workspace not 16-byte aligned");
    a.parts = reinterpret_cast<float*>(workspace);
  }
  if (q_dtype != SI_DT_F32) {
    if (kind == kF16) return launch_pages<kF16, false, 1, 1>(a, deal, st);
    if (kind == kBF16)
      return q_dtype == SI_DT_BF16 ? launch_pages<kBF16, false, 1, 1>(a, deal, st)
                                   : launch_pages<kBF16, false, 2, 1>(a, deal, st);
    if (kind == kI8) return launch_pages<kI8, false, 1, 1>(a, deal, st);
    if (kind == kI4 && a.D / a.g <= 8)
      return a.sdt == SI_DT_BF16 ? launch_pages<kI4, false, 1, 1>(a, deal, st)
                                 : launch_pages<kI4, false, 1, 2>(a, deal, st);
  }
  switch (kind) {
    case kF32: return launch_pages<kF32, true, 1, 1>(a, deal, st);
    case kF16: return launch_pages<kF16, true, 1, 1>(a, deal, st);
    case kBF16: return launch_pages<kBF16, true, 1, 1>(a, deal, st);
    case kI8: return launch_pages<kI8, true, 1, 1>(a, deal, st);
    default: return launch_pages<kI4, true, 1, 1>(a, deal, st);
  }
}
