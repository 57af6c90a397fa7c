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
// The lengths are read on the device, so a captured graph replays with new ones.
#include "si_pool_index.h"
#include "si_kv_common.h"

namespace si {
namespace {

constexpr int kRows = 16;        // query heads of an item
constexpr int kWaveTokens = 32;
constexpr int kTile = 4 * kWaveTokens;
constexpr int kParts = 512;      // workgroups of a dealt launch: two per CU
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
  int64_t pages;
  float scale;              // times log2(e)
  const void* pool[4];      // k, v, scale_k, scale_v
  int sdt;
  void* out;                // [B, Hk * group, D], q's type
  float* lse;               // [B, Hk * group] or NULL
  float* parts;             // [2 * kParts][rows][D + 2], or NULL: one block per item
  int part_rows;
};

// Storage kinds of a pool.
enum { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3, kI4 = 4 };

// N values from element el on of a row, widened to fp32 (int4: without their scale).
template <int KIND, int N>
__device__ __forceinline__ void load_row(const void* p, int64_t el, float* x) {
  if constexpr (KIND == kF32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + el + i);
      x[i] = w.x; x[i + 1] = w.y; x[i + 2] = w.z; x[i + 3] = w.w;
    }
  } else if constexpr (KIND == kF16 || KIND == kBF16) {
    uint32_t w[N / 2];
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p) + el;
    if constexpr (N == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(s);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(s);
      w[0] = u.x; w[1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (KIND == kBF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        x[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
        x[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
      }
    }
  } else if constexpr (KIND == kI8) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const int8_t*>(p) + el + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = (float)(int8_t)(w >> (8 * j));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint32_t w = *reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(p) + (el + i) / 2);
      x[i] = (float)((int)((w >> 4) & 0xfu) - 8);
      x[i + 1] = (float)((int)(w & 0xfu) - 8);
      x[i + 2] = (float)((int)((w >> 12) & 0xfu) - 8);
      x[i + 3] = (float)((int)((w >> 8) & 0xfu) - 8);
    }
  }
}

// Tiles of sequence b's items, and the first of its positions.
__device__ __forceinline__ int span_tiles(const AttnArgs& a, int b, int32_t* lo, int32_t* hi) {
  *hi = si_span_hi(a.lens[b], a.capacity);
  *lo = si_span_lo(*hi, a.window);
  return si_span_tiles(*lo, *hi, kTile);
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
  return total;
}

// A wave's running softmax over its positions: lane (r, kq) = (lane % 16, lane / 16)
// has query row r's maximum and sum over the positions of its kq, and the
// output's values d = (4 kq + i) J + j in o[j][i].
template <int J>
struct Running {
  float m, l;
  f32x4 o[J];
};

// Products in fp32 (v_mfma_f32_16x16x4_f32): A holds one k of 16 rows, so the
// scores are K times q transposed, [position][query row], and a lane has the
// scores of its own row at positions s * 16 + 4 kq + i. The probabilities are then
// in place as the second product's operand when its k runs over kq, and the
// output is V transposed times P, [d][query row]. Nothing passes between lanes
// but the row maxima.
template <int KIND, int DP>
__device__ __forceinline__ void wave_tile(const AttnArgs& a, const float* q, int b, int hk, int32_t t0,
                                          int32_t hi, Running<DP / 16>& st) {
  constexpr int J = DP / 16, M = DP / 32;
  const int lane = threadIdx.x & 63, c = lane & 15, kq = lane >> 4;
  // row of position t0 + lane % 32, and its scales (K's in the lower lanes, V's above)
  const int32_t t = t0 + (lane & 31);
  int32_t row = -1;
  if (t < hi) {
    const uint32_t pg = (uint32_t)t / (uint32_t)a.P;
    row = si_page_row(a.table[b * a.ts + pg], a.pages, hk, a.Hk, t - (int32_t)pg * a.P, a.P);
  }
  float sc = 0.0f;
  if (KIND == kI8 && row >= 0) sc = load_any(a.pool[lane < 32 ? 2 : 3], a.sdt, row);
  const int G = KIND == kI4 ? a.D / a.g : 1;
  f32x4 acc[2] = {};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int32_t kr = __shfl(row, s * 16 + c, 64);
    const int64_t base = (int64_t)(kr < 0 ? 0 : kr);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int d = (m * 4 + kq) * 8;
      float x[8] = {};
      if (d < a.D) {
        load_row<KIND, 8>(a.pool[0], base * a.D + d, x);
        if constexpr (KIND == kI4) {
          const float ks = load_any(a.pool[2], a.sdt, base * G + d / a.g);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= ks;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        acc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], q[m * 8 + e], acc[s], 0, 0, 0);
    }
  }
  int32_t vr[2][4];
  float p[2][4], top = st.m;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vr[s][i] = __shfl(row, s * 16 + kq * 4 + i, 64);
      float x = acc[s][i] * a.scale;
      if constexpr (KIND == kI8) x *= __shfl(sc, s * 16 + kq * 4 + i, 64);
      p[s][i] = vr[s][i] < 0 ? -INFINITY : x;
      top = fmaxf(top, p[s][i]);
    }
  }
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const float ref = top == -INFINITY ? 0.0f : top;  // nothing yet: every weight below is 0
  const float keep = __builtin_amdgcn_exp2f(st.m - ref);
  st.m = top;
  st.l *= keep;
#pragma unroll
  for (int j = 0; j < J; ++j) st.o[j] *= keep;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool live = vr[s][i] >= 0;
      float w = __builtin_amdgcn_exp2f(p[s][i] - ref);
      st.l += w;
      if constexpr (KIND == kI8) {
        const float vs = __shfl(sc, 32 + s * 16 + kq * 4 + i, 64);
        w *= vs;
      }
      const int64_t base = live ? vr[s][i] : 0;
      const int d = c * J;
      float x[J] = {};
      if (live && d < a.D) {  // rows that take no part count as zeros, whatever they hold
        load_row<KIND, J>(a.pool[1], base * a.D + d, x);
        if constexpr (KIND == kI4) {
          const float vs = load_any(a.pool[3], a.sdt, base * G + d / a.g);
#pragma unroll
          for (int j = 0; j < J; ++j) x[j] *= vs;
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
        st.o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], w, st.o[j], 0, 0, 0);
    }
  }
}

// DEALT: tiles dealt evenly to kParts blocks, partial results in a.parts. Otherwise
// block = item, which it finishes.
template <int KIND, int DP, bool DEALT>
__global__ __launch_bounds__(256, 2) void paged_attn(AttnArgs a) {
  constexpr int J = DP / 16, M = DP / 32;
  __shared__ float lds_o[4][kRows][DP + 4];
  __shared__ float lds_m[4][kRows], lds_l[4][kRows];
  __shared__ int64_t lds_scan[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 15, kq = lane >> 4;
  const int per = a.Hk * a.rb;  // items of a sequence

  // this block's tiles [f, end) in the row of all tiles, and where f lies
  int64_t f = 0, end = 0, total = 0;
  int b = 0, item = 0;
  int32_t ta = 0;
  if (DEALT) {
    int64_t mine = 0;
    const int chunk = (a.B + 255) / 256;
    const int b0 = tid * chunk, b1 = b0 + chunk < a.B ? b0 + chunk : a.B;
    int32_t lo, hi;
    for (int i = b0; i < b1; ++i) mine += (int64_t)span_tiles(a, i, &lo, &hi) * per;
    int64_t before;
    total = block_scan(mine, lds_scan, &before);
    const int64_t parts = si_part_count(total, kParts);
    if (blockIdx.x >= parts) return;
    f = si_part_begin(blockIdx.x, total, parts);
    end = si_part_begin(blockIdx.x + 1, total, parts);
    if (f >= before && f < before + mine) {
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
    b = (int)lds_scan[4];
    item = (int)lds_scan[5];
    ta = (int32_t)lds_scan[6];
  } else {
    b = blockIdx.x / per;
    item = blockIdx.x - b * per;
  }

  while (true) {
    int32_t lo, hi;
    const int n = span_tiles(a, b, &lo, &hi);
    const int32_t tb = !DEALT ? n : (int32_t)(ta + (end - f) < n ? ta + (end - f) : n);
    const int hk = item / a.rb, rb = item - hk * a.rb;
    const int rows = a.group - rb * kRows < kRows ? a.group - rb * kRows : kRows;
    const int64_t head0 = (int64_t)hk * a.group + rb * kRows;

    Running<J> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) st.o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float q[M * 8];
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = (m * 4 + kq) * 8 + e;
        q[m * 8 + e] = c < rows && d < a.D
                           ? load_any(a.q, a.qdt, b * a.qs[0] + (head0 + c) * a.qs[1] + d) : 0.0f;
      }
    }
    for (int32_t i = ta; i < tb; ++i) {
      const int32_t t0 = lo + i * kTile + wave * kWaveTokens;
      if (t0 < hi) wave_tile<KIND, DP>(a, q, b, hk, t0, hi, st);
    }

    // the four waves' results together
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
    __syncthreads();  // the previous item's results have been read
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
    for (int x = tid; x < rows * DP; x += 256) {
      const int r = x / DP, d = x - r * DP;
      float top = -INFINITY;
      for (int w = 0; w < 4; ++w) top = fmaxf(top, lds_m[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, val = 0.0f;
      for (int w = 0; w < 4; ++w) {
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
        float* part = a.parts + (slot * a.part_rows + r) * (a.D + 2);
        part[d] = val;
        if (d == 0) {
          part[a.D] = top;
          part[a.D + 1] = sum;
        }
      }
    }
    if (!DEALT) return;
    f += tb - ta;
    if (f >= end) return;
    ta = 0;
    if (++item == per) {
      item = 0;
      do { ++b; } while (span_tiles(a, b, &lo, &hi) == 0);  // f < end: one with tiles follows
    }
  }
}

// Joins the partial results of items that several blocks worked on, and gives the
// items without positions their zeros. Block (x, y): row y of item x, a thread a value.
__global__ __launch_bounds__(256) void paged_join(AttnArgs a) {
  __shared__ int64_t lds_scan[8];
  const int per = a.Hk * a.rb;
  const int b = blockIdx.x / per, item = blockIdx.x - b * per;
  const int hk = item / a.rb, rb = item - hk * a.rb;
  const int r = blockIdx.y;
  int64_t total_mine = 0, before_mine = 0;
  int32_t lo, hi;
  for (int i = threadIdx.x; i < a.B; i += blockDim.x) {
    const int64_t n = (int64_t)span_tiles(a, i, &lo, &hi) * per;
    total_mine += n;
    if (i < b) before_mine += n;
  }
  int64_t unused;
  const int64_t total = block_scan(total_mine, lds_scan, &unused);
  const int64_t before = block_scan(before_mine, lds_scan, &unused);
  if (r >= a.group - rb * kRows) return;
  const int n = span_tiles(a, b, &lo, &hi);
  const int64_t head = (int64_t)hk * a.group + rb * kRows + r;
  const int64_t o = (int64_t)b * a.Hk * a.group + head;
  const int d = threadIdx.x;
  if (n == 0) {
    if (d < a.D) store_any(a.out, a.qdt, o * a.D + d, 0.0f);
    if (d == 0 && a.lse) a.lse[o] = -INFINITY;
    return;
  }
  const int64_t f0 = before + (int64_t)item * n, parts = si_part_count(total, kParts);
  const int64_t w0 = si_part_of(f0, total, parts), w1 = si_part_of(f0 + n - 1, total, parts);
  if (w0 == w1) return;  // its block finished it
  float top = -INFINITY, sum = 0.0f, val = 0.0f;
  for (int64_t w = w0; w <= w1; ++w) {
    const bool inside = si_part_begin(w, total, parts) > f0;
    const float* part = a.parts + (si_part_slot(w, inside) * a.part_rows + r) * (a.D + 2);
    const float m = part[a.D], l = part[a.D + 1], x = d < a.D ? part[d] : 0.0f;
    const float up = fmaxf(top, m), ref = up == -INFINITY ? 0.0f : up;
    const float k0 = __builtin_amdgcn_exp2f(top - ref), k1 = __builtin_amdgcn_exp2f(m - ref);
    sum = sum * k0 + l * k1;
    val = val * k0 + x * k1;
    top = up;
  }
  if (d < a.D) store_any(a.out, a.qdt, o * a.D + d, sum == 0.0f ? 0.0f : val / sum);
  if (d == 0 && a.lse) a.lse[o] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
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
    const float ref = up == -INFINITY ? 0.0f : up;
    const float keep = __builtin_amdgcn_exp2f(top - ref);
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
  if (tid == 0 && a.lse) a.lse[out] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Whether an item's tiles are dealt (and joined): never where no item has more than
// one tile.
bool dealt(int64_t capacity, int64_t window) {
  const int64_t most = window > 0 && window < capacity ? window : capacity;
  return most > kTile;
}

template <int KIND, int DP>
int launch(const AttnArgs& a, bool deal, hipStream_t st) {
  const int64_t items = (int64_t)a.B * a.Hk * a.rb;
  if (deal) {
    paged_attn<KIND, DP, true><<<kParts, 256, 0, st>>>(a);
    const int rows = a.group < kRows ? a.group : kRows;
    paged_join<<<dim3((unsigned)items, (unsigned)rows), a.D <= 64 ? 64 : 128, 0, st>>>(a);
  } else {
    paged_attn<KIND, DP, false><<<(unsigned)items, 256, 0, st>>>(a);
  }
  return check_launch("si_paged_attn");
}

template <int KIND>
int launch_kind(const AttnArgs& a, bool deal, hipStream_t st) {
  return a.D <= 64 ? launch<KIND, 64>(a, deal, st) : launch<KIND, 128>(a, deal, st);
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" size_t si_paged_attn_workspace_bytes(int64_t Hq, int64_t Hk, int64_t D, int64_t capacity,
                                                int64_t window) {
  if (Hk <= 0 || Hq % Hk != 0 || D <= 0 || D > 128 || D % 8 != 0 || !dealt(capacity, window)) return 0;
  const int64_t group = Hq / Hk, rows = group < kRows ? group : kRows;
  return (size_t)(2 * kParts * rows * (D + 2)) * sizeof(float);
}

extern "C" int si_paged_attn(const void* q, int q_dtype, int64_t B, int64_t Hq, int64_t q_stride_b,
                             int64_t q_stride_h, int64_t Hk, int64_t D, const int32_t* table,
                             int64_t table_stride, int64_t table_width, const int32_t* lengths,
                             int64_t window, float scale, int64_t pages, int64_t page_size,
                             int precision, int dtype, int64_t group, void* const* pool, void* out,
                             float* lse, void* workspace, size_t workspace_bytes, si_stream_t stream) {
  clear_error();
  SI_CHECK_ARG(dtype_ok(q_dtype) && dtype_ok(dtype), "si_paged_attn: unsupported dtype");
  SI_CHECK_ARG(precision >= SI_PREC_FP32 && precision <= SI_PREC_INT4,
               "si_paged_attn: precision %d is not 0..3", precision);
  SI_CHECK_ARG(B >= 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && Hq < 65536 && D > 0 && D <= 512 &&
               B * Hq < ((int64_t)1 << 31), "si_paged_attn: bad shape");
  SI_CHECK_ARG(pages > 0 && page_size > 0 && pages < ((int64_t)1 << 31) && page_size < ((int64_t)1 << 31) &&
               pages <= (((int64_t)1 << 31) - 1) / Hk / page_size,
               "si_paged_attn: pools hold fewer than 2^31 rows");
  SI_CHECK_ARG(table_width >= 0 && table_width <= (((int64_t)1 << 31) - 1 - kTile) / page_size,
               "si_paged_attn: page tables reach fewer than 2^31 positions");
  SI_CHECK_ARG(window >= 0 && window < ((int64_t)1 << 31), "si_paged_attn: bad window");
  SI_CHECK_ARG(group > 0 && D % group == 0, "si_paged_attn: group must divide D");
  if (B == 0) return SI_OK;
  SI_CHECK_ARG(q && (table || table_width == 0) && lengths && pool && pool[0] && pool[1] && out,
               "si_paged_attn: NULL argument");
  SI_CHECK_ARG(precision < SI_PREC_INT8 || (pool[2] && pool[3]), "si_paged_attn: NULL scales");
  AttnArgs a = {};
  a.q = q;
  a.qs[0] = q_stride_b;
  a.qs[1] = q_stride_h;
  a.qdt = q_dtype;
  a.table = table;
  a.ts = table_stride;
  a.lens = lengths;
  a.capacity = table_width * page_size;
  a.B = (int)B;
  a.Hk = (int)Hk;
  a.group = (int)(Hq / Hk);
  a.rb = (int)ceil_div(a.group, kRows);
  a.P = (int)page_size;
  a.window = (int)window;
  a.D = (int)D;
  a.g = (int)group;
  a.pages = pages;
  a.scale = scale * kLog2e;
  uintptr_t bits = 0;
  for (int j = 0; j < 4; ++j) {
    a.pool[j] = pool[j];
    if (j < 2) bits |= reinterpret_cast<uintptr_t>(pool[j]);
  }
  a.sdt = dtype;
  a.out = out;
  a.lse = lse;
  a.part_rows = a.group < kRows ? a.group : kRows;
  const int kind = precision == SI_PREC_FP32 ? (dtype == SI_DT_F32 ? kF32 : dtype == SI_DT_F16 ? kF16 : kBF16)
                   : precision == SI_PREC_FP16 ? kF16 : precision == SI_PREC_INT8 ? kI8 : kI4;
  hipStream_t st = as_stream(stream);
  // chunks of eight values of a row, in one int4 group
  const bool tiles = D <= 128 && D % 8 == 0 && (bits & 15) == 0 && (kind != kI4 || group % 8 == 0);
  if (!tiles) {
    paged_attn_any<<<(unsigned)(B * Hq), 256, 0, st>>>(a, kind);
    return check_launch("si_paged_attn/any");
  }
  const bool deal = dealt(a.capacity, window);
  if (deal) {
    const size_t need = si_paged_attn_workspace_bytes(Hq, Hk, D, a.capacity, window);
    SI_CHECK_ARG(workspace && workspace_bytes >= need, "si_paged_attn: workspace of %zu bytes needed, got %zu",
                 need, workspace ? workspace_bytes : (size_t)0);
    a.parts = reinterpret_cast<float*>(workspace);
  }
  switch (kind) {
    case kF32: return launch_kind<kF32>(a, deal, st);
    case kF16: return launch_kind<kF16>(a, deal, st);
    case kBF16: return launch_kind<kBF16>(a, deal, st);
    case kI8: return launch_kind<kI8>(a, deal, st);
    default: return launch_kind<kI4>(a, deal, st);
  }
}
