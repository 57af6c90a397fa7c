// Page pool of many sequences (KVPagePool): rows quantized into slots as they are
// written, and read back.
//
// A pool holds one precision in tensors [pages, heads, page_size, ...], the row
// format of the paged store: the input's values ("fp32"), fp16, int8 with a scale
// per row, or int4 with a scale per group. A slot is page * page_size + offset;
// K and V of token t go to (come from) row (page, head, offset) of every head. A
// slot outside the pool is skipped when written and gives zeros when read.
//
// Both kernels move every byte once and are bound by HBM, at few tokens by the
// launch and one chain of loads (64 tokens x 8 heads: 3.8 and 3.9 us).
#include "si_pool_args.h"
#include "si_pool_index.h"
#include "si_rotate.h"
#include "si_row_quant.h"

namespace si {
namespace {

struct PoolArgs {
  const char* k;          // rows in (write)
  const char* v;
  char* ko;               // rows out (read), [T, heads, D]
  char* vo;
  int64_t ks[2], vs[2];   // elements between tokens and heads
  const int64_t* slots;
  int64_t T;
  int pages, H, P, D, g, prec;
  int sdt, odt;           // pool type; output type (read)
  int lpg, nl;            // lanes of an int4 group and of a row
  Buckets pool;           // the pool's tensors in the slots of `prec`
  Rotation rot;           // of K (write)
  int64_t pos_stride;
};

// ---------------------------------------------------------------------------
// Write
// ---------------------------------------------------------------------------

// 16 bytes of a row of dtype DT as fp32 values, and back.
template <int DT>
__device__ __forceinline__ void widen(const uint32_t w[4], float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == SI_DT_F32) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == SI_DT_BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      x[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
      x[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
    }
  }
}

// The chunk of a K row at d0 turned: its pairs' other values are pairs away
// (half), so a lane loads that chunk too, or lie in the chunk (interleaved).
// Rounded to the row's type, as rotating first and writing then would.
template <int DT>
__device__ __forceinline__ void rotate_chunk(const char* row, uint32_t w[4], int d0,
                                             const Rotation& r, const float2* cs) {
  constexpr int EPL = Chunk<DT>::EPL;
  constexpr int ES = DT == SI_DT_F32 ? 4 : 2;
  if (d0 >= 2 * r.pairs) return;
  float x[EPL];
  widen<DT>(w, x);
  if (r.interleaved) {
#pragma unroll
    for (int e = 0; e < EPL; e += 2) rotate_pair(cs[(d0 + e) / 2], x[e], x[e + 1]);
  } else {
    const bool first = d0 < r.pairs;
    const int p0 = first ? d0 : d0 - r.pairs;
    const uint4 o4 = *reinterpret_cast<const uint4*>(row + (first ? d0 + r.pairs : p0) * ES);
    const uint32_t o[4] = {o4.x, o4.y, o4.z, o4.w};
    float y[EPL];
    widen<DT>(o, y);
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (first) {
        rotate_pair(cs[p0 + e], x[e], y[e]);
      } else {
        rotate_pair(cs[p0 + e], y[e], x[e]);
      }
    }
  }
  copy_words<DT>(x, w);
}

// 16 bytes of a row of K and V: LPR lanes hold a row, nl of them values.
struct RowWords {
  uint32_t k[4], v[4];
};

template <int DT>
__device__ __forceinline__ void load_row(const PoolArgs& a, int64_t t, int h, int lane, RowWords& w) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  constexpr int ES = DT == SI_DT_F32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) w.k[i] = w.v[i] = 0;
  if (lane >= a.nl) return;
  const u32x4 k = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(a.k + (t * a.ks[0] + h * a.ks[1]) * ES + lane * 16));
  const u32x4 v = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(a.v + (t * a.vs[0] + h * a.vs[1]) * ES + lane * 16));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w.k[i] = k[i];
    w.v[i] = v[i];
  }
}

template <int DT, int LPR>
__device__ __forceinline__ void write_row(const PoolArgs& a, int lane, int32_t row, const RowWords& w) {
  constexpr int EPL = Chunk<DT>::EPL;
  constexpr int ES = DT == SI_DT_F32 ? 4 : 2;
  if (a.prec == SI_PREC_FP32) {  // the input's own type
    if (lane >= a.nl) return;
    const int64_t o = ((int64_t)row * a.D + lane * EPL) * ES;
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(a.pool.p[0]) + o) =
        make_uint4(w.k[0], w.k[1], w.k[2], w.k[3]);
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(a.pool.p[1]) + o) =
        make_uint4(w.v[0], w.v[1], w.v[2], w.v[3]);
    return;
  }
  if constexpr (DT == SI_DT_BF16) {
    pack_row_bf16<LPR, false>(w.k, w.v, a.prec, row, 0, 1, lane, a.lpg, a.pool, nullptr, nullptr, 0, a.nl);
  } else {
    float xk[EPL], xv[EPL];
    widen<DT>(w.k, xk);
    widen<DT>(w.v, xv);
    pack_row<DT, LPR, false>(xk, xv, a.prec, row, 0, 1, lane, a.lpg, a.pool, nullptr, nullptr, a.nl);
  }
}

// Block = RPP consecutive tokens of one head (neighbouring heads in neighbouring
// blocks), so rows that share a cache line of the pool are written together. The rows
// are loaded beside their slots, non-temporal: written and read back, 8192 x 32 rows of
// 128 bf16 take 76 us as int4 (78 with plain loads), 74 as int8 (81) and 94 unquantized
// (109), 4.6 to 5.7 TB/s; two rows a thread took 75.7, 75 and 96.
template <int DT, int LPR>
__global__ __launch_bounds__(256) void pool_write(PoolArgs a) {
  constexpr int RPP = 256 / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t tile = blockIdx.x / a.H;
  const int h = (int)(blockIdx.x - tile * a.H);
  const int64_t t = tile * RPP + threadIdx.x / LPR;
  if (t >= a.T) return;
  RowWords w;
  load_row<DT>(a, t, h, lane, w);
  const int32_t row = si_slot_row(a.slots[t], a.pages, h, a.H, a.P);
  if (row >= 0) write_row<DT, LPR>(a, lane, row, w);
}

// With a rotation: block = `tb` tokens and all their heads, whose cosines it
// computes once (2048 tokens x 8 heads of 128 bf16: 7.4 us for 16.8 MB).
template <int DT, int LPR>
__global__ __launch_bounds__(256) void pool_write_rotated(PoolArgs a, int tb) {
  constexpr int RPP = 256 / LPR;
  extern __shared__ float2 cs[];  // [tb][pairs]
  const int lane = threadIdx.x % LPR;
  const int64_t t0 = (int64_t)blockIdx.x * tb;
  const int nt = (int)(a.T - t0 < tb ? a.T - t0 : tb);
  for (int i = threadIdx.x; i < nt * a.rot.pairs; i += 256) {
    const int t = i / a.rot.pairs;
    cs[i] = pair_cos_sin(a.rot, (t0 + t) * a.pos_stride, i - t * a.rot.pairs);
  }
  __syncthreads();
  constexpr int ES = DT == SI_DT_F32 ? 4 : 2;
  for (int r = threadIdx.x / LPR; r < nt * a.H; r += RPP) {
    const int j = r / a.H, h = r - j * a.H;
    RowWords w;
    load_row<DT>(a, t0 + j, h, lane, w);
    const int32_t row = si_slot_row(a.slots[t0 + j], a.pages, h, a.H, a.P);
    if (row < 0) continue;
    if (lane < a.nl)
      rotate_chunk<DT>(a.k + ((t0 + j) * a.ks[0] + h * a.ks[1]) * ES, w.k, lane * Chunk<DT>::EPL, a.rot,
                       cs + j * a.rot.pairs);
    write_row<DT, LPR>(a, lane, row, w);
  }
}

// Any head size, group and alignment: a thread per row of K or V.
template <int DT>
__global__ __launch_bounds__(256) void pool_write_any(PoolArgs a, bool rotated) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rows = a.T * a.H;
  if (i >= 2 * rows) return;
  const int j = i >= rows;  // 0 k, 1 v
  const int64_t r = i - j * rows, t = r / a.H;
  const int h = (int)(r - t * a.H);
  const int32_t row = si_slot_row(a.slots[t], a.pages, h, a.H, a.P);
  if (row < 0) return;
  const char* src = j ? a.v : a.k;
  const int64_t el = j ? t * a.vs[0] + h * a.vs[1] : t * a.ks[0] + h * a.ks[1];
  const bool turn = rotated && j == 0;
  const int R = 2 * a.rot.pairs;
  auto value = [&](int d) {
    const float x = load_any(src, DT, el + d);
    if (!turn || d >= R) return x;
    const int half = a.rot.pairs;
    const int p = a.rot.interleaved ? d / 2 : d < half ? d : d - half;
    const bool first = a.rot.interleaved ? (d & 1) == 0 : d < half;
    const int od = a.rot.interleaved ? d ^ 1 : first ? d + half : d - half;
    const float y = load_any(src, DT, el + od);
    const float2 cs = pair_cos_sin(a.rot, t * a.pos_stride, p);
    float u = first ? x : y, w = first ? y : x;
    rotate_pair(cs, u, w);
    return round_to(first ? u : w, DT);
  };
  void* data = a.pool.p[4 * a.prec + j];
  if (a.prec == SI_PREC_FP32 || a.prec == SI_PREC_FP16) {
    for (int d = 0; d < a.D; ++d)
      store_any(data, a.prec == SI_PREC_FP16 ? SI_DT_F16 : DT, (int64_t)row * a.D + d, value(d));
    return;
  }
  const bool i8 = a.prec == SI_PREC_INT8;
  const int gs = i8 ? a.D : a.g, G = a.D / gs;
  const int64_t rb = (a.D + 1) / 2;
  uint32_t pending = 0;
  for (int g0 = 0; g0 < a.D; g0 += gs) {
    float m = 0.0f;
    for (int d = 0; d < gs; ++d) m = amax_fold(m, value(g0 + d));
    const float sc = quant_scale<DT>(m, i8 ? 127.0f : 7.0f);
    store_scalar<DT>(a.pool.p[4 * a.prec + 2 + j], (int64_t)row * G + g0 / gs, sc);
    for (int d = g0; d < g0 + gs; ++d) {
      const float q = clampf(quant_quotient<DT>(value(d), sc, 0.0f, false), i8 ? -128.0f : -8.0f,
                             i8 ? 127.0f : 7.0f);
      if (i8) {
        reinterpret_cast<int8_t*>(data)[(int64_t)row * a.D + d] = (int8_t)(int)q;
      } else {
        const uint32_t nib = (uint32_t)((int)q + 8) & 0xfu;
        if ((d & 1) == 0) pending = nib << 4;
        else reinterpret_cast<uint8_t*>(data)[row * rb + d / 2] = (uint8_t)(pending | nib);
      }
    }
  }
  if (!i8 && (a.D & 1)) reinterpret_cast<uint8_t*>(data)[row * rb + a.D / 2] = (uint8_t)pending;
}

// ---------------------------------------------------------------------------
// Read
// ---------------------------------------------------------------------------

// Eight values from d0 on of a pool row.
__device__ __forceinline__ void read8(const PoolArgs& a, int j, int32_t row, int d0, float* x) {
  const char* data = reinterpret_cast<const char*>(a.pool.p[4 * a.prec + j]);
  const void* scale = a.pool.p[4 * a.prec + 2 + j];
  const int64_t el = (int64_t)row * a.D + d0;
  if (a.prec == SI_PREC_INT8) {
    const uint2 w = *reinterpret_cast<const uint2*>(data + el);
    const float s = load_any(scale, a.sdt, row);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = (float)(int8_t)(w.x >> (8 * i)) * s;
      x[4 + i] = (float)(int8_t)(w.y >> (8 * i)) * s;
    }
  } else if (a.prec == SI_PREC_INT4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(data + (int64_t)row * (a.D / 2) + d0 / 2);
    const float s = load_any(scale, a.sdt, (int64_t)row * (a.D / a.g) + d0 / a.g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = (float)((int)((w >> (8 * i + 4)) & 0xfu) - 8) * s;
      x[2 * i + 1] = (float)((int)((w >> (8 * i)) & 0xfu) - 8) * s;
    }
  } else if (a.prec == SI_PREC_FP32 && a.sdt == SI_DT_F32) {
    const float4 u = *reinterpret_cast<const float4*>(data + el * 4);
    const float4 w = *reinterpret_cast<const float4*>(data + el * 4 + 16);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(data + el * 2);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (a.prec == SI_PREC_FP16 || a.sdt == SI_DT_F16) widen<SI_DT_F16>(w, x);
    else widen<SI_DT_BF16>(w, x);
  }
}

template <int ODT>
__device__ __forceinline__ void store8(char* p, const float* x) {
  if constexpr (ODT == SI_DT_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 16) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
    copy_words<ODT>(x, w);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Block = 256 / 2^lsh consecutive tokens of one head; eight values a thread. 8192 x 32
// int4 rows of 128 to bf16: 36.7 us, 4.8 TB/s.
template <int ODT>
__global__ __launch_bounds__(256) void pool_read(PoolArgs a, int lsh) {
  constexpr int ES = ODT == SI_DT_F32 ? 4 : 2;
  const int lane = threadIdx.x & ((1 << lsh) - 1);
  const int64_t tile = blockIdx.x / a.H;
  const int h = (int)(blockIdx.x - tile * a.H);
  const int64_t t = tile * (256 >> lsh) + (threadIdx.x >> lsh);
  if (t >= a.T || lane * 8 >= a.D) return;
  const int32_t row = si_slot_row(a.slots[t], a.pages, h, a.H, a.P);
  float xk[8] = {}, xv[8] = {};
  if (row >= 0) {
    read8(a, 0, row, lane * 8, xk);
    read8(a, 1, row, lane * 8, xv);
  }
  const int64_t o = ((t * a.H + h) * a.D + lane * 8) * ES;
  store8<ODT>(a.ko + o, xk);
  store8<ODT>(a.vo + o, xv);
}

// Any head size and group: a thread per value of K and V.
__global__ __launch_bounds__(256) void pool_read_any(PoolArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.T * a.H * a.D) return;
  const int64_t r = i / a.D, t = r / a.H;
  const int d = (int)(i - r * a.D), h = (int)(r - t * a.H);
  const int32_t row = si_slot_row(a.slots[t], a.pages, h, a.H, a.P);
  for (int j = 0; j < 2; ++j) {
    float x = 0.0f;
    const void* data = a.pool.p[4 * a.prec + j];
    const void* scale = a.pool.p[4 * a.prec + 2 + j];
    if (row >= 0) {
      const int64_t el = (int64_t)row * a.D + d;
      if (a.prec == SI_PREC_FP32) {
        x = load_any(data, a.sdt, el);
      } else if (a.prec == SI_PREC_FP16) {
        x = load_any(data, SI_DT_F16, el);
      } else if (a.prec == SI_PREC_INT8) {
        x = (float)reinterpret_cast<const int8_t*>(data)[el] * load_any(scale, a.sdt, row);
      } else {
        const uint32_t b = reinterpret_cast<const uint8_t*>(data)[(int64_t)row * ((a.D + 1) / 2) + d / 2];
        const int nib = (d & 1) ? (int)(b & 0xfu) : (int)(b >> 4);
        x = (float)(nib - 8) * load_any(scale, a.sdt, (int64_t)row * (a.D / a.g) + d / a.g);
      }
    }
    store_any(j ? a.vo : a.ko, a.odt, i, x);
  }
}

int check_rows(const char* what, const si_page_pool* p, int64_t T, const int64_t* slots) {
  const int rc = check_pool(what, p);
  if (rc != SI_OK) return rc;
  SI_CHECK_ARG(T >= 0 && T < ((int64_t)1 << 31) / p->heads, "%s: bad row count", what);
  SI_CHECK_ARG(slots || T == 0, "%s: NULL slots", what);
  return SI_OK;
}

PoolArgs pool_args(const si_page_pool& p, int64_t T, const int64_t* slots) {
  PoolArgs a = {};
  a.T = T;
  a.H = (int)p.heads;
  a.D = (int)p.D;
  a.pages = (int)p.pages;
  a.P = (int)p.page_size;
  a.prec = (int)p.precision;
  a.g = (int)p.group;
  a.sdt = (int)p.dtype;
  a.slots = slots;
  void* const t[4] = {p.k, p.v, p.scale_k, p.scale_v};
  for (int j = 0; j < 4; ++j) a.pool.p[4 * a.prec + j] = t[j];
  return a;
}

bool aligned16(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

template <int DT, int LPR>
void launch_write(const PoolArgs& a, bool rotated, hipStream_t st) {
  constexpr int RPP = 256 / LPR;
  if (rotated) {
    int tb = (int)ceil_div(RPP, a.H);
    while (tb > 1 && tb * a.rot.pairs > 4096) --tb;
    pool_write_rotated<DT, LPR><<<(unsigned)ceil_div(a.T, tb), 256, sizeof(float2) * tb * a.rot.pairs, st>>>(a, tb);
  } else {
    pool_write<DT, LPR><<<(unsigned)(ceil_div(a.T, RPP) * a.H), 256, 0, st>>>(a);
  }
}

template <int DT>
int write_rows(PoolArgs& a, bool rotated, hipStream_t st) {
  constexpr int EPL = Chunk<DT>::EPL;
  const bool whole = (a.ks[0] | a.ks[1] | a.vs[0] | a.vs[1] | a.D) % EPL == 0 && aligned16(a.k, a.v);
  int lpr = 8;
  while (lpr * EPL < a.D) lpr *= 2;
  // int4 groups of a power of two of lanes, or the whole row
  a.nl = a.D / EPL;
  a.lpg = a.g == a.D ? lpr : a.g / EPL;
  const bool groups = a.prec != SI_PREC_INT4 ||
                      (a.g % EPL == 0 && a.lpg >= 1 && (a.lpg & (a.lpg - 1)) == 0);
  const bool turns = !rotated || (a.rot.interleaved ? 2 * a.rot.pairs : a.rot.pairs) % EPL == 0;
  if (whole && groups && turns && lpr <= 64) {
    switch (lpr) {
      case 8: launch_write<DT, 8>(a, rotated, st); break;
      case 16: launch_write<DT, 16>(a, rotated, st); break;
      case 32: launch_write<DT, 32>(a, rotated, st); break;
      default: launch_write<DT, 64>(a, rotated, st); break;
    }
    return check_launch("si_pool_write");
  }
  pool_write_any<DT><<<(unsigned)ceil_div(2 * a.T * a.H, 256), 256, 0, st>>>(a, rotated);
  return check_launch("si_pool_write/any");
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_pool_write(const si_page_pool* pool, const void* k, const void* v, int64_t T,
                             int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                             int64_t v_stride_h, const int64_t* slots, const si_rotation* rotation,
                             const void* positions, int positions64, int64_t pos_stride,
                             si_stream_t stream) {
  clear_error();
  const int rc = check_rows("si_pool_write", pool, T, slots);
  if (rc != SI_OK) return rc;
  if (rotation != nullptr)
    SI_CHECK_ARG(rotation->pairs > 0 && 2 * rotation->pairs <= pool->D && rotation->freq && (positions || T == 0),
                 "si_pool_write: bad rotation");
  if (T == 0) return SI_OK;
  SI_CHECK_ARG(k && v, "si_pool_write: NULL argument");
  PoolArgs a = pool_args(*pool, T, slots);
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.ks[0] = k_stride_t;
  a.ks[1] = k_stride_h;
  a.vs[0] = v_stride_t;
  a.vs[1] = v_stride_h;
  const bool rotated = rotation != nullptr;
  if (rotated) a.rot = to_rotation(*rotation, positions, positions64, false);
  a.pos_stride = pos_stride;
  hipStream_t st = as_stream(stream);
  if (a.sdt == SI_DT_F32) return write_rows<SI_DT_F32>(a, rotated, st);
  if (a.sdt == SI_DT_F16) return write_rows<SI_DT_F16>(a, rotated, st);
  return write_rows<SI_DT_BF16>(a, rotated, st);
}

extern "C" int si_pool_read(const si_page_pool* pool, const int64_t* slots, int64_t T, void* out_k,
                            void* out_v, int out_dtype, si_stream_t stream) {
  clear_error();
  const int rc = check_rows("si_pool_read", pool, T, slots);
  if (rc != SI_OK) return rc;
  SI_CHECK_ARG(dtype_ok(out_dtype), "si_pool_read: unsupported output dtype %d", out_dtype);
  if (T == 0) return SI_OK;
  SI_CHECK_ARG(out_k && out_v, "si_pool_read: NULL argument");
  PoolArgs a = pool_args(*pool, T, slots);
  a.ko = reinterpret_cast<char*>(out_k);
  a.vo = reinterpret_cast<char*>(out_v);
  a.odt = out_dtype;
  hipStream_t st = as_stream(stream);
  const bool vec = a.D % 8 == 0 && (a.prec != SI_PREC_INT4 || a.g % 8 == 0) && aligned16(out_k, out_v);
  if (!vec) {
    SI_CHECK_ARG(ceil_div(T * a.H * a.D, 256) < ((int64_t)1 << 31), "si_pool_read: too many rows for one call");
    pool_read_any<<<(unsigned)ceil_div(T * a.H * a.D, 256), 256, 0, st>>>(a);
    return check_launch("si_pool_read/any");
  }
  int lsh = 0;
  while ((8 << lsh) < a.D) ++lsh;
  const unsigned grid = (unsigned)(ceil_div(T, 256 >> lsh) * a.H);
  if (out_dtype == SI_DT_F32) pool_read<SI_DT_F32><<<grid, 256, 0, st>>>(a, lsh);
  else if (out_dtype == SI_DT_F16) pool_read<SI_DT_F16><<<grid, 256, 0, st>>>(a, lsh);
  else pool_read<SI_DT_BF16><<<grid, 256, 0, st>>>(a, lsh);
  return check_launch("si_pool_read");
}
