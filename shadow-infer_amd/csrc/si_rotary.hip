// Rotary positions of query and key rows in one launch.
//
//   y_a = g (x_a cos pf - x_b sin pf),  y_b = g (x_b cos pf + x_a sin pf)
//
// for the pairs (a, b) of the first 2 * pairs values of every head; the others
// are copied. Each value is read and written once, so HBM bounds long inputs (8192
// tokens x 40 heads of 128 bf16: 41 us, 4.1 TB/s) and the launch short ones (one token:
// 3.6 us). The angles come from the positions, not from a table: a block computes the
// cosines of its tokens once, in 64 bits, keeps them in LDS and uses them for every
// head. Stores are plain, as what follows reads the rows: with non-temporal ones
// the kernel alone took 36 to 38 us, but together with a reader behind it 70.8 against
// 66.4; with device-scope ones 94. Four rows a thread took 53 us; one took 41 (interleaved)
// and 38.2 against 40.1 (half), but 4.66 against 4.58 at 1003 tokens x 24 heads of 80.
#include "si_rotate.h"

namespace si {
namespace {

struct RotaryRows {
  const char* src;
  char* dst;
  int64_t ss[3];  // elements between batches, tokens, heads
  int64_t ds[3];
  int heads;
};

struct RotaryArgs {
  RotaryRows t[2];
  Rotation rot;
  int64_t ps[2];  // elements between batches and tokens in the positions
  int64_t tokens;
  int S;          // tokens of a batch row
  int tb, hb;     // tokens and heads of a block
  int ush;        // log2 of the threads of a head row
  int rot_units, units;
};

template <int DT, int VE>
__device__ __forceinline__ void load_vals(const char* p, float* x) {
  if constexpr (VE == 1) {
    x[0] = load_any(p, DT, 0);
  } else {
    const uint4 w4 = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
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
}

template <int DT, int VE>
__device__ __forceinline__ void store_vals(char* p, const float* x) {
  if constexpr (VE == 1) {
    store_any(p, DT, 0, x[0]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SI_DT_F32) w[i] = __float_as_uint(x[i]);
      else if constexpr (DT == SI_DT_BF16) w[i] = f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
      else w[i] = f32_to_f16_bits(x[2 * i]) | (f32_to_f16_bits(x[2 * i + 1]) << 16);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Block (x, y): tokens [x * tb, ..) and heads [y * hb, ..) of q's and k's heads
// in a row. A unit is VE pairs: two chunks of VE values, pairs apart (half) or
// next to each other (interleaved), or one chunk of the values behind the pairs.
// Each thread loads the chunks of UN rows before it turns the first.
template <int DT, int VE, bool INTER, int UN>
__global__ __launch_bounds__(256) void rotary_rows(RotaryArgs a) {
  constexpr int ES = DT == SI_DT_F32 ? 4 : 2;
  extern __shared__ char lds[];
  float2* cs = reinterpret_cast<float2*>(lds);  // [tb][pairs]
  int64_t* off = reinterpret_cast<int64_t*>(lds + sizeof(float2) * a.tb * a.rot.pairs);  // [tb][4]
  const int64_t n0 = (int64_t)blockIdx.x * a.tb;
  const int nt = (int)(a.tokens - n0 < a.tb ? a.tokens - n0 : a.tb);
  const int pairs = a.rot.pairs;
  for (int i = threadIdx.x; i < nt * pairs; i += 256) {
    const int t = i / pairs, p = i - t * pairs;
    const int64_t n = n0 + t, b = n / a.S, s = n - b * a.S;
    cs[i] = pair_cos_sin(a.rot, b * a.ps[0] + s * a.ps[1], p);
  }
  for (int i = threadIdx.x; i < nt * 4; i += 256) {
    const int t = i >> 2, j = (i >> 1) & 1;
    const int64_t n = n0 + t, b = n / a.S, s = n - b * a.S;
    const int64_t* st = (i & 1) ? a.t[j].ds : a.t[j].ss;
    off[i] = b * st[0] + s * st[1];
  }
  __syncthreads();
  const int heads = a.t[0].heads + a.t[1].heads;
  const int h0 = blockIdx.y * a.hb;
  const int nh = heads - h0 < a.hb ? heads - h0 : a.hb;
  const int step = 256 >> a.ush, rows = nt * nh;
  for (int u = threadIdx.x & ((1 << a.ush) - 1); u < a.units; u += 1 << a.ush) {
    const bool turn = u < a.rot_units;
    // element offsets of the unit's one or two chunks
    const int d0 = turn ? (INTER ? 2 * u * VE : u * VE) : 2 * pairs + (u - a.rot_units) * VE;
    const int d1 = turn ? (INTER ? d0 + VE : d0 + pairs) : d0;
    for (int r0 = threadIdx.x >> a.ush; r0 < rows; r0 += step * UN) {
      float x[UN][2 * VE];
      char* dst[UN];
      int tok[UN];
      bool live[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int r = r0 + k * step;
        const int t = r / nh;
        int h = h0 + r - t * nh;
        const int j = h >= a.t[0].heads;
        if (j) h -= a.t[0].heads;
        const RotaryRows& rr = a.t[j];
        live[k] = r < rows;
        tok[k] = t;
        if (!live[k]) continue;
        const char* src = rr.src + (off[4 * t + 2 * j] + h * rr.ss[2]) * ES;
        dst[k] = rr.dst + (off[4 * t + 2 * j + 1] + h * rr.ds[2]) * ES;
        live[k] = turn || src != dst[k];  // in place, the other values stay as they are
        if (!live[k]) continue;
        load_vals<DT, VE>(src + d0 * ES, x[k]);
        if (turn) load_vals<DT, VE>(src + d1 * ES, x[k] + VE);
      }
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        if (!live[k]) continue;
        if (turn) {
          const float2* c = cs + tok[k] * pairs + u * VE;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            if (INTER) rotate_pair(c[e], x[k][2 * e], x[k][2 * e + 1]);
            else rotate_pair(c[e], x[k][e], x[k][VE + e]);
          }
        }
        store_vals<DT, VE>(dst[k] + d0 * ES, x[k]);
        if (turn) store_vals<DT, VE>(dst[k] + d1 * ES, x[k] + VE);
      }
    }
  }
}

constexpr int kUnroll = 2;

template <int DT, int VE>
void launch(const RotaryArgs& a, dim3 grid, size_t lds, hipStream_t st) {
  if (a.rot.interleaved) rotary_rows<DT, VE, true, kUnroll><<<grid, 256, lds, st>>>(a);
  else rotary_rows<DT, VE, false, kUnroll><<<grid, 256, lds, st>>>(a);
}

}  // namespace
}  // namespace si

using namespace si;

extern "C" int si_rotary(const si_rotation* rotation, const si_rotary_rows* q, const si_rotary_rows* k,
                         int dtype, int64_t B, int64_t S, int64_t D, int transpose,
                         const void* positions, int positions64, int64_t pos_stride_b,
                         int64_t pos_stride_s, si_stream_t stream) {
  clear_error();
  SI_CHECK_ARG(dtype_ok(dtype), "si_rotary: unsupported dtype %d", dtype);
  SI_CHECK_ARG(B >= 0 && S >= 0 && B < ((int64_t)1 << 31) && S < ((int64_t)1 << 31) &&
               B * S < ((int64_t)1 << 31), "si_rotary: bad batch");
  SI_CHECK_ARG(rotation != nullptr && q != nullptr, "si_rotary: NULL argument");
  const int64_t pairs = rotation->pairs;
  SI_CHECK_ARG(D > 0 && D <= 1024 && pairs > 0 && 2 * pairs <= D,
               "si_rotary: need 0 < 2 * pairs <= D <= 1024");
  RotaryArgs a = {};
  const si_rotary_rows* in[2] = {q, k};
  uintptr_t bits = 0;
  int64_t strides = 0;
  for (int j = 0; j < 2; ++j) {
    if (in[j] == nullptr) continue;
    SI_CHECK_ARG(in[j]->heads >= 0 && in[j]->heads < 65536, "si_rotary: bad head count");
    a.t[j].heads = (int)in[j]->heads;
    a.t[j].src = reinterpret_cast<const char*>(in[j]->src);
    a.t[j].dst = reinterpret_cast<char*>(in[j]->dst);
    for (int i = 0; i < 3; ++i) {
      a.t[j].ss[i] = in[j]->src_stride[i];
      a.t[j].ds[i] = in[j]->dst_stride[i];
      strides |= in[j]->src_stride[i] | in[j]->dst_stride[i];
    }
    bits |= reinterpret_cast<uintptr_t>(in[j]->src) | reinterpret_cast<uintptr_t>(in[j]->dst);
  }
  const int64_t tokens = B * S;
  const int heads = a.t[0].heads + a.t[1].heads;
  if (tokens == 0 || heads == 0) return SI_OK;
  for (int j = 0; j < 2; ++j)
    SI_CHECK_ARG(a.t[j].heads == 0 || (a.t[j].src && a.t[j].dst), "si_rotary: NULL argument");
  SI_CHECK_ARG(rotation->freq && positions, "si_rotary: NULL argument");
  a.rot = to_rotation(*rotation, positions, positions64, transpose);
  a.ps[0] = pos_stride_b;
  a.ps[1] = pos_stride_s;
  a.tokens = tokens;
  a.S = (int)S;
  // 16-byte chunks where every chunk of every row is aligned, else single values
  const int ve = dtype == SI_DT_F32 ? 4 : 8;
  const bool vec = pairs % ve == 0 && D % ve == 0 && strides % ve == 0 && (bits & 15) == 0;
  const int unit = vec ? ve : 1;
  a.rot_units = (int)pairs / unit;
  a.units = a.rot_units + (int)(D - 2 * pairs) / unit;
  while ((1 << a.ush) < a.units && a.ush < 8) ++a.ush;
  // A block takes whole tokens, enough for kUnroll rows a thread (at most 16, or
  // what 16 KB of cosines hold); few tokens are split over their heads instead.
  const int step = 256 >> a.ush;
  int64_t tb = ceil_div(2 * kUnroll * step, heads);
  if (tb > 16) tb = 16;
  while (tb > 1 && tb * pairs > 2048) --tb;
  a.hb = heads;
  if (ceil_div(tokens, tb) < 512) {
    tb = 1;
    if (tokens * ceil_div(heads, step) <= 1024) a.hb = step < heads ? step : heads;
  }
  a.tb = (int)tb;
  const dim3 grid((unsigned)ceil_div(tokens, tb), (unsigned)ceil_div(heads, a.hb));
  const size_t lds = (size_t)tb * (sizeof(float2) * pairs + 4 * sizeof(int64_t));
  hipStream_t st = as_stream(stream);
  if (dtype == SI_DT_F32) {
    if (vec) launch<SI_DT_F32, 4>(a, grid, lds, st);
    else launch<SI_DT_F32, 1>(a, grid, lds, st);
  } else if (dtype == SI_DT_F16) {
    if (vec) launch<SI_DT_F16, 8>(a, grid, lds, st);
    else launch<SI_DT_F16, 1>(a, grid, lds, st);
  } else {
    if (vec) launch<SI_DT_BF16, 8>(a, grid, lds, st);
    else launch<SI_DT_BF16, 1>(a, grid, lds, st);
  }
  return check_launch("si_rotary");
}
