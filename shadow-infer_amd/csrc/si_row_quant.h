// Row quantization shared by the KV pack, the paged store and the page pool:
// int8 (a scale per row) and int4 (a scale per group) codes of a row held by LPR
// lanes, with the loads and stores of its 16-byte chunks.
#pragma once

#include "si_kv_common.h"

namespace si {

// ---------------------------------------------------------------------------
// Quantization arithmetic shared by the fast and generic paths.
// ---------------------------------------------------------------------------

// Quotient round(T(x / s)) of Quantizer.quantize_int8/int4
// (utils/quantization.py:141, 177) before clamping.
//  - fp32/fp16 inputs: correctly rounded division, then rounding to T.
//  - bf16 inputs with s >= 2^-100: x * r with r = RN(1/s), corrected by one
//    fma on the exact remainder (Markstein's theorem: for r = RN(1/s) and a
//    faithful q0, q0 + (x - q0*s)*r rounds to RN(x/s)). The identity with the
//    correctly rounded path, after bf16 rounding and rint, has been checked
//    exhaustively over every bf16 x and every bf16 s >= 2^-100 on the CPU.
template <int DT>
__device__ __forceinline__ float quant_quotient(float x, float s, float r, bool fast) {
  float q;
  if (DT == SI_DT_BF16) {
    if (fast) {
      const float q0 = x * r;
      const float e = __builtin_fmaf(-q0, s, x);
      q = __builtin_fmaf(e, r, q0);
    } else {
      q = x / s;
    }
    q = bf16_bits_to_f32(f32_to_bf16_bits(q));
  } else if (DT == SI_DT_F16) {
    q = f16_bits_to_f32(f32_to_f16_bits(x / s));
  } else {
    q = x / s;
  }
  return rintf(q);
}

// s = T(amax / div); s == 0 -> 1 (utils/quantization.py:138-140, 175-176).
template <int DT>
__device__ __forceinline__ float quant_scale(float amax, float div) {
  float s = amax / div;
  if (DT == SI_DT_BF16) s = bf16_bits_to_f32(f32_to_bf16_bits(s));
  if (DT == SI_DT_F16) s = f16_bits_to_f32(f32_to_f16_bits(s));
  return s == 0.0f ? 1.0f : s;
}

template <int DT>
__device__ __forceinline__ void store_scalar(void* p, int64_t i, float v) {
  if (DT == SI_DT_F32) {
    reinterpret_cast<float*>(p)[i] = v;
  } else {
    const uint32_t h = DT == SI_DT_F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
    reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)h;
  }
}

__device__ __forceinline__ float clampf(float v, float lo, float hi) {
  return fminf(fmaxf(v, lo), hi);
}

// ---------------------------------------------------------------------------
// 16-byte chunk loads: EPL values of dtype DT, widened to fp32.
// ---------------------------------------------------------------------------

template <int DT>
struct Chunk {
  static constexpr int EPL = DT == SI_DT_F32 ? 4 : 8;
};

template <int DT>
__device__ __forceinline__ void load_chunk(const void* base, int64_t elem, float* out) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 raw = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) +
                                     elem * (DT == SI_DT_F32 ? 4 : 2)));
  const uint32_t w[4] = {raw[0], raw[1], raw[2], raw[3]};
  if (DT == SI_DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == SI_DT_BF16) {
        out[2 * i] = __uint_as_float(w[i] << 16);
        out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        out[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
        out[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
      }
    }
  }
}

template <int N>
__device__ __forceinline__ void store_f32(float* dst, const float* v) {
#pragma unroll
  for (int i = 0; i < N; i += 4)
    *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}

template <int N>
__device__ __forceinline__ void store_f16(uint16_t* dst, const float* v) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = f32_to_f16_bits(v[2 * i]) | (f32_to_f16_bits(v[2 * i + 1]) << 16);
  if constexpr (N == 8) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
}

// Bytes of N int8 codes.
template <int N>
__device__ __forceinline__ void store_i8(int8_t* dst, const float* q) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = ((uint32_t)(int)q[4 * i] & 0xffu) | (((uint32_t)(int)q[4 * i + 1] & 0xffu) << 8) |
           (((uint32_t)(int)q[4 * i + 2] & 0xffu) << 16) |
           (((uint32_t)(int)q[4 * i + 3] & 0xffu) << 24);
  if constexpr (N == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// N int4 codes -> N/2 bytes, high nibble first, nibble = code + 8.
template <int N>
__device__ __forceinline__ void store_i4(uint8_t* dst, const float* q) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint32_t hi = (uint32_t)((int)q[2 * i] + 8) & 0xfu;
    const uint32_t lo = (uint32_t)((int)q[2 * i + 1] + 8) & 0xfu;
    w |= ((hi << 4) | lo) << (8 * i);
  }
  if constexpr (N == 8) {
    *reinterpret_cast<uint32_t*>(dst) = w;
  } else {
    *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
  }
}

// Working-copy values of one chunk -> the 16 bytes of the input dtype.
template <int DT>
__device__ __forceinline__ void copy_words(const float* f, uint32_t* w) {
  if constexpr (DT == SI_DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = DT == SI_DT_F16 ? f32_to_f16_bits(f[2 * i]) : f32_to_bf16_bits(f[2 * i]);
      const uint32_t b = DT == SI_DT_F16 ? f32_to_f16_bits(f[2 * i + 1]) : f32_to_bf16_bits(f[2 * i + 1]);
      w[i] = a | (b << 16);
    }
  }
}

template <int DT, int LPR, bool WC>
__device__ __forceinline__ void pack_row(const float* xk, const float* xv, int c, int s, int b,
                                         int B, int lane, int lpg, const Buckets& bk,
                                         uint32_t* ck, uint32_t* cv, int nl = LPR) {
  constexpr int EPL = Chunk<DT>::EPL;
  const int D = EPL * nl;
  const bool on = lane < nl;  // lanes past the row hold zeros and store nothing
  const int64_t orow = (int64_t)s * B + b;
  const int64_t oel = orow * D + lane * EPL;
  if (c == SI_PREC_FP32) {
    if (on) {
      store_f32<EPL>(reinterpret_cast<float*>(bk.p[0]) + oel, xk);
      store_f32<EPL>(reinterpret_cast<float*>(bk.p[1]) + oel, xv);
    }
    if constexpr (WC) {
      copy_words<DT>(xk, ck);
      copy_words<DT>(xv, cv);
    }
    return;
  }
  if (c == SI_PREC_FP16) {
    if (on) {
      store_f16<EPL>(reinterpret_cast<uint16_t*>(bk.p[4]) + oel, xk);
      store_f16<EPL>(reinterpret_cast<uint16_t*>(bk.p[5]) + oel, xv);
    }
    if constexpr (WC) {
      float fk[EPL], fv[EPL];
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        fk[i] = f16_bits_to_f32(f32_to_f16_bits(xk[i]));
        fv[i] = f16_bits_to_f32(f32_to_f16_bits(xv[i]));
      }
      copy_words<DT>(fk, ck);
      copy_words<DT>(fv, cv);
    }
    return;
  }
  // int8 (per row) or int4 (per group): shared arithmetic.
  float gk = 0.0f, gv = 0.0f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    gk = amax_fold(gk, xk[i]);
    gv = amax_fold(gv, xv[i]);
  }
  for (int off = 1; off < lpg; off <<= 1) {
    gk = amax_fold(gk, __shfl_xor(gk, off, 64));
    gv = amax_fold(gv, __shfl_xor(gv, off, 64));
  }
  float mk = gk, mv = gv;
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) {
    if (off >= lpg) {
      mk = amax_fold(mk, __shfl_xor(mk, off, 64));
      mv = amax_fold(mv, __shfl_xor(mv, off, 64));
    }
  }
  const bool i8 = (c == SI_PREC_INT8);
  const float sk = quant_scale<DT>(i8 ? mk : gk, i8 ? 127.0f : 7.0f);
  const float sv = quant_scale<DT>(i8 ? mv : gv, i8 ? 127.0f : 7.0f);
  const bool fk = sk >= 7.8886090522101181e-31f;  // 2^-100
  const bool fv = sv >= 7.8886090522101181e-31f;
  const float rk = 1.0f / sk;
  const float rv = 1.0f / sv;
  const float lo = i8 ? -128.0f : -8.0f;
  const float hi = i8 ? 127.0f : 7.0f;
  float qk[EPL], qv[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    qk[i] = clampf(quant_quotient<DT>(xk[i], sk, rk, fk), lo, hi);
    qv[i] = clampf(quant_quotient<DT>(xv[i], sv, rv, fv), lo, hi);
  }
  if constexpr (WC) {
    float fk2[EPL], fv2[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      fk2[i] = qk[i] + 0.0f;  // the integer code as a value (-0 -> +0)
      fv2[i] = qv[i] + 0.0f;
    }
    copy_words<DT>(fk2, ck);
    copy_words<DT>(fv2, cv);
  }
  if (!on) return;
  if (i8) {
    store_i8<EPL>(reinterpret_cast<int8_t*>(bk.p[8]) + oel, qk);
    store_i8<EPL>(reinterpret_cast<int8_t*>(bk.p[9]) + oel, qv);
    if (lane == 0) {
      store_scalar<DT>(bk.p[10], orow, sk);
      store_scalar<DT>(bk.p[11], orow, sv);
    }
  } else {
    const int64_t rb = (int64_t)B * D / 2;  // int4 bytes per entry (D even)
    const int64_t boff = (int64_t)s * rb + ((int64_t)b * D + lane * EPL) / 2;
    store_i4<EPL>(reinterpret_cast<uint8_t*>(bk.p[12]) + boff, qk);
    store_i4<EPL>(reinterpret_cast<uint8_t*>(bk.p[13]) + boff, qv);
    if ((lane & (lpg - 1)) == 0) {
      const int64_t si = orow * (nl < lpg ? 1 : nl / lpg) + lane / lpg;
      store_scalar<DT>(bk.p[14], si, sk);
      store_scalar<DT>(bk.p[15], si, sv);
    }
  }
}

// ---------------------------------------------------------------------------
// bf16 fast path. Same results as pack_row<SI_DT_BF16> with fewer VALU
// instructions per element (the pack kernel is VALU-bound):
//  * |x| maxima on raw bf16 bit patterns with packed 16-bit integer max (the
//    abs bit patterns order like the values; NaN patterns order above inf, so
//    a NaN still wins), butterflies inside 16-lane rows by DPP;
//  * scale = bf16(amax / d) by q0 = amax*RN(1/d) plus one fma correction, and
//    the element quotient by r = RN(1/s) plus one fma correction; both equal
//    correctly rounded division after the bf16 rounding and round-to-integer
//    that follow (checked exhaustively over all bf16 inputs by
//    tests/native/quotient_check.c);
//  * clamp, then add 1.5*2^23: the add rounds to an integer (ties to even) and
//    the low bits of the sum are the two's-complement code.
// ---------------------------------------------------------------------------

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_abs_bf16x8(const uint32_t w[4]) {
  u16x2 a = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
  u16x2 b = __builtin_bit_cast(u16x2, w[1] & 0x7fff7fffu);
  u16x2 c = __builtin_bit_cast(u16x2, w[2] & 0x7fff7fffu);
  u16x2 d = __builtin_bit_cast(u16x2, w[3] & 0x7fff7fffu);
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(a, b),
                                            __builtin_elementwise_max(c, d));
  return (uint32_t)(m.x > m.y ? m.x : m.y);
}

// v = max(v, v of lane ^ OFF) for a butterfly inside aligned groups of lanes.
// OFF 1/2 are quad permutes; OFF 4/8 use the half-row / row mirrors, which pair
// the same groups once the previous steps made each sub-group uniform.
template <int OFF>
__device__ __forceinline__ uint32_t bfly_max(uint32_t v) {
  int o;
  if constexpr (OFF == 1) o = __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);
  else if constexpr (OFF == 2) o = __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);
  else if constexpr (OFF == 4) o = __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false);
  else if constexpr (OFF == 8) o = __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false);
  else o = __shfl_xor((int)v, OFF, 64);
  return v > (uint32_t)o ? v : (uint32_t)o;
}

// Row maximum over LPR lanes; *grp receives the maximum over groups of lpg lanes.
template <int LPR>
__device__ __forceinline__ uint32_t row_group_max(uint32_t v, int lpg, uint32_t* grp) {
  uint32_t g = v;
  if constexpr (LPR > 1) { v = bfly_max<1>(v); if (lpg == 2) g = v; }
  if constexpr (LPR > 2) { v = bfly_max<2>(v); if (lpg == 4) g = v; }
  if constexpr (LPR > 4) { v = bfly_max<4>(v); if (lpg == 8) g = v; }
  if constexpr (LPR > 8) { v = bfly_max<8>(v); if (lpg == 16) g = v; }
  if constexpr (LPR > 16) { v = bfly_max<16>(v); if (lpg == 32) g = v; }
  if constexpr (LPR > 32) { v = bfly_max<32>(v); }
  if (lpg == LPR) g = v;
  *grp = g;
  return v;
}

// bf16(amax / d) with 0 -> 1; h = abs bf16 bits of amax.
__device__ __forceinline__ float bf16_scale(uint32_t h, float d, float rd) {
  const float a = __uint_as_float(h << 16);
  float q;
  if (h < 0x7f80u) {
    const float q0 = a * rd;
    q = __builtin_fmaf(__builtin_fmaf(-q0, d, a), rd, q0);
  } else {
    q = a / d;  // inf or NaN amax
  }
  const float s = bf16_bits_to_f32(f32_to_bf16_bits(q));
  return s == 0.0f ? 1.0f : s;
}

constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23

// Integer code (as the low bits of the returned word) of one bf16 value x.
__device__ __forceinline__ uint32_t quant_bf16(float x, float s, float r, bool fast, float lo,
                                               float hi) {
  float q;
  if (fast) {
    const float q0 = x * r;
    q = round_bf16_finite(__builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0));
  } else {
    q = bf16_bits_to_f32(f32_to_bf16_bits(x / s));
  }
  q = __builtin_amdgcn_fmed3f(q, lo, hi);
  return __float_as_uint(q + kMagic);
}

// Low bytes of four words -> one word.
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Two integer codes (words from quant_bf16) -> their bf16 values in one word.
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t q0, uint32_t q1) {
  const uint32_t a = __float_as_uint(__uint_as_float(q0) - kMagic) >> 16;  // exact in bf16
  const uint32_t b = __float_as_uint(__uint_as_float(q1) - kMagic) & 0xffff0000u;
  return a | b;
}

// Bucket row stores of the bf16 pack. Token order (rows of a block anywhere
// in the bucket): plain stores. Bucket order: device-scope (sc1) buffer
// stores from the block's first row, which write the lines through as they
// leave: 7B layer, headline protocol, pack 40.8 -> 39.0 us, and an unpack
// right after the pack as fast as before (55.0 us). A non-temporal store made
// the pack as fast but pushed the buckets out of the last-level cache, so an
// unpack that follows the pack took 27% longer.
template <typename T>
__device__ __forceinline__ void st_row(void* p, T v) {
  *reinterpret_cast<T*>(p) = v;
}

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

// Raw buffer from byte `first` of a bucket (block-uniform); `off` is the
// byte offset from there (a block's rows span a few KB).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(void* bucket, int64_t first) {
  return __builtin_amdgcn_make_buffer_rsrc(wave_uniform(reinterpret_cast<char*>(bucket) + first),
                                           (short)0, -1, 0x00020000);
}
__device__ __forceinline__ void st_dev(void* bucket, int64_t first, uint32_t off, u32x4_t v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, rows_rsrc(bucket, first), (int)off, 0, 16);
}
__device__ __forceinline__ void st_dev(void* bucket, int64_t first, uint32_t off, u32x2_t v) {
  __builtin_amdgcn_raw_buffer_store_b64(v, rows_rsrc(bucket, first), (int)off, 0, 16);
}
__device__ __forceinline__ void st_dev(void* bucket, int64_t first, uint32_t off, uint32_t v) {
  __builtin_amdgcn_raw_buffer_store_b32(v, rows_rsrc(bucket, first), (int)off, 0, 16);
}

// DEV: bucket rows stored with st_dev relative to bucket row `row0` (the
// block's first row; every row of the block is at most a few KB past it).
template <int LPR, bool WC, bool DEV = false>
__device__ __forceinline__ void pack_row_bf16(const uint32_t wk[4], const uint32_t wv[4], int c,
                                              int s, int b, int B, int lane, int lpg,
                                              const Buckets& bk, uint32_t* ck, uint32_t* cv,
                                              int64_t row0 = 0, int nl = LPR) {
  const int D = 8 * nl;
  const bool on = lane < nl;  // lanes past the row hold zeros and store nothing
  const int64_t orow = (int64_t)s * B + b;
  const int64_t oel = orow * D + lane * 8;
  const uint32_t rel = (uint32_t)((orow - row0) * D + lane * 8);  // element offset from row0
  if (c == SI_PREC_FP16 || c == SI_PREC_FP32) {
    if (!on) return;
    float xk[8], xv[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xk[2 * i] = __uint_as_float(wk[i] << 16);
      xk[2 * i + 1] = __uint_as_float(wk[i] & 0xffff0000u);
      xv[2 * i] = __uint_as_float(wv[i] << 16);
      xv[2 * i + 1] = __uint_as_float(wv[i] & 0xffff0000u);
    }
    if (c == SI_PREC_FP16) {
      typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
      u32x4 hk, hv;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hk[i] = f32_to_f16_bits(xk[2 * i]) | (f32_to_f16_bits(xk[2 * i + 1]) << 16);
        hv[i] = f32_to_f16_bits(xv[2 * i]) | (f32_to_f16_bits(xv[2 * i + 1]) << 16);
      }
      if constexpr (DEV) {
        st_dev(bk.p[4], row0 * D * 2, rel * 2, hk);
        st_dev(bk.p[5], row0 * D * 2, rel * 2, hv);
      } else {
        st_row(reinterpret_cast<uint16_t*>(bk.p[4]) + oel, hk);
        st_row(reinterpret_cast<uint16_t*>(bk.p[5]) + oel, hv);
      }
      if constexpr (WC) {
        float fk[8], fv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          fk[i] = f16_bits_to_f32(f32_to_f16_bits(xk[i]));
          fv[i] = f16_bits_to_f32(f32_to_f16_bits(xv[i]));
        }
        copy_words<SI_DT_BF16>(fk, ck);
        copy_words<SI_DT_BF16>(fv, cv);
      }
    } else {
      store_f32<8>(reinterpret_cast<float*>(bk.p[0]) + oel, xk);
      store_f32<8>(reinterpret_cast<float*>(bk.p[1]) + oel, xv);
      if constexpr (WC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ck[i] = wk[i];
          cv[i] = wv[i];
        }
      }
    }
    return;
  }
  uint32_t gk, gv;
  const uint32_t mk = row_group_max<LPR>(max_abs_bf16x8(wk), lpg, &gk);
  const uint32_t mv = row_group_max<LPR>(max_abs_bf16x8(wv), lpg, &gv);
  const bool i8 = (c == SI_PREC_INT8);
  const float d = i8 ? 127.0f : 7.0f;
  const float rd = i8 ? 0.0078740157186985016f : 0.14285714924335480f;  // RN(1/d)
  const float sk = bf16_scale(i8 ? mk : gk, d, rd);
  const float sv = bf16_scale(i8 ? mv : gv, d, rd);
  const bool fk = sk >= 7.8886090522101181e-31f && sk < 3.0e38f;
  const bool fv = sv >= 7.8886090522101181e-31f && sv < 3.0e38f;
  const float rk = 1.0f / sk;
  const float rv = 1.0f / sv;
  const float lo = i8 ? -128.0f : -8.0f;
  const float hi = i8 ? 127.0f : 7.0f;
  uint32_t qk[8], qv[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    qk[2 * i] = quant_bf16(__uint_as_float(wk[i] << 16), sk, rk, fk, lo, hi);
    qk[2 * i + 1] = quant_bf16(__uint_as_float(wk[i] & 0xffff0000u), sk, rk, fk, lo, hi);
    qv[2 * i] = quant_bf16(__uint_as_float(wv[i] << 16), sv, rv, fv, lo, hi);
    qv[2 * i + 1] = quant_bf16(__uint_as_float(wv[i] & 0xffff0000u), sv, rv, fv, lo, hi);
  }
  if constexpr (WC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ck[i] = codes_bf16x2(qk[2 * i], qk[2 * i + 1]);
      cv[i] = codes_bf16x2(qv[2 * i], qv[2 * i + 1]);
    }
  }
  if (!on) return;
  if (i8) {
    const u32x2_t k8{bytes4(qk[0], qk[1], qk[2], qk[3]), bytes4(qk[4], qk[5], qk[6], qk[7])};
    const u32x2_t v8{bytes4(qv[0], qv[1], qv[2], qv[3]), bytes4(qv[4], qv[5], qv[6], qv[7])};
    if constexpr (DEV) {
      st_dev(bk.p[8], row0 * D, rel, k8);
      st_dev(bk.p[9], row0 * D, rel, v8);
    } else {
      st_row(reinterpret_cast<int8_t*>(bk.p[8]) + oel, k8);
      st_row(reinterpret_cast<int8_t*>(bk.p[9]) + oel, v8);
    }
    if (lane == 0) {
      reinterpret_cast<uint16_t*>(bk.p[10])[orow] = (uint16_t)(__float_as_uint(sk) >> 16);
      reinterpret_cast<uint16_t*>(bk.p[11])[orow] = (uint16_t)(__float_as_uint(sv) >> 16);
    }
  } else {
    // Byte = ((q0 & 0xF) << 4 | (q1 & 0xF)) ^ 0x88: the two's-complement nibble
    // with its top bit flipped is the offset-binary nibble q + 8.
    uint32_t bkk[4], bvv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bkk[j] = __builtin_amdgcn_ubfe(qk[2 * j], 0, 4) << 4 | __builtin_amdgcn_ubfe(qk[2 * j + 1], 0, 4);
      bvv[j] = __builtin_amdgcn_ubfe(qv[2 * j], 0, 4) << 4 | __builtin_amdgcn_ubfe(qv[2 * j + 1], 0, 4);
    }
    const int64_t rb = (int64_t)B * D / 2;
    const int64_t boff = (int64_t)s * rb + ((int64_t)b * D + lane * 8) / 2;
    const uint32_t k4 = bytes4(bkk[0], bkk[1], bkk[2], bkk[3]) ^ 0x88888888u;
    const uint32_t v4 = bytes4(bvv[0], bvv[1], bvv[2], bvv[3]) ^ 0x88888888u;
    if constexpr (DEV) {  // D even: row r's int4 bytes start at r * D / 2
      st_dev(bk.p[12], row0 * (D / 2), rel / 2, k4);
      st_dev(bk.p[13], row0 * (D / 2), rel / 2, v4);
    } else {
      st_row(reinterpret_cast<uint8_t*>(bk.p[12]) + boff, k4);
      st_row(reinterpret_cast<uint8_t*>(bk.p[13]) + boff, v4);
    }
    if ((lane & (lpg - 1)) == 0) {
      const int64_t si = orow * (nl < lpg ? 1 : nl / lpg) + lane / lpg;
      reinterpret_cast<uint16_t*>(bk.p[14])[si] = (uint16_t)(__float_as_uint(sk) >> 16);
      reinterpret_cast<uint16_t*>(bk.p[15])[si] = (uint16_t)(__float_as_uint(sv) >> 16);
    }
  }
}

}  // namespace si
