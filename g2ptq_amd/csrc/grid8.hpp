// The integer grid of run-time data (tokens, keys and values): device helpers
// shared by the token quantiser and the paged cache.
//
//   symmetric:   s = max|x| / ((2^b − 1)/2),              z = 0
//   asymmetric:  s = (max(x, 0) − min(x, 0)) / (2^b − 1), z = clamp(round(minq − min(x, 0)/s))
//   q = clamp(round(x/s) + z, minq, maxq),  x̂ = s·(q − z)
//
// (the weight quantizer's grid, utils/quant_utils.py:8-68, for one group of
// values).  Every quotient is rounded to fp32 before it is rounded to a code,
// so codes equal the same expression evaluated by torch in fp32 bit for bit.
// Unlike weights, run-time data may be all zero (padding): s = 0, and codes
// and zero point are 0.  A NaN or an infinity in the values makes s NaN or
// infinite, with codes and zero point 0, so x̂ = s·0 is NaN in the whole
// group.  Compile with -ffp-contract=off.
#pragma once
#include "common.hpp"

namespace g2ptq {

// Eight consecutive values of a row as fp32; DT 0 bf16, 1 fp16, 2 fp32.
// vec: the address is a multiple of 16 bytes.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, bool vec, int n, float (&v)[8]) {
  if constexpr (DT == 2) {
    const float* x = static_cast<const float*>(p) + at;
    if (vec && n >= 8) {
      const float4 a = *reinterpret_cast<const float4*>(x);
      const float4 b = *reinterpret_cast<const float4*>(x + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
      v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? x[i] : 0.f;
    }
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(p) + at;
    uint32_t w[4];
    if (vec && n >= 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(x);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (2 * i < n ? x[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)x[2 * i + 1] << 16 : 0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 0) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
}

// Eight fp32 values to a row of dtype DT (round to nearest even, NaN kept).
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, bool vec, int n, const float (&v)[8]) {
  if constexpr (DT == 2) {
    float* x = static_cast<float*>(p) + at;
    if (vec && n >= 8) {
      *reinterpret_cast<float4*>(x) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(x + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = v[i];
    }
  } else {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == 0) h[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
      else h[i] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
    }
    uint16_t* x = static_cast<uint16_t*>(p) + at;
    if (vec && n >= 8) {
      uint4 w;
      w.x = h[0] | (uint32_t)h[1] << 16, w.y = h[2] | (uint32_t)h[3] << 16;
      w.z = h[4] | (uint32_t)h[5] << 16, w.w = h[6] | (uint32_t)h[7] << 16;
      *reinterpret_cast<uint4*>(x) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = h[i];
    }
  }
}

// The same at any address that is aligned for the type: sixteen bytes are one instruction wherever
// they lie.  MI355X, RMS norm of 4096 rows of 4099 with residual: 33 µs, 75 a value at a time.
template <int DT>
__device__ __forceinline__ void load8_any(const void* p, int64_t at, int n, float (&v)[8]) {
  if constexpr (DT == 2) {
    const float* x = static_cast<const float*>(p) + at;
    if (n >= 8) {
      __builtin_memcpy(v, x, 16);
      __builtin_memcpy(v + 4, x + 4, 16);
    } else {
      // (no branch a value: their loads are under way together)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      if (n > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[i < n ? i : 0];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.f;
      }
    }
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(p) + at;
    uint32_t w[4];
    if (n >= 8) {
      __builtin_memcpy(w, x, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = 0;
      if (n > 0) {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = x[i < n ? i : 0];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = i < n ? h[i] : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | h[2 * i + 1] << 16;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 0) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8_any(void* p, int64_t at, int n, const float (&v)[8]) {
  if constexpr (DT == 2) {
    float* x = static_cast<float*>(p) + at;
    if (n >= 8) {
      __builtin_memcpy(x, v, 16);
      __builtin_memcpy(x + 4, v + 4, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = v[i];
    }
  } else {
    uint16_t* x = static_cast<uint16_t*>(p) + at;
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == 0) h[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
      else h[i] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
    }
    if (n >= 8) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
      __builtin_memcpy(x, w, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = h[i];
    }
  }
}

// Range of a group: the largest |x| by its bits, which orders NaN above infinity
// above every number; in the asymmetric grid min(x, 0) and max(x, 0) too.
template <bool SYM>
struct Range {
  float lo = 0.f, hi = 0.f;
  uint32_t top = 0;
  __device__ __forceinline__ void add(float x) {
    if (!SYM) {
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    top = max(top, __float_as_uint(x) & 0x7fffffffu);
  }
  __device__ __forceinline__ void merge(float l, float h, uint32_t t) {
    if (!SYM) {
      lo = fminf(lo, l);
      hi = fmaxf(hi, h);
    }
    top = max(top, t);
  }
};

// x of another lane of the same 16: neighbours, pairs, halves of 8, halves of 16 (once
// all lanes below agree, the mirrors bring the other half's value).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL, bool SYM>
__device__ __forceinline__ void merge_dpp(Range<SYM>& r) {
  float l = 0.f, h = 0.f;
  if (!SYM) {
    l = __uint_as_float(dpp<CTRL>(__float_as_uint(r.lo)));
    h = __uint_as_float(dpp<CTRL>(__float_as_uint(r.hi)));
  }
  r.merge(l, h, dpp<CTRL>(r.top));
}

// Over L neighbouring lanes (a power of two); every lane gets the result.
template <int L, bool SYM>
__device__ __forceinline__ void reduce_range(Range<SYM>& r) {
  if (L >= 2) merge_dpp<0xb1>(r);    // quad_perm 1 0 3 2
  if (L >= 4) merge_dpp<0x4e>(r);    // quad_perm 2 3 0 1
  if (L >= 8) merge_dpp<0x141>(r);   // row_half_mirror
  if (L >= 16) merge_dpp<0x140>(r);  // row_mirror
#pragma unroll
  for (int o = 16; o < L; o *= 2)
    r.merge(SYM ? 0.f : __shfl_xor(r.lo, o), SYM ? 0.f : __shfl_xor(r.hi, o),
            __shfl_xor(r.top, o));
}

struct Grid {
  float s, z, y, minq, maxq;
  bool plain;  // s where the corrected product below is the IEEE quotient wherever it matters
};

template <bool SYM>
__device__ __forceinline__ Grid make_grid(const Range<SYM>& r, int bits) {
  Grid g;
  const float levels = (float)((1 << bits) - 1);
  g.minq = -(float)(1 << (bits - 1));
  g.maxq = (float)((1 << (bits - 1)) - 1);
  const float m = __uint_as_float(r.top);
  if (SYM) {
    g.s = __fdiv_rn(m, 0.5f * levels);
    g.z = 0.f;
  } else {
    // top > the bits of infinity: a NaN among the values
    g.s = r.top > 0x7f800000u ? m : __fdiv_rn(__fsub_rn(r.hi, r.lo), levels);
    const float t = rintf(__fsub_rn(g.minq, __fdiv_rn(r.lo, g.s)));
    g.z = t < g.minq ? g.minq : (t > g.maxq ? g.maxq : t);
  }
  if (!(g.s > 0.f && g.s < __builtin_inff())) g.z = 0.f;
  g.y = __fdiv_rn(1.f, g.s);
  g.plain = g.s >= 0x1p-80f && g.s <= 0x1p100f;
  return g;
}

// x/s rounded to fp32, rounded to an integer, offset and clamped.  Markstein's
// corrected product (quant.hip) gives the IEEE quotient for s in [2^-80,
// 2^100] and every x that does not round to code 0; smaller quotients round to
// 0 either way.  Three operations instead of the division's eleven.
__device__ __forceinline__ int to_code(const Grid& g, float x) {
  float q;
  if (g.plain) {
    const float a = __fmul_rn(x, g.y);
    q = __fmaf_rn(__fmaf_rn(-g.s, a, x), g.y, a);
  } else {
    q = __fdiv_rn(x, g.s);
    if (!(fabsf(q) < __builtin_inff())) q = 0.f;  // 0/0, NaN and infinite groups
  }
  q = rintf(q) + g.z;
  return (int)fminf(fmaxf(q, g.minq), g.maxq);
}

}  // namespace g2ptq
