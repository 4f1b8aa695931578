// Root-mean-square norm of rows, with the residual's addition, and its 8-bit codes.
//
//   s = x + r (r may be absent),  y_c = s_c·w_c / sqrt(Σ s²/C + ε)
//   codes, scale and zero point of y's row on the grid of grid8.hpp with 8 bits
//
// Sums, the root and y are fp32 whatever the types: y is computed from the unrounded s and
// quantized unrounded; s and y are rounded once where they are stored.  Squares that leave
// fp32's range are taken of the row scaled by a power of two.
#include <algorithm>

#include "grid8.hpp"

namespace g2ptq {
namespace {

struct NormArgs {
  const void *x, *r, *w;
  int64_t xo, xi, ro, ri;  // strides of row / inner and row % inner (elements)
  int64_t rows, first;     // and the launch's first row
  uint32_t inner;
  int C, wtype;
  float eps;
  void *y, *sum;           // rows of C, each nullable
  int8_t* codes;           // rows of ldc bytes
  int64_t ldc;
  float *scale, *zero;
};

__device__ __forceinline__ void load_weight(const NormArgs& a, int c, int n, float (&v)[8]) {
  if (a.wtype == 0) load8_any<0>(a.w, c, n, v);
  else if (a.wtype == 1) load8_any<1>(a.w, c, n, v);
  else load8_any<2>(a.w, c, n, v);
}

// Over the L lanes of a row (L = 256: the workgroup, by its waves' results in LDS).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int o = 1; o < (L < 64 ? L : 64); o *= 2) v += __shfl_xor(v, o);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < L / 64; ++w) v += lds[w];
  }
  return v;
}
template <int L, bool SYM>
__device__ __forceinline__ void row_range(Range<SYM>& r, float (*lds)[3]) {
  reduce_range<(L < 64 ? L : 64)>(r);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) {
      float* p = lds[threadIdx.x >> 6];
      p[0] = r.lo, p[1] = r.hi, p[2] = __uint_as_float(r.top);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < L / 64; ++w) r.merge(lds[w][0], lds[w][1], __float_as_uint(lds[w][2]));
  }
}

// L lanes walk a row, eight values at a time: V pieces kept in registers, or read again
// for each use (V = 0).  Q: 0 y alone, 1 symmetric codes, 2 asymmetric ones.  Bound by the bytes:
// MI355X, under the profiler, 8192 × 4096 bf16 with residual to codes and sum 53–55 µs (235 MB,
// 4.3 TB/s), 262144 heads of 128 27–29 µs (134 MB, 4.9 TB/s); one row of 4096 4.1–4.5 µs, the
// latencies of a launch, the loads and two reductions.  These stay bare where a row is few bytes for
// its workgroup, to codes without a residual most: replayed, 8192 × 4096 28.8 µs (101 MB, 3.5 TB/s),
// 4096 × 4099 25.4 (50 MB), 2048 × 8192 18.4 (50 MB), 1024 × 16384, read three times, 26 (50 MB).
template <int DT, int Q, int L, int V>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormArgs a) {
  constexpr bool SYM = Q != 2;
  constexpr int STEP = L * 8, N = V ? V : 1;
  __shared__ float sums[2][4], ranges[2][4][3];
  const int64_t row = a.first + (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= a.rows) return;  // (L = 256: a whole workgroup)
  const int c0 = threadIdx.x % L * 8;
  const int64_t o = a.inner == 1 ? row : row / a.inner, i = row - o * a.inner;
  const int64_t xat = o * a.xo + i * a.xi, rat = o * a.ro + i * a.ri;
  float s[N][8], w[N][8];

  auto fetch = [&](int c, float (&v)[8]) {
    load8_any<DT>(a.x, xat + c, a.C - c, v);
    if (a.r) {
      float u[8];
      load8_any<DT>(a.r, rat + c, a.C - c, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += u[j];
    }
  };
  // f(piece, its first column) for every piece
  auto each = [&](auto f) {
    if constexpr (V > 0) {
#pragma unroll
      for (int p = 0; p < V; ++p) f(p, c0 + p * STEP);
    } else {
      for (int c = c0; c < a.C; c += STEP) f(0, c);
    }
  };

  float ss = 0.f;
  if constexpr (V > 0) {
    each([&](int p, int c) { fetch(c, s[p]); });
    each([&](int p, int c) { load_weight(a, c, a.C - c, w[p]); });
  }
  each([&](int p, int c) {
    if constexpr (V == 0) fetch(c, s[0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __fmaf_rn(s[p][j], s[p][j], ss);
    // (sum and y may be x or r: a piece is stored after its last fetch)
    if constexpr (V > 0)
      if (a.sum && c < a.C) store8_any<DT>(a.sum, row * a.C + c, a.C - c, s[p]);
  });
  ss = row_sum<L>(ss, sums[0]);
  // k: a power of two that s is scaled by
  float k = 1.f, eps = a.eps;
  if (!(ss < 0x1p120f) || ss < 0x1p-80f) {
    Range<true> m;
    each([&](int p, int c) {
      if constexpr (V == 0) fetch(c, s[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) m.add(s[p][j]);
    });
    row_range<L>(m, ranges[0]);
    const float big = fmaxf(__uint_as_float(m.top), __fsqrt_rn(eps));
    if (m.top < 0x7f800000u && big > 0.f) {
      const int e = min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126);
      k = __uint_as_float((uint32_t)(127 - e) << 23);
      eps = eps * k * k;
      ss = 0.f;
      each([&](int p, int c) {
        if constexpr (V == 0) fetch(c, s[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __fmaf_rn(s[p][j] * k, s[p][j] * k, ss);
      });
      ss = row_sum<L>(ss, sums[1]);
    }
  }
  const float inv = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)a.C) + eps));
  auto norm = [&](int p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[p][j] = s[p][j] * k * inv * w[p][j];
  };
  if constexpr (V > 0) each([&](int p, int c) { norm(p); });
  auto value = [&](int p, int c, bool last) {
    if constexpr (V == 0) {
      fetch(c, s[0]);
      if (last && a.sum && c < a.C) store8_any<DT>(a.sum, row * a.C + c, a.C - c, s[0]);
      load_weight(a, c, a.C - c, w[0]);
      norm(0);
    }
  };
  if constexpr (Q == 0) {
    each([&](int p, int c) {
      value(p, c, true);
      if (c < a.C) store8_any<DT>(a.y, row * a.C + c, a.C - c, s[p]);
    });
  } else {
    Range<SYM> r;
    each([&](int p, int c) {
      value(p, c, false);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.C) r.add(s[p][j]);
    });
    row_range<L>(r, ranges[1]);
    const Grid g = make_grid<SYM>(r, 8);
    if (c0 == 0) {
      a.scale[row] = g.s;
      if (!SYM) a.zero[row] = g.z;
    }
    const int C16 = (a.C + 15) / 16 * 16;
    auto codes = [&](int p, int c) {
      uint32_t u[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.C) u[j >> 2] |= ((uint32_t)to_code(g, s[p][j]) & 0xffu) << (8 * (j & 3));
      *reinterpret_cast<uint2*>(a.codes + row * a.ldc + c) = make_uint2(u[0], u[1]);
      if (a.y && c < a.C) store8_any<DT>(a.y, row * a.C + c, a.C - c, s[p]);
    };
    if constexpr (V > 0) {
      each([&](int p, int c) { if (c < C16) codes(p, c); });
    } else {
      for (int c = c0; c < C16; c += STEP) {
        value(0, c, true);
        codes(0, c);
      }
    }
  }
}

struct CodesArgs {
  const int8_t* codes;
  int64_t ldc, T, K;
  const float *scale, *zero;
  void* out;
  int shift;
};

// Sixteen codes a thread.  out = scale·(code − zero), rounded to its type.  Bound by the bytes:
// MI355X, 8192 × 4096 to bf16 17.5–17.8 µs (101 MB, 5.7 TB/s: the codes lie in the last cache).
template <int DT>
__global__ __launch_bounds__(256) void dequantize_tokens_kernel(CodesArgs a) {
  const int64_t c = row_cell(a.shift) * 16;
  if (c >= a.K) return;
  const int n = (int)min<int64_t>(16, a.K - c);
  for (int64_t t = row_first(a.shift); t < a.T; t += row_step(a.shift)) {
    const int8_t* p = a.codes + t * a.ldc + c;
    const float s = a.scale[t], z = a.zero ? a.zero[t] : 0.f;
    uint32_t u[4] = {0, 0, 0, 0};
    if (n == 16) {
      __builtin_memcpy(u, p, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < n) u[j >> 2] |= (uint32_t)(uint8_t)p[j] << (8 * (j & 3));
    }
    float v[2][8];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      v[j >> 3][j & 7] = s * ((float)(int8_t)(u[j >> 2] >> (8 * (j & 3))) - z);
    store8_any<DT>(a.out, t * a.K + c, n, v[0]);
    if (n > 8) store8_any<DT>(a.out, t * a.K + c + 8, n - 8, v[1]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int DT, int Q, int L, int V>
int launch_norm(hipStream_t st, NormArgs& a) {
  constexpr int PER = 256 / L;
  for (a.first = 0; a.first < a.rows; a.first += kMaxGroups * PER) {
    const dim3 grid((unsigned)std::min(cdiv(a.rows - a.first, PER), kMaxGroups));
    hipLaunchKernelGGL((rms_norm_kernel<DT, Q, L, V>), grid, dim3(256), 0, st, a);
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}

// As few lanes a row as hold it in one or two pieces each: narrow rows share a wave, and only
// those that four waves hold need barriers.  MI355X, bf16 with residual, against a workgroup a
// row: 16384 × 512 13.3 and 21.1 µs, 8192 × 1000 11.9 and 16.2 (64 × 1000 4.5 and 3.4); against a
// wave a row: 8192 × 2048 23.1 and 26.0, 8192 × 4096 57 and 97.  Rows of 8193 values and more are
// read again for each use where there are many: 2048 × 16384 61 µs, 71 with eight pieces in
// registers, 1024 × 9000 18.4 and 21.5, but 512 × 16384 19.8 and 16.1, 64 rows 11.6 and 9.4, to
// codes 16.7 and 10.8; 2048 × 8192 24.4 with four in registers and 29.8 read again.
template <int DT, int Q>
int norm_by_size(hipStream_t st, NormArgs& a) {
  if (a.C <= 64) return launch_norm<DT, Q, 8, 1>(st, a);
  if (a.C <= 128) return launch_norm<DT, Q, 16, 1>(st, a);
  if (a.C <= 256) return launch_norm<DT, Q, 32, 1>(st, a);
  if (a.C <= 512) return launch_norm<DT, Q, 64, 1>(st, a);
  if (a.C <= 1024) return launch_norm<DT, Q, 64, 2>(st, a);
  if (a.C <= 2048) return launch_norm<DT, Q, 256, 1>(st, a);
  if (a.C <= 4096) return launch_norm<DT, Q, 256, 2>(st, a);
  if (a.C <= 8192) return launch_norm<DT, Q, 256, 4>(st, a);
  if (a.C <= 16384 && a.rows <= 512) return launch_norm<DT, Q, 256, 8>(st, a);
  return launch_norm<DT, Q, 256, 0>(st, a);
}

template <int DT>
int norm_by_codes(hipStream_t st, NormArgs& a, int sym) {
  if (!a.codes) return norm_by_size<DT, 0>(st, a);
  return sym ? norm_by_size<DT, 1>(st, a) : norm_by_size<DT, 2>(st, a);
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_rms_norm(void* stream, const void* x, int64_t x_outer, int64_t x_inner,
                              const void* r, int64_t r_outer, int64_t r_inner, int dtype,
                              const void* w, int wtype, int64_t rows, int64_t inner, int64_t C,
                              float eps, void* y, void* sum, int sym, int8_t* codes, int64_t ldc,
                              float* scale, float* zero) {
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2 && wtype >= 0 && wtype <= 2,
              "rms_norm: dtype codes %d and %d", dtype, wtype);
  G2PTQ_CHECK(rows >= 0 && inner >= 1 && inner < (1ll << 31) && C >= 1 && C <= 65536,
              "rms_norm: %lld rows in groups of %lld of %lld columns (1 to 65536 columns)",
              (long long)rows, (long long)inner, (long long)C);
  G2PTQ_CHECK(eps >= 0.f && eps < __builtin_inff(), "rms_norm: eps is %g", (double)eps);
  if (rows == 0) return G2PTQ_OK;
  G2PTQ_CHECK(x && w && (y || codes), "rms_norm: null pointer");
  if (codes) {
    G2PTQ_CHECK(scale && (sym || zero), "rms_norm: null scales or zero points");
    G2PTQ_CHECK(ldc % 16 == 0 && ldc >= cdiv(C, 16) * 16 && aligned16(codes),
                "rms_norm: codes need 16-byte aligned rows of at least %lld bytes",
                (long long)(cdiv(C, 16) * 16));
  }
  NormArgs a{x, r, w, x_outer, x_inner, r_outer, r_inner, rows, 0, (uint32_t)inner, (int)C,
             wtype, eps, y, sum, codes, ldc, scale, zero};
  hipStream_t st = as_stream(stream);
  if (dtype == 0) return norm_by_codes<0>(st, a, sym);
  if (dtype == 1) return norm_by_codes<1>(st, a, sym);
  return norm_by_codes<2>(st, a, sym);
}

extern "C" int g2ptq_dequantize_tokens(void* stream, const int8_t* codes, int64_t ldc,
                                       const float* scale, const float* zero, int64_t T, int64_t K,
                                       void* out, int dtype) {
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2, "dequantize_tokens: dtype code %d", dtype);
  G2PTQ_CHECK(T >= 0 && K >= 0 && K <= 65536, "dequantize_tokens: %lld tokens of %lld columns",
              (long long)T, (long long)K);
  if (T == 0 || K == 0) return G2PTQ_OK;
  G2PTQ_CHECK(codes && scale && out, "dequantize_tokens: null pointer");
  const RowLaunch l = row_launch(cdiv(K, 16), T);
  CodesArgs a{codes, ldc, T, K, scale, zero, out};
  a.shift = l.shift;
  hipStream_t st = as_stream(stream);
#define G2_DQ(DT) \
  hipLaunchKernelGGL((dequantize_tokens_kernel<DT>), l.grid, dim3(256), 0, st, a)
  if (dtype == 0) G2_DQ(0);
  else if (dtype == 1) G2_DQ(1);
  else G2_DQ(2);
#undef G2_DQ
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}
