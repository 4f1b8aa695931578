// Linears in 8-bit integers.
//
//   tokens:   s_t, z_t and codes c[t][k] of every token's row on the grid of
//             grid8.hpp with 8 bits (z_t = 0 in the symmetric grid)
//   product:  Y[t][n] = s_t·w_n·(Σ_k c[t][k]·W[n][k] − z_t·Σ_k W[n][k]) + b_n
//
// The sums are exact 32-bit integers (|c − z| ≤ 255, |W| ≤ 128 and K ≤ 65536
// stay below 2^31) and are scaled in fp32, so the result does not depend on
// the order of summation.
#include <algorithm>

#include "grid8.hpp"

namespace g2ptq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int64_t kMaxK = 65536;

// ---------------------------------------------------------------------------
// Token quantiser: one workgroup per token.  Codes are written in rows of ldc
// bytes, columns from K up to the next multiple of 16 as zeros.
// ---------------------------------------------------------------------------
template <int DT, bool SYM>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(const void* __restrict__ x,
                                                              int64_t K, int64_t ldx, bool vec,
                                                              int8_t* __restrict__ codes,
                                                              int64_t ldc, float* scale,
                                                              float* zero) {
  __shared__ float slo[4], shi[4];
  __shared__ uint32_t stop[4];
  const int64_t t = blockIdx.x, row = t * ldx;
  Range r;
  for (int64_t k = threadIdx.x * 8; k < K; k += 256 * 8) {
    float v[8];
    load8<DT>(x, row + k, vec, (int)min<int64_t>(8, K - k), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.add(v[i]);
  }
  reduce_range<64>(r);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) slo[wave] = r.lo, shi[wave] = r.hi, stop[wave] = r.top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) r.merge(slo[w], shi[w], stop[w]);
  const Grid g = make_grid<SYM>(r, 8);
  if (threadIdx.x == 0) {
    scale[t] = g.s;
    if (!SYM) zero[t] = g.z;
  }
  const int64_t K16 = (K + 15) / 16 * 16;
  for (int64_t k = threadIdx.x * 8; k < K16; k += 256 * 8) {
    float v[8];
    const int n = (int)min<int64_t>(8, K - k);
    load8<DT>(x, row + k, vec, n, v);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i >> 2] |= ((uint32_t)to_code(g, v[i]) & 0xffu) << (8 * (i & 3));
    *reinterpret_cast<uint2*>(codes + t * ldc + k) = make_uint2(w[0], w[1]);
  }
}

// ---------------------------------------------------------------------------
// Product: one workgroup of four waves computes a 64 × 64 tile (tokens ×
// channels), 32 × 32 per wave, in steps of 64 columns through LDS.
// ---------------------------------------------------------------------------
struct GemmI8 {
  const int8_t* A;  // codes, T rows of lda bytes, readable to the next multiple of 16 columns
  int64_t lda;
  const int8_t* W;  // weights, N rows of ldw bytes, zero from K to the next multiple of 16
  int64_t ldw;
  const float *sx, *zx, *sw, *bias;
  const int32_t* wsum;
  void* out;
  int64_t T, N, K, ldo;
  int dtype;
};

// Y[t][n] from the integer sum.
__device__ __forceinline__ void finish(const GemmI8& a, int64_t t, int64_t n, int acc) {
  if (a.zx) acc = (int)((uint32_t)acc - (uint32_t)(int)a.zx[t] * (uint32_t)a.wsum[n]);
  float y = __fmul_rn(__fmul_rn((float)acc, a.sx[t]), a.sw[n]);
  if (a.bias) y = __fadd_rn(y, a.bias[n]);
  const int64_t o = t * a.ldo + n;
  if (a.dtype == 0) static_cast<uint16_t*>(a.out)[o] = __builtin_bit_cast(uint16_t, (__bf16)y);
  else if (a.dtype == 1) static_cast<_Float16*>(a.out)[o] = (_Float16)y;
  else static_cast<float*>(a.out)[o] = y;
}

__global__ __launch_bounds__(256) void gemm_i8_kernel(GemmI8 a) {
  __shared__ __attribute__((aligned(16))) int8_t As[64 * 80], Ws[64 * 80];
  const int64_t t0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1, lr = lane & 31, lh = lane >> 5;
  const int row = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
  const int64_t K16 = (a.K + 15) / 16 * 16;
  i32x16 acc;
#pragma unroll
  for (int v = 0; v < 16; ++v) acc[v] = 0;
  for (int64_t k = 0; k < K16; k += 64) {
    uint4 av = make_uint4(0, 0, 0, 0), wv = av;
    if (t0 + row < a.T && k + c < K16)
      av = *reinterpret_cast<const uint4*>(a.A + (t0 + row) * a.lda + k + c);
    if (n0 + row < a.N && k + c < K16)
      wv = *reinterpret_cast<const uint4*>(a.W + (n0 + row) * a.ldw + k + c);
    *reinterpret_cast<uint4*>(As + row * 80 + c) = av;
    *reinterpret_cast<uint4*>(Ws + row * 80 + c) = wv;
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const i32x4 x = *reinterpret_cast<const i32x4*>(As + (wm * 32 + lr) * 80 + ks * 32 + lh * 16);
      const i32x4 w = *reinterpret_cast<const i32x4*>(Ws + (wn * 32 + lr) * 80 + ks * 32 + lh * 16);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(x, w, acc, 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t t = t0 + wm * 32 + 8 * (v >> 2) + 4 * lh + (v & 3), n = n0 + wn * 32 + lr;
    if (t < a.T && n < a.N) finish(a, t, n, acc[v]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int quantize_tokens(hipStream_t st, const void* x, int dtype, int64_t T, int64_t K, int64_t ldx,
                    int sym, int8_t* codes, int64_t ldc, float* scale, float* zero) {
  const bool vec = aligned16(x) && ldx * (dtype == 2 ? 4 : 2) % 16 == 0;
#define G2_QT(DT, SYM)                                                                       \
  hipLaunchKernelGGL((quantize_tokens_kernel<DT, SYM>), dim3((unsigned)T), dim3(256), 0, st, \
                     x, K, ldx, vec, codes, ldc, scale, zero)
  if (dtype == 0) { if (sym) G2_QT(0, true); else G2_QT(0, false); }
  else if (dtype == 1) { if (sym) G2_QT(1, true); else G2_QT(1, false); }
  else { if (sym) G2_QT(2, true); else G2_QT(2, false); }
#undef G2_QT
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}

int gemm_i8(hipStream_t st, const GemmI8& a) {
  hipLaunchKernelGGL(gemm_i8_kernel, dim3((unsigned)cdiv(a.N, 64), (unsigned)cdiv(a.T, 64)),
                     dim3(256), 0, st, a);
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}

int check_tokens(const char* who, const void* x, int dtype, int64_t T, int64_t K, int64_t ldx) {
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype code %d", who, dtype);
  G2PTQ_CHECK(T >= 0 && T < (1ll << 22) && K >= 1 && K <= kMaxK,
              "%s: %lld tokens of %lld columns (fewer than 4194304 tokens of 1 to %lld columns)",
              who, (long long)T, (long long)K, (long long)kMaxK);
  G2PTQ_CHECK(T == 0 || (x && ldx >= K), "%s: null tokens or a row stride below %lld", who,
              (long long)K);
  return G2PTQ_OK;
}

int check_product(const char* who, const GemmI8& a) {
  G2PTQ_CHECK(a.dtype >= 0 && a.dtype <= 2, "%s: dtype code %d", who, a.dtype);
  G2PTQ_CHECK(a.T >= 0 && a.T < (1ll << 22) && a.K >= 1 && a.K <= kMaxK && a.N >= 0 &&
                  a.N < (1ll << 31),
              "%s: %lld tokens × %lld columns × %lld channels", who, (long long)a.T,
              (long long)a.K, (long long)a.N);
  if (a.T == 0 || a.N == 0) return G2PTQ_OK;
  G2PTQ_CHECK(a.W && a.sw && a.out && a.ldo >= a.N, "%s: null pointer or output stride", who);
  const int64_t K16 = cdiv(a.K, 16) * 16;
  G2PTQ_CHECK(a.ldw >= K16 && a.ldw % 16 == 0 && aligned16(a.W),
              "%s: weights need 16-byte aligned rows of at least %lld bytes", who, (long long)K16);
  return G2PTQ_OK;
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_quantize_tokens(void* stream, const void* x, int dtype, int64_t T, int64_t K,
                                     int64_t ldx, int sym, int8_t* codes, int64_t ldc,
                                     float* scale, float* zero) {
  G2PTQ_TRY(check_tokens("quantize_tokens", x, dtype, T, K, ldx));
  if (T == 0) return G2PTQ_OK;
  G2PTQ_CHECK(codes && scale && (sym || zero), "quantize_tokens: null output");
  G2PTQ_CHECK(ldc % 16 == 0 && ldc >= cdiv(K, 16) * 16 && aligned16(codes),
              "quantize_tokens: codes need 16-byte aligned rows of at least %lld bytes",
              (long long)(cdiv(K, 16) * 16));
  return quantize_tokens(as_stream(stream), x, dtype, T, K, ldx, sym, codes, ldc, scale, zero);
}

extern "C" int g2ptq_int8_gemm_workspace(int64_t T, int64_t N, int64_t K, size_t* bytes) {
  G2PTQ_CHECK(bytes && T >= 0 && N >= 0 && K >= 1 && K <= kMaxK, "int8_gemm_workspace: bad sizes");
  *bytes = 0;
  return G2PTQ_OK;
}

extern "C" int g2ptq_int8_gemm(void* stream, const int8_t* codes, int64_t ldc, const float* scale,
                               const float* zero, const int8_t* W, int64_t ldw,
                               const float* wscale, const int32_t* wsum, const float* bias,
                               int64_t T, int64_t N, int64_t K, void* out, int dtype, int64_t ldo,
                               void* ws, size_t ws_bytes) {
  GemmI8 a{codes, ldc, W, ldw, scale, zero, wscale, bias, wsum, out, T, N, K, ldo, dtype};
  G2PTQ_TRY(check_product("int8_gemm", a));
  if (T == 0 || N == 0) return G2PTQ_OK;
  G2PTQ_CHECK(codes && scale && (!zero || wsum), "int8_gemm: null codes, scales or weight sums");
  G2PTQ_CHECK(ldc % 16 == 0 && ldc >= cdiv(K, 16) * 16 && aligned16(codes),
              "int8_gemm: codes need 16-byte aligned rows of at least %lld bytes",
              (long long)(cdiv(K, 16) * 16));
  return gemm_i8(as_stream(stream), a);
}

namespace {
// Workspace of g2ptq_int8_linear: codes, scales, zero points, then the product's.
struct LinearWs {
  int64_t ldc, codes, scale, zero, gemm;
  LinearWs(int64_t T, int64_t K) {
    ldc = cdiv(K, 16) * 16;
    codes = 0;
    scale = cdiv(T * ldc, 256) * 256;
    zero = scale + cdiv(T * 4, 256) * 256;
    gemm = zero + cdiv(T * 4, 256) * 256;
  }
};
}  // namespace

extern "C" int g2ptq_int8_linear_workspace(int64_t T, int64_t N, int64_t K, size_t* bytes) {
  G2PTQ_CHECK(T >= 0 && K >= 1, "int8_linear_workspace: bad sizes");
  G2PTQ_TRY(g2ptq_int8_gemm_workspace(T, N, K, bytes));
  *bytes += (size_t)LinearWs(T, K).gemm;
  return G2PTQ_OK;
}

extern "C" int g2ptq_int8_linear(void* stream, const void* x, int dtype, int64_t T, int64_t K,
                                 int64_t ldx, int sym, const int8_t* W, int64_t ldw,
                                 const float* wscale, const int32_t* wsum, const float* bias,
                                 int64_t N, void* out, int64_t ldo, void* ws, size_t ws_bytes) {
  G2PTQ_TRY(check_tokens("int8_linear", x, dtype, T, K, ldx));
  GemmI8 a{nullptr, 0, W, ldw, nullptr, nullptr, wscale, bias, wsum, out, T, N, K, ldo, dtype};
  G2PTQ_TRY(check_product("int8_linear", a));
  if (T == 0 || N == 0) return G2PTQ_OK;
  G2PTQ_CHECK(sym || wsum, "int8_linear: asymmetric tokens need the weights' sums");
  size_t need;
  G2PTQ_TRY(g2ptq_int8_linear_workspace(T, N, K, &need));
  if (!ws || ws_bytes < need) {
    set_error("int8_linear: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return G2PTQ_ERR_WORKSPACE;
  }
  G2PTQ_CHECK(aligned16(ws), "int8_linear: workspace not 16-byte aligned");
  const LinearWs l(T, K);
  char* base = static_cast<char*>(ws);
  int8_t* codes = reinterpret_cast<int8_t*>(base + l.codes);
  float* scale = reinterpret_cast<float*>(base + l.scale);
  float* zero = sym ? nullptr : reinterpret_cast<float*>(base + l.zero);
  hipStream_t st = as_stream(stream);
  G2PTQ_TRY(quantize_tokens(st, x, dtype, T, K, ldx, sym, codes, l.ldc, scale, zero));
  a.A = codes, a.lda = l.ldc, a.sx = scale, a.zx = zero;
  return gemm_i8(st, a);
}
