// Linears in 8-bit integers.
//
//   tokens:   s_t, z_t and codes c[t][k] of every token's row on the grid of
//             grid8.hpp with 8 bits (z_t = 0 in the symmetric grid)
//   product:  Y[t][n] = s_t·w_n·(Σ_k c[t][k]·W[n][k] − z_t·Σ_k W[n][k]) + b_n
//
// The sums are exact 32-bit integers (|c − z| ≤ 255, |W| ≤ 128 and K ≤ 65536
// stay below 2^31) and are scaled in fp32, so the result does not depend on
// the order of summation.  A sum is rounded to fp32 once (2^-24 of it), then by the
// scales' products and to the output's type.
#include <algorithm>
#include <type_traits>

#include "grid8.hpp"

namespace g2ptq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int64_t kMaxK = 65536;

// ---------------------------------------------------------------------------
// Token quantiser: one workgroup per token, its row in registers between the range and
// the codes where it fits (V pieces of eight values per thread; V = 0: read again).
// Codes are written in rows of ldc bytes, columns from K up to the next multiple of 16
// as zeros.  Bound by memory for many tokens (MI355X, 8192 × 4096 bf16 18.2 µs, 5.5 TB/s),
// by latency for few (64 × 4096 3.4 µs).
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint2 eight_codes(const Grid& g, const float (&v)[8], int n) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 2] |= ((uint32_t)to_code(g, v[i]) & 0xffu) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

template <int DT, bool SYM, int V>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(const void* __restrict__ x, int K,
                                                              int64_t ldx, bool vec,
                                                              int8_t* __restrict__ codes,
                                                              int64_t ldc, float* scale,
                                                              float* zero) {
  __shared__ float slo[4], shi[4];
  __shared__ uint32_t stop[4];
  const int64_t t = blockIdx.x, row = t * ldx;
  const int k0 = threadIdx.x * 8;
  float v[V ? V : 1][8];
  Range<SYM> r;
  if constexpr (V > 0) {
#pragma unroll
    for (int p = 0; p < V; ++p) load8<DT>(x, row + k0 + p * 2048, vec, K - k0 - p * 2048, v[p]);
#pragma unroll
    for (int p = 0; p < V; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) r.add(v[p][i]);
  } else {
    for (int k = k0; k < K; k += 2048) {
      load8<DT>(x, row + k, vec, K - k, v[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.add(v[0][i]);
    }
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
  const int K16 = (K + 15) / 16 * 16;
  if constexpr (V > 0) {
#pragma unroll
    for (int p = 0; p < V; ++p) {
      const int k = k0 + p * 2048;
      if (k < K16) *reinterpret_cast<uint2*>(codes + t * ldc + k) = eight_codes(g, v[p], K - k);
    }
  } else {
    for (int k = k0; k < K16; k += 2048) {
      load8<DT>(x, row + k, vec, K - k, v[0]);
      *reinterpret_cast<uint2*>(codes + t * ldc + k) = eight_codes(g, v[0], K - k);
    }
  }
}

// ---------------------------------------------------------------------------
// Products.  v_mfma_i32_*_i8: both operands' rows run along K, so that a lane's
// 16 bytes of a row are its operand as they lie in memory.
// ---------------------------------------------------------------------------
struct GemmI8 {
  const int8_t* A;  // codes, T rows of lda bytes, readable to the next multiple of 16 columns
  int64_t lda;
  const int8_t* W;  // weights, N rows of ldw bytes, zero from K to the next multiple of 256
  int64_t ldw;
  const float *sx, *zx, *sw, *bias;
  const int32_t* wsum;
  void* out;
  int64_t T, N, K, ldo;
  int dtype;
};

// Y[t][n] from the integer sum.
__device__ __forceinline__ float scaled(const GemmI8& a, float sx, int zx, int acc, float sw,
                                        int wsum, float bias) {
  acc = (int)((uint32_t)acc - (uint32_t)zx * (uint32_t)wsum);
  return __fadd_rn(__fmul_rn(__fmul_rn((float)acc, sx), sw), bias);
}
__device__ __forceinline__ void store_y(const GemmI8& a, int64_t o, float y) {
  if (a.dtype == 0) static_cast<uint16_t*>(a.out)[o] = __builtin_bit_cast(uint16_t, (__bf16)y);
  else if (a.dtype == 1) static_cast<_Float16*>(a.out)[o] = (_Float16)y;
  else static_cast<float*>(a.out)[o] = y;
}

// Tiles of BM tokens × BN channels by WM × WN waves, 32×32 products.  K advances 128
// bytes a stage through two LDS buffers; the loads of a stage are issued two stages
// ahead into registers and written to the other buffer during the products, one
// barrier a stage.  LDS rows are 128 bytes, the 16-byte chunk c of row r at
// c ^ f(r), f(r) = (r & 7) ^ ((r >> 3) & 1): fragment reads (16 consecutive rows, one
// chunk) are free of bank conflicts.  S > 1: S groups of waves share K and add their
// integer sums in LDS (tiles too few for the chip, which then wait for each stage's loads).
// Tiles of 256 × 256 are bound by the matrix cores, with clocks as the power allows (MI355X,
// the product alone under the profiler, fastest and average: 8192 × 14336 × 4096 424 and 485
// µs, 2.0–2.27 POP/s; a large library product reaches 2.35); small ones by the latency of
// their stages and of the launch (777 × 1000 × 2752 11.4 and 12.4 µs; 48 × 14336 × 4096 12.8
// and 14.1 µs, 4.2–4.6 TB/s of weights).
constexpr int KS = 128;
__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// A wave's rows × columns of the tile: scaled, turned in LDS (its own part of it) so that
// rows are written in 16-byte pieces.  32×32 output: lane holds rows
// 8(v/4) + 4·(lane/32) + v%4 of column lane%32.
template <int DT, int MT, int NTL>
__device__ __forceinline__ void finish_tile(const GemmI8& a, const i32x16 (&acc)[MT][NTL],
                                            int64_t t0, int64_t n0, const float* sxL,
                                            const int* zxL, int8_t* mine, int lane) {
  // (also read back as what was written: another scalar type could be read before the writes)
  using Out = std::conditional_t<DT == 0, __bf16, std::conditional_t<DT == 1, _Float16, float>>;
  constexpr int E = sizeof(Out), BYTES = NTL * 32 * E, PITCH = BYTES + 16;
  constexpr int LPR = BYTES / 16, RPP = 64 / LPR;  // lanes of a row, rows of a pass
  const int lr = lane & 31, lh = lane >> 5;
  float sw[NTL], bias[NTL];
  int wsum[NTL];
#pragma unroll
  for (int n = 0; n < NTL; ++n) {
    const int64_t j = min<int64_t>(n0 + n * 32 + lr, a.N - 1);
    sw[n] = a.sw[j];
    bias[n] = a.bias ? a.bias[j] : 0.f;
    wsum[n] = a.zx ? a.wsum[j] : 0;
  }
  const bool whole = n0 + NTL * 32 <= a.N && a.ldo * E % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int r = 8 * (v >> 2) + 4 * lh + (v & 3);
      const float sx = sxL[m * 32 + r];
      const int zx = zxL[m * 32 + r];
#pragma unroll
      for (int n = 0; n < NTL; ++n) {
        const float y = scaled(a, sx, zx, acc[m][n][v], sw[n], wsum[n], bias[n]);
        *reinterpret_cast<Out*>(mine + r * PITCH + (n * 32 + lr) * E) = (Out)y;
      }
    }
    __builtin_amdgcn_wave_barrier();
    int8_t* out = static_cast<int8_t*>(a.out) + ((t0 + m * 32) * a.ldo + n0) * E;
    const int rows = (int)min<int64_t>(32, a.T - t0 - m * 32);
    if (whole) {
#pragma unroll
      for (int p = 0; p < 32 / RPP; ++p) {
        const int r = p * RPP + lane / LPR, c = lane % LPR * 16;
        if (r < rows)
          *reinterpret_cast<i32x4*>(out + r * a.ldo * E + c) =
              *reinterpret_cast<const i32x4*>(mine + r * PITCH + c);
      }
    } else {
      const int cols = (int)min<int64_t>(NTL * 32, a.N - n0);
      for (int i = lane; i < 32 * NTL * 32; i += 64) {
        const int r = i / (NTL * 32), c = i % (NTL * 32);
        if (r < rows && c < cols)
          *reinterpret_cast<Out*>(out + (r * a.ldo + c) * E) =
              *reinterpret_cast<const Out*>(mine + r * PITCH + c * E);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN * S) void gemm_i8_kernel(GemmI8 a, int tm, int tn) {
  constexpr int NT = 64 * WM * WN;                      // threads of a group
  constexpr int MT = BM / WM / 32, NTL = BN / WN / 32;  // 32×32 tiles of a wave
  constexpr int AL = BM * 8 / NT, BL = BN * 8 / NT;     // 16-byte loads of a thread per stage
  __shared__ __attribute__((aligned(16))) int8_t Lall[S][2][(BM + BN) * KS];
  __shared__ float sxL[BM];
  __shared__ int zxL[BM];

  // Workgroups go round the 8 XCDs: an XCD takes a contiguous range of tiles, in bands of
  // eight token tiles walked channel tile by channel tile.
  const int total = tm * tn;
  int id;
  {
    const int q8 = total >> 3, r8 = total & 7, xcd = blockIdx.x & 7;
    id = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
  }
  const int band = id / (8 * tn), in = id - band * 8 * tn, h = min(8, tm - band * 8);
  const int64_t t0 = (int64_t)(band * 8 + in % h) * BM, n0 = (int64_t)(in / h) * BN;

  const int group = S == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  const int tid = (int)threadIdx.x - group * NT, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, lh = lane >> 5, wm = wave / WN, wn = wave % WN;
  int8_t(&Ls)[2][(BM + BN) * KS] = Lall[group];
  if ((int)threadIdx.x < BM) {
    const int64_t i = min<int64_t>(t0 + threadIdx.x, a.T - 1);
    sxL[threadIdx.x] = a.sx[i];
    zxL[threadIdx.x] = a.zx ? (int)a.zx[i] : 0;
  }
  const int row = tid >> 3, c = tid & 7;  // load i: row + i·NT/8
  const int8_t* Ab = a.A + t0 * a.lda;
  const int8_t* Wb = a.W + n0 * a.ldw;
  uint32_t aoff[AL], boff[BL];  // (rows past the end read the last row)
#pragma unroll
  for (int i = 0; i < AL; ++i)
    aoff[i] = (uint32_t)min<int64_t>(row + i * (NT / 8), a.T - 1 - t0) * (uint32_t)a.lda;
#pragma unroll
  for (int i = 0; i < BL; ++i)
    boff[i] = (uint32_t)min<int64_t>(row + i * (NT / 8), a.N - 1 - n0) * (uint32_t)a.ldw + c * 16;
  const int lpos = row * KS + ((c ^ swz(row)) << 4);  // (NT/8 is a multiple of 16)
  const uint32_t klast = (uint32_t)((a.K + 15) / 16 * 16 - 16);
  // stages, even in number (weights are zero past K), and the group's share of them
  const int all = (int)((a.K + 255) / 256 * 2);
  const int each = S == 1 ? all : (all + 2 * S - 1) / (2 * S) * 2;
  const int first = group * each, nk = min(first + each, all);
  i32x4 xa[AL], xb[BL], ya[AL], yb[BL];
#define G2_LOAD(R, st)                                                              \
  do {                                                                              \
    const uint32_t k_ = (uint32_t)min(st, all - 1) * KS;                            \
    const uint32_t ka_ = min(k_ + c * 16, klast);                                   \
    _Pragma("unroll") for (int i = 0; i < AL; ++i)                                  \
      R##a[i] = *reinterpret_cast<const i32x4*>(Ab + (aoff[i] + ka_));              \
    _Pragma("unroll") for (int i = 0; i < BL; ++i)                                  \
      R##b[i] = *reinterpret_cast<const i32x4*>(Wb + (boff[i] + k_));               \
  } while (0)
#define G2_STORE(R, buf)                                                            \
  do {                                                                              \
    _Pragma("unroll") for (int i = 0; i < AL; ++i)                                  \
      *reinterpret_cast<i32x4*>(&Ls[buf][lpos + i * (NT / 8) * KS]) = R##a[i];      \
    _Pragma("unroll") for (int i = 0; i < BL; ++i)                                  \
      *reinterpret_cast<i32x4*>(&Ls[buf][BM * KS + lpos + i * (NT / 8) * KS]) = R##b[i]; \
  } while (0)
  i32x16 acc[MT][NTL];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NTL; ++n)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[m][n][v] = 0;
#define G2_MMA(buf)                                                                       \
  do {                                                                                    \
    const int8_t* As_ = Ls[buf];                                                          \
    const int8_t* Bs_ = Ls[buf] + BM * KS;                                                \
    _Pragma("unroll") for (int ks = 0; ks < KS / 32; ++ks) {                              \
      const int c_ = ks * 2 + lh;                                                         \
      i32x4 av[MT], bv[NTL];                                                              \
      _Pragma("unroll") for (int m = 0; m < MT; ++m) {                                    \
        const int r_ = wm * (BM / WM) + m * 32 + lr;                                      \
        av[m] = *reinterpret_cast<const i32x4*>(As_ + r_ * KS + ((c_ ^ swz(r_)) << 4));   \
      }                                                                                   \
      _Pragma("unroll") for (int n = 0; n < NTL; ++n) {                                   \
        const int r_ = wn * (BN / WN) + n * 32 + lr;                                      \
        bv[n] = *reinterpret_cast<const i32x4*>(Bs_ + r_ * KS + ((c_ ^ swz(r_)) << 4));   \
      }                                                                                   \
      _Pragma("unroll") for (int m = 0; m < MT; ++m)                                      \
      _Pragma("unroll") for (int n = 0; n < NTL; ++n)                                     \
        acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[m], bv[n], acc[m][n], 0, 0, 0); \
    }                                                                                     \
  } while (0)
  // Spreads a stage's LDS writes and loads over its products (256 × 256: 32 products, 8
  // writes, 8 loads, 24 reads a wave).
#define G2_PATTERN()                                                                      \
  do {                                                                                    \
    if constexpr (MT == 4 && NTL == 2) {                                                  \
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0); /* DS read  */                   \
      _Pragma("unroll") for (int r_ = 0; r_ < 8; ++r_) {                                  \
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0); /* MFMA */                     \
        __builtin_amdgcn_sched_group_barrier(0x200, 1, 0); /* DS write */                 \
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                \
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); /* VMEM read */                \
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                \
        if (r_ < 6) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);                    \
      }                                                                                   \
    }                                                                                     \
    __builtin_amdgcn_sched_barrier(0);                                                    \
  } while (0)
  G2_LOAD(x, first);
  G2_STORE(x, 0);
  G2_LOAD(x, first + 1);
  G2_LOAD(y, first + 2);
  __syncthreads();
  for (int kt = first; kt < first + each; kt += 2) {
    __builtin_amdgcn_sched_barrier(0);
    if (S == 1 || kt < nk) G2_MMA(0);      // stage kt
    G2_STORE(x, 1);  // stage kt + 1
    G2_LOAD(x, kt + 3);
    G2_PATTERN();
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    if (S == 1 || kt < nk) G2_MMA(1);      // stage kt + 1
    G2_STORE(y, 0);  // stage kt + 2
    G2_LOAD(y, kt + 4);
    G2_PATTERN();
    __syncthreads();
  }
#undef G2_LOAD
#undef G2_STORE
#undef G2_MMA
#undef G2_PATTERN
  if constexpr (S > 1) {  // the groups' sums, in the first group's registers
    int* sums = reinterpret_cast<int*>(&Lall[0][0][0]);
    constexpr int TILE = MT * NTL * 16 * NT;
    static_assert((S - 1) * TILE * 4 <= (int)sizeof(Lall), "sums do not fit");
    if (group > 0)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NTL; ++n)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            sums[(group - 1) * TILE + ((m * NTL + n) * 16 + v) * NT + tid] = acc[m][n][v];
    __syncthreads();
    if (group == 0)
#pragma unroll
      for (int g = 0; g < S - 1; ++g)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NTL; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v)
              acc[m][n][v] += sums[g * TILE + ((m * NTL + n) * 16 + v) * NT + tid];
    __syncthreads();
    if (group > 0) return;
  }
  constexpr int MINE = 32 * (NTL * 32 * 4 + 16);  // a wave's part of LDS
  static_assert(WM * WN * MINE <= (int)sizeof(Lall), "output does not fit");
  int8_t* mine = &Lall[0][0][0] + wave * MINE;
  const int64_t tw = t0 + wm * (BM / WM), nw = n0 + wn * (BN / WN);
  const float* sx = sxL + wm * (BM / WM);
  const int* zx = zxL + wm * (BM / WM);
  if (nw >= a.N) return;
  if (a.dtype == 0) finish_tile<0, MT, NTL>(a, acc, tw, nw, sx, zx, mine, lane);
  else if (a.dtype == 1) finish_tile<1, MT, NTL>(a, acc, tw, nw, sx, zx, mine, lane);
  else finish_tile<2, MT, NTL>(a, acc, tw, nw, sx, zx, mine, lane);
}

// Few tokens (TB blocks of 16): the weights' bytes are what counts.  A workgroup takes
// 16·R channels; its eight waves take turns at blocks of 128 columns, with weights and
// codes straight from memory into v_mfma_i32_16x16x64_i8 (channels × tokens: lane
// (n, g) holds 16 bytes of row n at 16·g of 64 columns, so that a load covers 64
// consecutive bytes of 16 rows).  The waves' integer sums meet in LDS.
// FUSED: the tokens themselves are quantized here, by every workgroup, into LDS (one or
// two tokens: cheaper than another launch before this one).
// Bound by the weights' bytes and, where those are few, by the launch and the latency of
// the first loads: MI355X, back to back over weights that no cache holds, one token fused,
// 4096 × 4096 9.4 µs (1.8 TB/s; 6.7 where the last cache holds them), 14336 × 4096 17 µs
// (3.5 TB/s), 8192 × 28672 55 µs (4.3 TB/s); 16 tokens and their quantiser, 14336 × 4096 21 µs.
template <int R, int TB, bool FUSED, int DT, bool SYM>
__global__ __launch_bounds__(512) void gemm_i8_few_kernel(GemmI8 a, const void* __restrict__ x,
                                                          int64_t ldx, bool vec) {
  constexpr int NW = 8;
  extern __shared__ __attribute__((aligned(16))) int8_t cL[];  // FUSED: T rows of K256 codes
  __shared__ __attribute__((aligned(16))) int sL[NW][TB * 16][R * 16 + 4];
  __shared__ float sxL[FUSED ? 16 : 1], zxL[FUSED ? 16 : 1];
  __shared__ float rlo[NW], rhi[NW];
  __shared__ uint32_t rtop[NW];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * R);
  const int nb = (int)((a.K + 255) / 256 * 2);  // blocks of 128 columns; weights are zero past K
  const int K256 = nb * 128;
  const int8_t* wrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    wrow[r] = a.W + min<int64_t>(n0 + 16 * r + n, a.N - 1) * a.ldw + g * 16;
  // the first weights are on their way while the tokens are prepared
  i32x4 w0[R][2], w1[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w0[r][i] = *reinterpret_cast<const i32x4*>(wrow[r] + min(wave, nb - 1) * 128 + i * 64);
      w1[r][i] = *reinterpret_cast<const i32x4*>(wrow[r] + min(wave + NW, nb - 1) * 128 + i * 64);
    }
  if constexpr (FUSED) {
    for (int t = 0; t < (int)a.T; ++t) {
      Range<SYM> r;
      for (int k = tid * 8; k < a.K; k += 512 * 8) {
        float v[8];
        load8<DT>(x, t * ldx + k, vec, min(8, (int)a.K - k), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.add(v[i]);
      }
      reduce_range<64>(r);
      if (lane == 0) rlo[wave] = r.lo, rhi[wave] = r.hi, rtop[wave] = r.top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) r.merge(rlo[w], rhi[w], rtop[w]);
      const Grid gr = make_grid<SYM>(r, 8);
      if (tid == 0) sxL[t] = gr.s, zxL[t] = gr.z;
      for (int k = tid * 8; k < K256; k += 512 * 8) {
        float v[8];
        load8<DT>(x, t * ldx + k, vec, (int)a.K - k, v);
        *reinterpret_cast<uint2*>(cL + t * K256 + k) = eight_codes(gr, v, (int)a.K - k);
      }
      __syncthreads();
    }
  }
  const int8_t* arow[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int64_t t = min<int64_t>(16 * b + n, a.T - 1);
    arow[b] = FUSED ? cL + t * K256 + g * 16 : a.A + t * a.lda;
  }
  const int klast = (int)((a.K + 15) / 16 * 16 - 16);
  i32x4 acc[R][TB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[r][b] = i32x4{0, 0, 0, 0};
#define G2_FEW(W, blk)                                                                         \
  do {                                                                                         \
    i32x4 x_[TB][2];                                                                           \
    _Pragma("unroll") for (int b = 0; b < TB; ++b)                                             \
    _Pragma("unroll") for (int i = 0; i < 2; ++i)                                              \
      x_[b][i] = *reinterpret_cast<const i32x4*>(                                              \
          arow[b] + (FUSED ? (blk) * 128 + i * 64 : min((blk) * 128 + i * 64 + g * 16, klast))); \
    _Pragma("unroll") for (int i = 0; i < 2; ++i)                                              \
    _Pragma("unroll") for (int r = 0; r < R; ++r)                                              \
    _Pragma("unroll") for (int b = 0; b < TB; ++b)                                             \
      acc[r][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(W[r][i], x_[b][i], acc[r][b], 0, 0, 0); \
    if ((blk) + 2 * NW < nb) {                                                                 \
      _Pragma("unroll") for (int r = 0; r < R; ++r)                                            \
      _Pragma("unroll") for (int i = 0; i < 2; ++i)                                            \
        W[r][i] = *reinterpret_cast<const i32x4*>(wrow[r] + ((blk) + 2 * NW) * 128 + i * 64);  \
    }                                                                                          \
  } while (0)
  for (int blk = wave; blk < nb; blk += 2 * NW) {
    G2_FEW(w0, blk);
    if (blk + NW < nb) G2_FEW(w1, blk + NW);
  }
#undef G2_FEW
  // lane holds channels 4g .. 4g + 3 of token n
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b)
      *reinterpret_cast<i32x4*>(&sL[wave][16 * b + n][16 * r + 4 * g]) = acc[r][b];
  __syncthreads();
  for (int i = tid; i < (int)a.T * 4 * R; i += 512) {
    const int t = i / (4 * R), j = i % (4 * R) * 4;
    i32x4 s = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) s += *reinterpret_cast<const i32x4*>(&sL[w][t][j]);
    const float sx = FUSED ? sxL[t] : a.sx[t];
    const int zx = FUSED ? (int)zxL[t] : a.zx ? (int)a.zx[t] : 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t ch = n0 + j + v;
      if (ch < a.N)
        store_y(a, t * a.ldo + ch,
                scaled(a, sx, zx, s[v], a.sw[ch], zx != 0 ? a.wsum[ch] : 0,
                       a.bias ? a.bias[ch] : 0.f));
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int quantize_tokens(hipStream_t st, const void* x, int dtype, int64_t T, int64_t K, int64_t ldx,
                    int sym, int8_t* codes, int64_t ldc, float* scale, float* zero) {
  const bool vec = aligned16(x) && ldx * (dtype == 2 ? 4 : 2) % 16 == 0;
#define G2_QV(DT, SYM, V)                                                                       \
  hipLaunchKernelGGL((quantize_tokens_kernel<DT, SYM, V>), dim3((unsigned)T), dim3(256), 0, st, \
                     x, (int)K, ldx, vec, codes, ldc, scale, zero)
#define G2_QT(DT, SYM)                     \
  do {                                      \
    if (K <= 4096) G2_QV(DT, SYM, 2);       \
    else if (K <= 8192) G2_QV(DT, SYM, 4);  \
    else if (K <= 16384) G2_QV(DT, SYM, 8); \
    else G2_QV(DT, SYM, 0);                 \
  } while (0)
  if (dtype == 0) { if (sym) G2_QT(0, true); else G2_QT(0, false); }
  else if (dtype == 1) { if (sym) G2_QT(1, true); else G2_QT(1, false); }
  else { if (sym) G2_QT(2, true); else G2_QT(2, false); }
#undef G2_QV
#undef G2_QT
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}

// Channels of a workgroup of few tokens, /16: enough workgroups for every CU first, then
// fewer workgroups that read the codes again.  MI355X, 16 tokens, K 4096, 1 / 2 / 4:
// 4096 channels 12.0 / 12.7 / 16.4 µs, 8192 16.5 / 15.2 / 18.1, 14336 24.7 / 22.4 / 20.4.
int few_rows(int64_t N) { return N >= 16 * 4 * 192 ? 4 : N >= 16 * 2 * 192 ? 2 : 1; }

// Whether the weights are streamed for few tokens or tiled: up to 32 tokens, and up to 64
// where 64-channel tiles would leave half the CUs idle.  MI355X, streamed against tiles,
// K 4096: 32 tokens × 8192 17.7 against 19.2 µs, × 14336 22.0 against 21.9; 48 × 8192 19.5
// against 19.9, × 14336 25.6 against 23.2; 64 × 4096 18.2 against 18.7, × 12288 26.9
// against 22.9.
bool few_tokens(int64_t T, int64_t N) { return T <= 32 || (T <= 64 && N <= 64 * 128); }

template <int R, int TB>
void launch_few(hipStream_t st, const GemmI8& a) {
  hipLaunchKernelGGL((gemm_i8_few_kernel<R, TB, false, 0, true>),
                     dim3((unsigned)cdiv(a.N, 16 * R)), dim3(512), 0, st, a, nullptr, 0, false);
}

template <int R>
void launch_few(hipStream_t st, const GemmI8& a) {
  if (a.T <= 16) launch_few<R, 1>(st, a);
  else if (a.T <= 32) launch_few<R, 2>(st, a);
  else if constexpr (R < 4) {  // (more channels are tiled)
    if (a.T <= 48) launch_few<R, 3>(st, a);
    else launch_few<R, 4>(st, a);
  }
}

template <int BM, int BN, int WM, int WN, int S>
void launch_tiles(hipStream_t st, const GemmI8& a) {
  const int64_t tm = cdiv(a.T, BM), tn = cdiv(a.N, BN);
  hipLaunchKernelGGL((gemm_i8_kernel<BM, BN, WM, WN, S>), dim3((unsigned)(tm * tn)),
                     dim3(64 * WM * WN * S), 0, st, a, (int)tm, (int)tn);
}

int gemm_i8(hipStream_t st, const GemmI8& a) {
  if (few_tokens(a.T, a.N)) {
    const int r = few_rows(a.N);
    if (r == 4) launch_few<4>(st, a);
    else if (r == 2) launch_few<2>(st, a);
    else launch_few<1>(st, a);
  } else {
    // The largest tile that still fills the chip.  MI355X, product alone: 256 against 128 at
    // 256 tiles of 256 (4096³) 64 against 86 µs; 128 against 64 at 256 tiles of 128
    // (1024 × 4096, K 4096) 28 against 34 µs, at 128 of them (512 × 4096, K 14336) 71
    // against 54 µs; 208 tiles of 64 (777 × 1000, K 2752) 10.4 µs with K shared by four
    // groups, 12.8 µs without (back to back over the same operands, as the others here).
    if (cdiv(a.T, 256) * cdiv(a.N, 256) >= 192) launch_tiles<256, 256, 2, 4, 1>(st, a);
    else if (cdiv(a.T, 128) * cdiv(a.N, 128) >= 224) launch_tiles<128, 128, 2, 2, 1>(st, a);
    else if (cdiv(a.T, 64) * cdiv(a.N, 64) > 512) launch_tiles<64, 64, 2, 2, 1>(st, a);
    else if (cdiv(a.T, 64) * cdiv(a.N, 64) > 256) launch_tiles<64, 64, 2, 2, 2>(st, a);
    else launch_tiles<64, 64, 2, 2, 4>(st, a);
  }
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}

// Tokens quantized and multiplied in one launch: one token, or two of up to 16384 columns
// (LDS holds the codes).  MI355X, over weights that no cache holds, fused against apart: one
// token, 4096 × 4096 9.4 against 10.8 µs, K 14336 19.1 against 25.7, 8192 channels of K 28672
// 53 against 62; two, 4096 × 4096 10.8 against 11.1, K 11008 21.0 against 23.1; four, 13.4
// against 11.2.
bool fused(int64_t T, int64_t K) { return T <= 2 && T * K <= 32768; }
template <int DT, bool SYM>
void launch_fused(hipStream_t st, const GemmI8& a, const void* x, int64_t ldx, bool vec) {
  const size_t lds = (size_t)(a.T * (cdiv(a.K, 256) * 256));
#define G2_FU(R)                                                                             \
  hipLaunchKernelGGL((gemm_i8_few_kernel<R, 1, true, DT, SYM>), dim3((unsigned)cdiv(a.N, 16 * R)), \
                     dim3(512), lds, st, a, x, ldx, vec)
  // (four: one token × 14336 channels 18.1 µs, two 17.0)
  if (few_rows(a.N) >= 2) G2_FU(2);
  else G2_FU(1);
#undef G2_FU
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
  // (a launch has 512 threads for 32 channels of few tokens, or for 256 × 256 outputs)
  G2PTQ_CHECK(a.T >= 0 && a.T < (1ll << 22) && a.K >= 1 && a.K <= kMaxK && a.N >= 0 &&
                  cdiv(a.N, 32) < kMaxGroups && cdiv(a.T, 256) * cdiv(a.N, 256) < kMaxGroups,
              "%s: %lld tokens × %lld columns × %lld channels are too many", who, (long long)a.T,
              (long long)a.K, (long long)a.N);
  if (a.T == 0 || a.N == 0) return G2PTQ_OK;
  G2PTQ_CHECK(a.W && a.sw && a.out && a.ldo >= a.N, "%s: null pointer or output stride", who);
  const int64_t K256 = cdiv(a.K, 256) * 256;
  G2PTQ_CHECK(a.ldw >= K256 && a.ldw % 16 == 0 && a.ldw < (1 << 20) && aligned16(a.W),
              "%s: weights need 16-byte aligned rows of at least %lld bytes", who,
              (long long)K256);
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
  G2PTQ_CHECK(ldc % 16 == 0 && ldc >= cdiv(K, 16) * 16 && ldc < (1 << 20) && aligned16(codes),
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
  if (!fused(T, K)) *bytes += (size_t)LinearWs(T, K).gemm;
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
  if (fused(T, K)) {
    const bool vec = aligned16(x) && ldx * (dtype == 2 ? 4 : 2) % 16 == 0;
    hipStream_t st = as_stream(stream);
    if (dtype == 0) { if (sym) launch_fused<0, true>(st, a, x, ldx, vec); else launch_fused<0, false>(st, a, x, ldx, vec); }
    else if (dtype == 1) { if (sym) launch_fused<1, true>(st, a, x, ldx, vec); else launch_fused<1, false>(st, a, x, ldx, vec); }
    else { if (sym) launch_fused<2, true>(st, a, x, ldx, vec); else launch_fused<2, false>(st, a, x, ldx, vec); }
    G2PTQ_LAUNCHED();
    return G2PTQ_OK;
  }
  size_t need;
  G2PTQ_TRY(g2ptq_int8_linear_workspace(T, N, K, &need));
  if (need && (!ws || ws_bytes < need)) {
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
