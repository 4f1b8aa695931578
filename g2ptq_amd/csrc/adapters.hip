// Low-rank adapters of many requests beside a shared projection.
//
//   out_t = base_t + s_a·U_a·(D_a·x_t),  a = index_t  (out_t = base_t where there is none)
//
// Two products on the matrix cores: h = D·x into fp32 workspace (K split over workgroups, the
// shares summed in order), then U·h.  Sums are fp32.  h enters the second product as two
// 16-bit numbers, its rounding and what that left out, so that it keeps 16 bits and more
// (bf16) or 21 and more below the row's largest (fp16, whose rows are scaled by a power of
// two to its range).
//
// Tokens are taken in windows of 64.  A window's adapters are found by comparing the index of
// every lane (no sort, no launch of its own); each is multiplied with its own tokens only.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace g2ptq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWindow = 64;  // tokens
constexpr int kRankGroup = 64;

struct AdapterArgs {
  const uint16_t* x;
  int64_t ldx;
  const int32_t* index;
  int64_t T, K, N, n;
  const uint16_t *down, *up;  // n × R × Kp and n × Np × R, zero where padded
  int64_t R, Kp, Np;
  const int32_t* rank;
  const float* scale;
  float* h;                   // parts × T × R
  int parts, slots;
  const uint16_t* base;       // nullable
  int64_t ldb;
  uint16_t* out;
  int64_t ldo;
  int* flags;
  bool vx, vo;                // rows of x, of base and out are 16-byte aligned
  int64_t window;             // the launch's first
};

template <bool F16>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ float widen(uint16_t v) {
  return F16 ? (float)__builtin_bit_cast(_Float16, v) : __uint_as_float((uint32_t)v << 16);
}
template <bool F16>
__device__ __forceinline__ uint16_t narrow(float v) {
  return F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}

// Eight values from p, those from n on zero.
__device__ __forceinline__ u32x4 piece(const uint16_t* p, bool vec, int64_t n) {
  if (vec && n >= 8) return *reinterpret_cast<const u32x4*>(p);
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = (2 * i < n ? p[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] << 16 : 0u);
  return v;
}

// f(adapter, list of its tokens in the window, their number) for every adapter whose first
// token of the window is at a lane that this slot takes.  The list is the wave's own.
template <typename F>
__device__ __forceinline__ void each_adapter(const AdapterArgs& a, int64_t t0, int slot,
                                             int32_t idx, uint8_t* list, F f) {
  const int lane = threadIdx.x & 63;
  for (int first = slot; first < kWindow; first += a.slots) {
    const int32_t which = __builtin_amdgcn_readlane(idx, first);
    if (which < 0) continue;
    const uint64_t same = __ballot(idx == which);
    if (__builtin_ctzll(same) != first) continue;
    __builtin_amdgcn_wave_barrier();
    if (idx == which) list[__popcll(same & ((1ull << lane) - 1))] = (uint8_t)lane;
    __builtin_amdgcn_wave_barrier();
    f(which, __popcll(same));
  }
}

__device__ __forceinline__ int32_t index_of_lane(const AdapterArgs& a, int64_t t0) {
  const int64_t t = t0 + (threadIdx.x & 63);
  int32_t idx = t < a.T ? a.index[t] : -1;
  if (idx >= a.n) {
    if (threadIdx.x < 64 && blockIdx.y == 0) atomicOr(a.flags, G2PTQ_FLAG_BAD_INDEX);
    idx = -1;
  }
  return idx;
}

// h of 16·TB tokens for 16·RB ranks from r0 on: ranks × tokens, 64 columns of K a step (lane
// (n, g) holds 16 of row n from 16·g on).  The workgroup's waves and the launch's parts take
// turns at the steps.
template <bool F16, int RB, int TB>
__device__ __forceinline__ void shrink(const AdapterArgs& a, int64_t t0, int which, int64_t r0,
                                       const uint8_t* list, int count, f32x4 (*sums)[16][64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const uint16_t* xrow[TB];
  const uint16_t* drow[RB];
#pragma unroll
  for (int b = 0; b < TB; ++b)
    xrow[b] = a.x + (t0 + list[min(16 * b + n, count - 1)]) * a.ldx;
#pragma unroll
  for (int r = 0; r < RB; ++r) drow[r] = a.down + ((int64_t)which * a.R + r0 + 16 * r + n) * a.Kp;
  f32x4 acc[RB][TB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[r][b] = f32x4{0, 0, 0, 0};
  for (int64_t k = (int64_t)(blockIdx.y * 4 + wave) * 64 + g * 16; k - g * 16 < a.Kp;
       k += a.parts * 256) {
    u32x4 d[RB][2], x[TB][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < RB; ++r) d[r][i] = *reinterpret_cast<const u32x4*>(drow[r] + k + 8 * i);
#pragma unroll
      for (int b = 0; b < TB; ++b) x[b][i] = piece(xrow[b] + k + 8 * i, a.vx, a.K - k - 8 * i);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[r][b] = mfma<F16>(d[r][i], x[b][i], acc[r][b]);
  }
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b) sums[wave][r * TB + b][lane] = acc[r][b];
  __syncthreads();
  for (int i = threadIdx.x; i < RB * TB * 64; i += 256) {
    const int at = i >> 6, l = i & 63, t = at % TB * 16 + (l & 15);
    if (t < count) {
      f32x4 s = sums[0][at][l];
#pragma unroll
      for (int w = 1; w < 4; ++w) s += sums[w][at][l];
      // lane (token, ranks 4g .. 4g + 3)
      *reinterpret_cast<f32x4*>(a.h + ((int64_t)blockIdx.y * a.T + t0 + list[t]) * a.R + r0 +
                                at / TB * 16 + (l >> 4) * 4) = s;
    }
  }
  __syncthreads();
}

template <bool F16>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(AdapterArgs a) {
  __shared__ f32x4 sums[4][16][64];
  __shared__ uint8_t lists[4][kWindow];
  const int64_t t0 = (a.window + blockIdx.x / a.slots) * kWindow;
  uint8_t* list = lists[threadIdx.x >> 6];
  each_adapter(a, t0, blockIdx.x % a.slots, index_of_lane(a, t0), list, [&](int which, int count) {
    const int rank = a.rank[which];
    for (int64_t r0 = 0; r0 < rank; r0 += kRankGroup) {
      const int blocks = (int)min<int64_t>(kRankGroup, rank - r0 + 15) / 16;
      if (count <= 16) {
        if (blocks <= 1) shrink<F16, 1, 1>(a, t0, which, r0, list, count, sums);
        else if (blocks <= 2) shrink<F16, 2, 1>(a, t0, which, r0, list, count, sums);
        else if (blocks <= 3) shrink<F16, 3, 1>(a, t0, which, r0, list, count, sums);
        else shrink<F16, 4, 1>(a, t0, which, r0, list, count, sums);
      } else {
        if (blocks <= 1) shrink<F16, 1, 4>(a, t0, which, r0, list, count, sums);
        else if (blocks <= 2) shrink<F16, 2, 4>(a, t0, which, r0, list, count, sums);
        else if (blocks <= 3) shrink<F16, 3, 4>(a, t0, which, r0, list, count, sums);
        else shrink<F16, 4, 4>(a, t0, which, r0, list, count, sums);
      }
    }
  });
}

// Eight ranks of a token's h from r on, scaled; zero behind the adapter's own (`left` of them:
// a padded row's zeros times an infinity are no zeros).
__device__ __forceinline__ void load_h(const AdapterArgs& a, int64_t t, int64_t r, int64_t left,
                                       float scale, float (&v)[8]) {
  const float* p = a.h + t * a.R + r;
  f32x4 s[2] = {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
  for (int i = 1; i < a.parts; ++i) {
    p += a.T * a.R;
    s[0] += *reinterpret_cast<const f32x4*>(p);
    s[1] += *reinterpret_cast<const f32x4*>(p + 4);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < left ? s[i >> 2][i & 3] * scale : 0.f;
}

// Sixteen channels from c on of a token's row: out = base + add.
template <bool F16>
__device__ __forceinline__ void add_row(const AdapterArgs& a, int64_t t, int64_t c,
                                        const float (&add)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t n = a.N - c - 8 * i;
    if (n <= 0) return;
    u32x4 v = {0, 0, 0, 0};
    if (a.base) v = piece(a.base + t * a.ldb + c + 8 * i, a.vo, n);
    uint16_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t b = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
      h[j] = narrow<F16>(a.base ? widen<F16>(b) + add[8 * i + j] : add[8 * i + j]);
    }
    uint16_t* o = a.out + t * a.ldo + c + 8 * i;
    if (a.vo && n >= 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
      *reinterpret_cast<u32x4*>(o) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) o[j] = h[j];
    }
  }
}

// 16·TB tokens × the wave's 64 channels from c0 on: channels × tokens; row m of block j is
// channel 16·(m / 4) + 4·j + m % 4, so that a lane ends with 16 channels in a row.  A step
// of 32 is 16 ranks twice: with h rounded, and with what that left out.
template <bool F16, int TB>
__device__ __forceinline__ void expand(const AdapterArgs& a, int64_t t0, int which, int64_t c0,
                                       const uint8_t* list, int count, int from) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const float scale = a.scale[which];
  const int64_t rank = a.rank[which];
  const uint16_t* urow = a.up + ((int64_t)which * a.Np + c0 + (n >> 2) * 16 + (n & 3)) * a.R;
  const bool low = g >= 2;
  const int part = (g & 1) * 8;
  int64_t token[TB];
  float fit[TB];       // the row's power of two
  bool infinite[TB];
  f32x4 acc[TB][4];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    token[b] = t0 + list[min(from + 16 * b + n, count - 1)];
    fit[b] = 1.f, infinite[b] = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[b][j] = f32x4{0, 0, 0, 0};
    if constexpr (F16) {
      uint32_t top = 0;
      for (int64_t r = part; r - part < rank; r += 16) {
        float v[8];
        load_h(a, token[b], r, rank - r, scale, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));  // (lanes n, n + 16: all ranks)
      infinite[b] = top >= 0x7f800000u;
      if (!infinite[b] && top) fit[b] = __uint_as_float((uint32_t)min(254, max(1, 127 + 14 + 127 - (int)(top >> 23))) << 23);
    }
  }
  for (int64_t r = 0; r < rank; r += 16) {
    u32x4 u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      u[j] = *reinterpret_cast<const u32x4*>(urow + 4 * j * a.R + r + part);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      float v[8];
      load_h(a, token[b], r + part, rank - r - part, scale, v);
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f = v[i] * fit[b];
        // (beside an infinity or a NaN finite terms do not count, and fp16 has no room for them)
        if (F16 && infinite[b] && fabsf(f) < __builtin_inff()) f = 0.f;
        uint16_t q = narrow<F16>(f);
        if (low) {
          const float left = f - widen<F16>(q);
          q = narrow<F16>(fabsf(left) < __builtin_inff() ? left : 0.f);
        }
        if (i & 1) w[i >> 1] |= (uint32_t)q << 16;
        else w[i >> 1] = q;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[b][j] = mfma<F16>(u[j], w, acc[b][j]);
    }
  }
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    if (from + 16 * b + n >= count) continue;
    const float back = F16 ? __fdiv_rn(1.f, fit[b]) : 1.f;
    float add[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) add[i] = acc[b][i >> 2][i & 3] * back;
    add_row<F16>(a, token[b], c0 + g * 16, add);
  }
}

template <bool F16>
__global__ __launch_bounds__(256) void adapter_expand_kernel(AdapterArgs a) {
  __shared__ uint8_t lists[4][kWindow];
  const int64_t t0 = (a.window + blockIdx.x / a.slots) * kWindow;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, slot = blockIdx.x % a.slots;
  const int64_t c0 = (int64_t)blockIdx.y * 256 + wave * 64;
  if (c0 >= a.N) return;
  const int32_t idx = index_of_lane(a, t0);
  uint8_t* list = lists[wave];
  each_adapter(a, t0, slot, idx, list, [&](int which, int count) {
    if (count <= 16) expand<F16, 1>(a, t0, which, c0, list, count, 0);
    else expand<F16, 4>(a, t0, which, c0, list, count, 0);
  });
  if (a.out != a.base) {  // rows without an adapter
    const float none[16] = {};
    for (int t = slot; t < kWindow && t0 + t < a.T; t += a.slots)
      if (__builtin_amdgcn_readlane(idx, t) < 0 && lane < 4) add_row<F16>(a, t0 + t, c0 + lane * 16, none);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workgroups of a window: one adapter each where there are few windows (every token may have
// its own), fewer where windows fill the chip.
int slots_of(int64_t T, int64_t n) {
  const int64_t windows = cdiv(T, kWindow);
  int64_t s = std::min<int64_t>(std::min<int64_t>(kWindow, n), T);
  while (s > 2 && windows * s > 1024) s /= 2;
  return (int)std::max<int64_t>(1, s);
}

// Shares of K: enough workgroups for the chip where there are few.
int parts_of(int64_t T, int64_t K, int64_t n) {
  const int64_t groups = cdiv(T, kWindow) * slots_of(T, n);
  int p = 1;
  while (p < 8 && groups * p < 512 && K >= (int64_t)p * 2 * 512) p *= 2;
  return p;
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_adapters_workspace(int64_t T, int64_t K, int64_t n, int64_t R,
                                        size_t* bytes) {
  G2PTQ_CHECK(bytes && T >= 0 && T < (1ll << 31) && K >= 1 && n >= 1 && R >= 16,
              "adapters_workspace: bad sizes");
  *bytes = (size_t)parts_of(T, K, n) * T * R * 4;
  return G2PTQ_OK;
}

extern "C" int g2ptq_adapters(void* stream, const g2ptq_adapter_set* set, const void* x,
                              int64_t ldx, const int32_t* index, int64_t T, const void* base,
                              int64_t ldb, void* out, int64_t ldo, void* ws, size_t ws_bytes) {
  G2PTQ_CHECK(set, "adapters: null set");
  G2PTQ_CHECK(set->dtype == 0 || set->dtype == 1, "adapters: dtype code %d (bf16 or fp16)",
              set->dtype);
  G2PTQ_CHECK(set->n >= 1 && set->n < (1ll << 31) && set->K >= 1 && set->K <= (1 << 20) &&
                  set->N >= 1 && set->N <= (1 << 20) && set->R >= 16 && set->R <= 512 &&
                  set->R % 16 == 0,
              "adapters: %lld adapters of %lld ranks, %lld columns, %lld channels",
              (long long)set->n, (long long)set->R, (long long)set->K, (long long)set->N);
  G2PTQ_CHECK(T >= 0 && T < (1ll << 31), "adapters: %lld tokens", (long long)T);
  if (T == 0) return G2PTQ_OK;
  G2PTQ_CHECK(set->down && set->up && set->rank && set->scale && set->flags && x && index && out,
              "adapters: null pointer");
  G2PTQ_CHECK(aligned16(set->down) && aligned16(set->up) && aligned16(ws),
              "adapters: weights or workspace not 16-byte aligned");
  size_t need;
  G2PTQ_TRY(g2ptq_adapters_workspace(T, set->K, set->n, set->R, &need));
  if (!ws || ws_bytes < need) {
    set_error("adapters: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return G2PTQ_ERR_WORKSPACE;
  }
  AdapterArgs a{};
  a.x = static_cast<const uint16_t*>(x), a.ldx = ldx, a.index = index;
  a.T = T, a.K = set->K, a.N = set->N, a.n = set->n;
  a.down = static_cast<const uint16_t*>(set->down), a.up = static_cast<const uint16_t*>(set->up);
  a.R = set->R, a.Kp = cdiv(set->K, 64) * 64, a.Np = cdiv(set->N, 64) * 64;
  a.rank = set->rank, a.scale = set->scale;
  a.h = static_cast<float*>(ws);
  a.parts = parts_of(T, set->K, set->n), a.slots = slots_of(T, set->n);
  a.base = static_cast<const uint16_t*>(base), a.ldb = ldb;
  a.out = static_cast<uint16_t*>(out), a.ldo = ldo;
  a.flags = set->flags;
  a.vx = aligned16(x) && ldx % 8 == 0;
  a.vo = aligned16(base) && aligned16(out) && ldb % 8 == 0 && ldo % 8 == 0;
  hipStream_t st = as_stream(stream);
  const int64_t windows = cdiv(T, kWindow), most = (1 << 20) / a.slots;
  for (a.window = 0; a.window < windows; a.window += most) {
    const unsigned groups = (unsigned)(std::min(windows - a.window, most) * a.slots);
    const dim3 shrink(groups, a.parts), expand(groups, (unsigned)cdiv(set->N, 256));
    if (set->dtype == 0) {
      hipLaunchKernelGGL((adapter_shrink_kernel<false>), shrink, dim3(256), 0, st, a);
      hipLaunchKernelGGL((adapter_expand_kernel<false>), expand, dim3(256), 0, st, a);
    } else {
      hipLaunchKernelGGL((adapter_shrink_kernel<true>), shrink, dim3(256), 0, st, a);
      hipLaunchKernelGGL((adapter_expand_kernel<true>), expand, dim3(256), 0, st, a);
    }
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}
