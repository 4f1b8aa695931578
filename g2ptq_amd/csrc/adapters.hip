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
//
// Bound by memory where tokens are many: MI355X, under the profiler, 5100 tokens of eight
// requests with four adapters of ranks 32 and 64, 4096 to 14336: D·x 16–18 µs (its 42 MB of
// tokens at a copy's rate 8), U·h 77–83 (292 MB of rows in and out: 57; a launch that only copies
// them through the same mapping takes some 70).  Every share of the channels reads h's shares of K
// again, 42 MB there.  By latency where tokens are few: 48 with 32 adapters of rank 16, 4096 × 4096,
// 3.7–4.1 and 6.3–6.6 µs: index, adapter, operands and sums follow each other through memory.  By
// the adapters' weights where tokens take turns at many of them: every window reads its own again
// (2048 tokens of 40 adapters of rank 16, 4096 × 4096: 71 µs for 12 of bytes).
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

struct AdapterArgs {
  const uint16_t* x;
  int64_t ldx;
  const int32_t* index;
  int64_t T, K, N, n;
  const uint16_t *down, *up;  // n × R × Kp and n × Np × R in the products' order
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
  bool infinite;              // some weights of up are infinite
  bool odd;                   // rows of x may start between 32-bit words
  bool aligned;               // rows of base and out are 16-byte aligned
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

// Eight values from p on, at any address: sixteen bytes are one instruction wherever they lie
// (MI355X, 2048 tokens of rank 64, 4097 × 4097: 37 µs, 39 with a load and a store a value).
__device__ __forceinline__ u32x4 piece(const uint16_t* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// Eight values of a row of `size` from c ≥ 0 on, those behind its end zero: the last eight moved
// down, so that no value waits for another's branch.
__device__ __forceinline__ u32x4 piece(const uint16_t* row, int64_t c, int64_t size) {
  if (c + 8 <= size) return piece(row + c);
  if (size >= 8) {
    const int64_t past = c + 8 - size;
    const u32x4 v = piece(row + c - past);
    const uint64_t low = v[0] | (uint64_t)v[1] << 32, high = v[2] | (uint64_t)v[3] << 32;
    const int s = 16 * (int)(past & 3);
    const uint64_t a = past >= 8 ? 0 : past >= 4 ? high : low, b = past >= 4 ? 0 : high;
    const uint64_t l = a >> s | b << 1 << (63 - s), h = b >> s;
    return u32x4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
  }
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = (c + 2 * i < size ? row[c + 2 * i] : 0u) |
           (c + 2 * i + 1 < size ? (uint32_t)row[c + 2 * i + 1] << 16 : 0u);
  return v;
}

// f(adapter, number of its tokens) for every adapter that this slot takes, with `list` (the wave's
// own) their lanes.  none: tokens without an adapter too, as −1.  A slot takes every slots-th run
// of equal neighbours, and of these the ones that open with the window's first token of theirs.
// MI355X, 421 tokens of 20 adapters of rank 16, 3500 × 2651: 15 µs, 36 where a slot took every
// slots-th token (prompts of as many tokens as there are slots all met in one).
template <typename F>
__device__ __forceinline__ void each_adapter(const AdapterArgs& a, int slot, int32_t idx,
                                             bool none, uint8_t* list, F f) {
  const int lane = threadIdx.x & 63;
  // (the lane below's; −3 below the first)
  const int32_t before = __builtin_amdgcn_update_dpp(-3, idx, 0x138, 0xf, 0xf, false);
  const bool head = idx >= (none ? -1 : 0) && before != idx;
  const int runs = __popcll(__ballot(head) & ((1ull << lane) - 1));
  uint64_t lanes = __ballot(head && runs % a.slots == slot);
  while (lanes) {
    const int first = __builtin_ctzll(lanes);
    const int32_t which = __builtin_amdgcn_readlane(idx, first);
    const uint64_t same = __ballot(idx == which);
    lanes &= ~same;
    if (__builtin_ctzll(same) != first) continue;  // another slot's
    __builtin_amdgcn_wave_barrier();
    if (idx == which) list[__popcll(same & ((1ull << lane) - 1))] = (uint8_t)lane;
    __builtin_amdgcn_wave_barrier();
    f(which, __popcll(same));
  }
}

// The adapter of the lane's token: −1 none, −2 no token.
__device__ __forceinline__ int32_t index_of_lane(const AdapterArgs& a, int64_t t0) {
  const int64_t t = t0 + (threadIdx.x & 63);
  if (t >= a.T) return -2;
  const int32_t idx = a.index[t];
  if (idx >= a.n && threadIdx.x < 64 && blockIdx.y == 0) atomicOr(a.flags, G2PTQ_FLAG_BAD_INDEX);
  return idx >= a.n ? -1 : max(idx, -1);
}

// h of 16·TB tokens for up to 16·RB ranks from r0 on: ranks × tokens, 64 columns of K a step
// (lane (n, g) holds 16 of row n from 16·g on).  The workgroup's waves and the launch's parts
// take turns at steps, whatever TB is: a token's sums are added in an order that its neighbours
// have no part in.  U steps' loads are under way together.
// ODD: rows may start between two 32-bit words.  There the memory takes a load of sixteen bytes
// apart, so the words are loaded that hold the values (two bytes before the first and behind the
// last share theirs and are shifted out).  MI355X, both launches, 777 tokens of rank 20, 2047 to 2751:
// 20.4 µs, 23.2 without; 2048 tokens of rank 64, 4097 × 4097: 36.7 and 43.5.
template <bool F16, int RB, int TB, bool ODD>
__device__ __forceinline__ void shrink(const AdapterArgs& a, int64_t t0, int which, int64_t r0,
                                       int blocks, const uint8_t* list, int count,
                                       f32x4 (*sums)[RB * 4][64]) {
  constexpr int U = TB == 1 ? 2 : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const uint16_t* xrow[TB];
  const uint16_t* drow[RB];
  uint32_t odd[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    xrow[b] = a.x + (t0 + list[min(16 * b + n, count - 1)]) * a.ldx + g * 16;
    odd[b] = ODD ? (uint32_t)(reinterpret_cast<uintptr_t>(xrow[b]) >> 1) & 1 : 0;
  }
#pragma unroll
  for (int r = 0; r < RB; ++r)  // (blocks that the adapter lacks: the first again, not stored)
    drow[r] = a.down + ((int64_t)which * a.R + r0 + (r < blocks ? 16 * r : 0)) * a.Kp + lane * 8;
  f32x4 acc[RB][TB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[r][b] = f32x4{0, 0, 0, 0};
  struct Step {
    u32x4 d[RB][2], x[TB][2];
    uint32_t end[TB];
  };
  auto products = [&](const Step& s) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[r][b] = mfma<F16>(s.d[r][i], s.x[b][i], acc[r][b]);
  };
  auto fetch = [&](Step& s, int64_t k) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
        s.d[r][i] = *reinterpret_cast<const u32x4*>(drow[r] + k * 16 + 512 * i);
#pragma unroll
      for (int b = 0; b < TB; ++b) s.x[b][i] = piece(xrow[b] + k + 8 * i - odd[b]);
    }
    if (ODD)  // (the last value's word; rows on words have no use for a ninth)
#pragma unroll
      for (int b = 0; b < TB; ++b)
        s.end[b] = *reinterpret_cast<const uint32_t*>(xrow[b] + k + 14 + odd[b]);
  };
  auto shift = [&](Step& s) {
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t next = i < 7 ? s.x[b][(i + 1) >> 2][(i + 1) & 3] : s.end[b];
        s.x[b][i >> 2][i & 3] =
            __builtin_amdgcn_alignbit(next, s.x[b][i >> 2][i & 3], 16 * odd[b]);
      }
  };
  const int each = a.parts * 4;
  int step = blockIdx.y * 4 + wave;
  const int whole = (int)(a.K / 64);
  for (; step + (U - 1) * each < whole; step += U * each) {
    Step s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(s[u], (int64_t)(step + u * each) * 64);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ODD) shift(s[u]);
      products(s[u]);
    }
  }
  if (U > 1 && step < whole) {
    Step s;
    fetch(s, (int64_t)step * 64);
    if (ODD) shift(s);
    products(s);
    step += each;
  }
  // the last columns
  for (; step * 64 < a.Kp; step += each) {
    const int64_t k = (int64_t)step * 64;
    Step s;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
        s.d[r][i] = *reinterpret_cast<const u32x4*>(drow[r] + k * 16 + 512 * i);
#pragma unroll
      for (int b = 0; b < TB; ++b)
        s.x[b][i] = piece(xrow[b] - g * 16, k + g * 16 + 8 * i, a.K);
    }
    products(s);
  }
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int b = 0; b < TB; ++b) sums[wave][r * TB + b][lane] = acc[r][b];
  __syncthreads();
  for (int i = threadIdx.x; i < blocks * TB * 64; i += 256) {
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

template <bool F16, int RB, bool ODD>
__global__ __launch_bounds__(256, 2) void adapter_shrink_kernel(AdapterArgs a) {
  __shared__ f32x4 sums[4][RB * 4][64];
  __shared__ uint8_t lists[4][kWindow];
  const uint32_t windows = gridDim.x / (uint32_t)a.slots, slot = blockIdx.x / windows;
  const int64_t t0 = (a.window + blockIdx.x - slot * windows) * kWindow;
  uint8_t* list = lists[threadIdx.x >> 6];
  each_adapter(a, slot, index_of_lane(a, t0), false, list, [&](int which, int count) {
    const int blocks = (a.rank[which] + 15) / 16;
    for (int r = 0; r < blocks; r += RB) {
      const int here = min(RB, blocks - r);
      if (count <= 16) shrink<F16, RB, 1, ODD>(a, t0, which, r * 16, here, list, count, sums);
      else shrink<F16, RB, 4, ODD>(a, t0, which, r * 16, here, list, count, sums);
    }
  });
}

// The shares of eight ranks' sums, all loads under way together.
template <int P>
__device__ __forceinline__ void sum_parts(const float* p, int64_t next, f32x4 (&s)[2]) {
  f32x4 v[P][2];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    v[i][0] = *reinterpret_cast<const f32x4*>(p + i * next);
    v[i][1] = *reinterpret_cast<const f32x4*>(p + i * next + 4);
  }
  s[0] = v[0][0], s[1] = v[0][1];
#pragma unroll
  for (int i = 1; i < P; ++i) s[0] += v[i][0], s[1] += v[i][1];
}

// Eight ranks of a token's h from r on, scaled; zero behind the adapter's own (`left` of them:
// a padded row's zeros times an infinity are no zeros).
__device__ __forceinline__ void load_h(const AdapterArgs& a, int64_t t, int64_t r, int64_t left,
                                       float scale, float (&v)[8]) {
  const float* p = a.h + t * a.R + r;
  const int64_t next = a.T * a.R;
  f32x4 s[2];
  if (a.parts == 8) sum_parts<8>(p, next, s);
  else if (a.parts == 4) sum_parts<4>(p, next, s);
  else if (a.parts == 2) sum_parts<2>(p, next, s);
  else sum_parts<1>(p, next, s);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < left ? s[i >> 2][i & 3] * scale : 0.f;
}

// Eight channels from c on of a token's row: out = base + add.  IO: kPieces where rows are whole
// pieces of eight, kStream where they are aligned too and the caches are to keep other data
// besides, kRagged otherwise.
enum : int { kRagged, kPieces, kStream };
template <int IO>
__device__ __forceinline__ u32x4 base_piece(const AdapterArgs& a, int64_t t, int64_t c) {
  if (!a.base) return u32x4{0, 0, 0, 0};
  // (channels behind the last: the first again, not stored)
  if (IO == kRagged) return piece(a.base + t * a.ldb, c, a.N);
  const uint16_t* p = a.base + t * a.ldb + (c < a.N ? c : 0);
  if (IO == kStream) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return piece(p);
}
template <bool F16, int IO>
__device__ __forceinline__ void store_piece(const AdapterArgs& a, int64_t t, int64_t c, u32x4 base,
                                            f32x4 lo, f32x4 hi) {
  const int64_t n = a.N - c;
  uint16_t* o = a.out + t * a.ldo + c;
  uint16_t h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float add = j < 4 ? lo[j & 3] : hi[j & 3];
    h[j] = narrow<F16>(widen<F16>((uint16_t)(base[j >> 1] >> (16 * (j & 1)))) + add);
  }
  if (n <= 0) return;
  if (IO != kRagged || n >= 8) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
    if (IO == kStream) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(o));
    else __builtin_memcpy(o, &v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) o[j] = h[j];
  }
}

// An adapter's tokens' h into LDS as it enters the product: per token and 16 ranks four pieces
// of 16 bytes, both halves of the ranks rounded, then what the rounding left out.  Two, four or
// eight lanes take a token.  back: what a token's products are multiplied with, fp16's rows being brought
// to the top of its range by a power of two.  INF: some weights are infinite, and take the sign of
// finite terms beside an infinity.
template <bool F16, bool INF>
__device__ __forceinline__ void stage_h(const AdapterArgs& a, int64_t t0, int which,
                                        const uint8_t* list, int count, u32x4* hL, int pitch,
                                        float* back) {
  const float scale = a.scale[which];
  const int rank = a.rank[which], pieces = (rank + 15) / 16 * 2;
  constexpr float most = F16 ? 65504.f : 0x1.fep127f;
  const int shift = pieces <= 2 ? 1 : pieces <= 4 ? 2 : 3, lanes = 1 << shift;
  for (int i = threadIdx.x; (i & ~255) < count << shift; i += 256) {
    const int t = i >> shift, l = i & (lanes - 1);
    const int64_t token = t0 + list[min(t, count - 1)];
    float fit = 1.f;
    bool infinite = false;
    float v[8];
    if (l < pieces) load_h(a, token, l * 8, rank - l * 8, scale, v);
    if constexpr (F16) {
      uint32_t top = 0;
      for (int p = l; p < pieces; p += lanes) {
        if (p != l) load_h(a, token, p * 8, rank - p * 8, scale, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
      }
      for (int o = 1; o < lanes; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o));
      infinite = top >= 0x7f800000u;
      if (!infinite && top)
        fit = __uint_as_float((uint32_t)min(254, max(1, 268 - (int)(top >> 23))) << 23);
      if (l == 0 && t < count) back[t] = __fdiv_rn(1.f, fit);
    }
    for (int p = l; p < pieces; p += lanes) {
      // (ranks from 64 on, and then all of fp16's, are read again)
      if (p != l || (F16 && pieces > lanes)) load_h(a, token, p * 8, rank - p * 8, scale, v);
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float f = v[j] * fit;
        // (beside an infinity or a NaN finite terms do not count, and fp16 has no room for them)
        if (F16 && infinite && fabsf(f) < __builtin_inff())
          f = INF && f != 0.f ? copysignf(1.f, f) : 0.f;
        // (what is above the type's largest number goes into what is left out, infinities and NaN
        // too; infinite weights meet the rounding alone, which has to keep those)
        const bool all = INF && !(fabsf(f) < __builtin_inff());
        const uint16_t q = narrow<F16>(all ? f : __builtin_amdgcn_fmed3f(f, -most, most));
        const uint16_t u = narrow<F16>(all ? 0.f : f - widen<F16>(q));
        if (j & 1) hi[j >> 1] |= (uint32_t)q << 16, lo[j >> 1] |= (uint32_t)u << 16;
        else hi[j >> 1] = q, lo[j >> 1] = u;
      }
      if (t < count) {
        u32x4* o = hL + t * pitch + (p >> 1) * 4 + (p & 1);
        o[0] = hi, o[2] = lo;
      }
    }
  }
}

// Two weights as what h's rounding left out takes them: zero for infinities and NaN, which h's
// rounding has taken (times a remainder of zero or of the other sign they would make a NaN of it).
template <bool F16>
__device__ __forceinline__ uint32_t finite16(uint32_t w) {
  constexpr uint32_t top = F16 ? 0x7c00 : 0x7f80;
  return ((w & top) == top ? 0 : w & 0xffff) | ((w >> 16 & top) == top ? 0 : w & 0xffff0000);
}

// 16-byte pieces of a token's 64 sums in LDS, one of them against bank conflicts.
constexpr int kTurn = 17;

// 16·TB tokens × 64 channels at a time, channels × tokens.  A step of 32 is 16 ranks twice:
// with h rounded, and with what that left out.  The sums are turned in LDS so that eight lanes
// read and write 128 consecutive bytes of a token's row.  A wave walks its channels, and for
// each 64 the window's tokens; what comes next is loaded before what was computed is stored.
// RB: blocks of 16 ranks whose weights are held together.  INF: some weights are infinite.
template <bool F16, int IO, int RB, int TB, bool INF>
__device__ __forceinline__ void expand(const AdapterArgs& a, int64_t t0, int which,
                                       const uint8_t* list, int count, int chunk, int chunks,
                                       u32x4* hL, int pitch, float* back, f32x4* turn) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, row = lane >> 3, col = lane & 7;
  const int blocks = (a.rank[which] + 15) / 16;
  // (the weights as they enter the product: per 64 channels and 16 ranks four pieces of 16
  // channels × 2 halves of the ranks)
  const uint16_t* up = a.up + (int64_t)which * a.Np * a.R + (lane & 31) * 8;
  u32x4 w[RB][4], base[TB][2];
  auto weights = [&](int chunk, int r0) {
    const uint16_t* u = up + ((int64_t)chunk * (a.R / 16) + r0) * 1024;
#pragma unroll
    for (int r = 0; r < RB; ++r)
      if (r0 + r < blocks)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[r][j] = *reinterpret_cast<const u32x4*>(u + (r * 4 + j) * 256);
    if (INF && lane >= 32)  // (these lanes' weights are for what h's rounding left out)
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r0 + r < blocks)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[r][j][i] = finite16<F16>(w[r][j][i]);
  };
  auto token = [&](int t) { return t0 + list[min(t, count - 1)]; };
  auto bases = [&](int chunk, int from) {
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        base[b][i] = base_piece<IO>(a, token(from + 16 * b + 8 * i + row),
                                     (int64_t)chunk * 64 + col * 8);
  };
  int from = 0;
  stage_h<F16, INF>(a, t0, which, list, count, hL, pitch, back);
  __syncthreads();
  if (chunk < chunks) weights(chunk, 0), bases(chunk, 0);
  while (chunk < chunks) {
    f32x4 acc[TB][4];
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[b][j] = f32x4{0, 0, 0, 0};
    for (int r0 = 0; r0 < blocks; r0 += RB) {
      if (blocks > RB) weights(chunk, r0);
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r0 + r < blocks)
#pragma unroll
          for (int b = 0; b < TB; ++b) {
            const u32x4 v = hL[min(from + 16 * b + n, count - 1) * pitch + (r0 + r) * 4 + g];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[b][j] = mfma<F16>(w[r][j], v, acc[b][j]);
          }
    }
    u32x4 old[TB][2];
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) old[b][i] = base[b][i];
    const int64_t c = (int64_t)chunk * 64 + col * 8;
    const int those = from;
    from += 16 * TB;
    if (from >= count) {
      from = 0, chunk += 4;
      if (chunk < chunks && blocks <= RB) weights(chunk, 0);
    }
    if (chunk < chunks) bases(chunk, from);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      if (those + 16 * b >= count) break;
      const float f = F16 ? back[min(those + 16 * b + n, count - 1)] : 1.f;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 4; ++j)  // lane (token n, channels 16j + 4g .. + 3)
        turn[n * kTurn + j * 4 + g] = F16 ? acc[b][j] * f : acc[b][j];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = those + 16 * b + 8 * i + row;
        const f32x4* p = turn + (8 * i + row) * kTurn + col * 2;
        if (t < count) store_piece<F16, IO>(a, t0 + list[t], c, old[b][i], p[0], p[1]);
      }
    }
  }
  __syncthreads();
}

// A window's channels are shared by `shares` workgroups, each walking its own range.  First come
// the first slots: they have the work where a window's tokens share an adapter.
template <bool F16, int IO, int RB, bool INF>
__global__ __launch_bounds__(256, 3) void adapter_expand_kernel(AdapterArgs a, int pitch,
                                                                int shares) {
  extern __shared__ u32x4 hL[];
  __shared__ uint8_t lists[4][kWindow];
  __shared__ float back[kWindow];
  __shared__ f32x4 turns[4][16 * kTurn];
  const uint32_t groups = gridDim.x / (uint32_t)shares;
  const uint32_t group = blockIdx.x / (uint32_t)shares, share = blockIdx.x - group * shares;
  const uint32_t windows = groups / (uint32_t)a.slots, slot = group / windows;
  const uint32_t window = group - slot * windows;
  const int64_t t0 = (a.window + window) * kWindow;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int all = (int)(a.Np / 64), each = (all + 4 * shares - 1) / (4 * shares) * 4;
  const int first = share * each + wave, last = min((int)(share + 1) * each, all);
  uint8_t* list = lists[wave];
  each_adapter(a, slot, index_of_lane(a, t0), a.out != a.base, list, [&](int which, int count) {
    if (which < 0) {  // rows without an adapter
      // (−0 is the number that changes nothing: a base of −0 stays, and no base is +0)
      const f32x4 none = {-0.f, -0.f, -0.f, -0.f};
      const int row = lane >> 3;
      for (int64_t c = (int64_t)first * 64 + (lane & 7) * 8; c < min<int64_t>(a.N, last * 64);
           c += 256) {
        u32x4 v[kWindow / 8];  // all loads under way together
#pragma unroll
        for (int i = 0; i < kWindow / 8; ++i)
          if (8 * i < count) v[i] = base_piece<IO>(a, t0 + list[min(8 * i + row, count - 1)], c);
#pragma unroll
        for (int i = 0; i < kWindow / 8; ++i)
          if (8 * i + row < count)
            store_piece<F16, IO>(a, t0 + list[8 * i + row], c, v[i], none, none);
      }
      return;
    }
    f32x4* turn = turns[wave];
    if (count <= 16)
      expand<F16, IO, RB, 1, INF>(a, t0, which, list, count, first, last, hL, pitch, back, turn);
    else
      expand<F16, IO, RB, 2, INF>(a, t0, which, list, count, first, last, hL, pitch, back, turn);
  });
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workgroups of a window: one for every token of a single window (each may have its own adapter),
// one for every adapter of a few, fewer where windows fill the chip and mostly hold one.
// MI355X, 4096 × 4096, windows · slots up to 1024 against 512: 8192 tokens of four requests of
// rank 16 46 and 54 µs, of rank 64 66 and 66, of 40 adapters of rank 16 in any order 235 and 286,
// 2048 of those 71 and 72; against one slot: 64 tokens of 32 adapters 9.7 and 86, 1024 of four
// requests 14.1 and 14.1, but 64 of a single adapter 12.7 and 10.9.
int slots_of(int64_t T, int64_t n) {
  const int64_t windows = cdiv(T, kWindow);
  if (windows == 1) return (int)T;
  int64_t s = std::min<int64_t>(kWindow, n + 1);
  while (s > 2 && windows * s > 1024) s /= 2;
  return (int)s;
}
// Workgroups that have an adapter's tokens, at least: a window's tokens are one request's
// where there are many, and every token may have its own where there are few.
int64_t busy_of(int64_t T, int64_t n) {
  return std::max<int64_t>(cdiv(T, kWindow), T <= kWindow ? std::min(T, n) : 0);
}

// Shares of K: enough workgroups for the chip where there are few, 128 columns a wave at least.
// MI355X, 4096 × 4096, with and without: 64 tokens of 32 adapters 9.7 and 11.0 µs, 256 tokens of
// eight 10.3 and 16.9, 2048 of rank 64 29 and 46.  Up to 1024 workgroups instead of 256: 8192 of
// rank 64 73 against 66 (the second product reads every share), 2048 29 and 29.
int parts_of(int64_t T, int64_t K, int64_t n) {
  int p = 1;
  while (p < 8 && busy_of(T, n) * p < 256 && cdiv(K, 64) >= p * 8) p *= 2;
  return p;
}
// Shares of the channels: 256 each where windows are few.  MI355X, against the power of two below:
// 1800 tokens of five adapters of rank 64 to 2560 channels 27.1 and 32.6 µs, 200 of eight of rank
// 16 to 11008 12.1 and 13.2; against up to 2048 busy workgroups instead of 512, 1000 tokens to
// 11008 19.6 and 20.9, 64 of eight adapters 10.9 and 10.6.  Otherwise a power of two, so that an
// XCD, which takes every eighth workgroup, has the same shares of all windows and keeps their
// weights in its L2.  Each prepares h again, so that they are fewer where windows may hold many
// adapters.  MI355X, 4096 × 4096, against six shares in the order of windows: 8192 tokens of four
// requests of rank 16 46.3 and 47.7 µs, of rank 64 66 and 68, 2048 of rank 64 29 and 32; against
// twice as many shares: 2048 of 40 adapters in any order 70 and 82, 512 of 32 of rank 32 33 and 39.
int64_t channel_shares(int64_t T, int64_t N, int64_t n) {
  const int64_t rounds = cdiv(N, 256), windows = cdiv(T, kWindow);
  const int64_t mixed = std::min<int64_t>(windows * std::min<int64_t>(n, kWindow) / 4, 128);
  const int64_t groups = std::max(busy_of(T, n), mixed);
  if (rounds * groups <= 512 && rounds * windows * slots_of(T, n) <= 2048) return rounds;
  int64_t shares = 1;
  while (shares * 2 <= rounds && shares * 2 * groups <= 768) shares *= 2;
  return shares;
}

// Rows that no cache will hold are kept out of the caches.  MI355X, 5100 tokens × 14336 channels
// (292 MB in and out), rank 64, both launches: 100 µs, 104 without (x stays cached too).
bool streamed(const AdapterArgs& a) { return a.aligned && a.T * a.N >= 1 << 26; }

template <bool F16, int RB>
int launch_adapters(hipStream_t st, AdapterArgs& a) {
  const int64_t shares = channel_shares(a.T, a.N, a.n);
  const int64_t windows = cdiv(a.T, kWindow), most = (1 << 22) / (a.slots * shares);
  // a token's pieces in LDS, and one more against bank conflicts
  const int pitch = (int)(a.R / 4) + 1;
  const size_t lds = (size_t)kWindow * pitch * 16;
  for (a.window = 0; a.window < windows; a.window += most) {
    const unsigned groups = (unsigned)(std::min(windows - a.window, most) * a.slots);
#define G2_SHRINK(ODD) \
  hipLaunchKernelGGL((adapter_shrink_kernel<F16, RB, ODD>), dim3(groups, a.parts), dim3(256), 0, st, a)
    if (a.odd) G2_SHRINK(true);
    else G2_SHRINK(false);
#undef G2_SHRINK
    G2PTQ_LAUNCHED();
    const dim3 grid((unsigned)(groups * shares));
    // (weights of 32 ranks at a time: 64 leave a SIMD fewer waves.  Both launches: 2048 tokens of
    // rank 64, 4096 × 4096, 29.3 and 30.2 µs; 5100 tokens of rank 64 to 14336 channels 100 and 96)
#define G2_EXPAND(IO, RANKS, INF)                                                                 \
  hipLaunchKernelGGL((adapter_expand_kernel<F16, IO, RANKS, INF>), grid, dim3(256), lds, st, a,  \
                     pitch, (int)shares)
    if (a.infinite) G2_EXPAND(kRagged, 1, true);
    else if (a.N % 8) G2_EXPAND(kRagged, RB < 2 ? 1 : 2, false);
    else if (streamed(a)) G2_EXPAND(kStream, RB < 2 ? 1 : 2, false);
    else G2_EXPAND(kPieces, RB < 2 ? 1 : 2, false);
#undef G2_EXPAND
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}

template <bool F16>
int adapters_by_rank(hipStream_t st, AdapterArgs& a) {
  if (a.R <= 16) return launch_adapters<F16, 1>(st, a);
  if (a.R <= 32) return launch_adapters<F16, 2>(st, a);
  return launch_adapters<F16, 4>(st, a);
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
  const int dtype = set->dtype & ~G2PTQ_ADAPTERS_INFINITE;
  G2PTQ_CHECK(dtype == 0 || dtype == 1, "adapters: dtype code %d (bf16 or fp16)", set->dtype);
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
  a.infinite = set->dtype & G2PTQ_ADAPTERS_INFINITE;
  a.odd = reinterpret_cast<uintptr_t>(x) % 4 || (ldx % 2 && T > 1);
  a.aligned = aligned16(base) && aligned16(out) && ldb % 8 == 0 && ldo % 8 == 0;
  hipStream_t st = as_stream(stream);
  return dtype == 0 ? adapters_by_rank<false>(st, a) : adapters_by_rank<true>(st, a);
}
