// Causal attention of ragged chunks of new tokens over the paged cache.
//
//   o[i] = Σ_j p_ij·v̂_j / Σ_j p_ij,   p_ij = exp(c·q_i·k̂_j − max_j(c·q_i·k̂_j))
//
// over the keys j ≤ p_i of the query's sequence, p_i = kv_len − q_len + i the
// position of its i-th new token.  k̂ = s(u − z) and v̂ are what the cache holds
// (kvcache.hip).  A query without keys (kv_len < q_len) gets zeros.
//
// Rows.  The G query heads that share a head of the cache read the same keys and
// values, so the rows of a product are (token, head of the group) pairs: row r
// of a sequence and cache head is token r / G, head r % G.
//
// Numbers.  u − z is an integer of at most 255, exact in fp16 (formed as
// (u − z)·2^-9 from the subnormal fp16 whose bits are u).  A query row is scaled
// by a power of two so that its largest element is in [2^15, 2^16), the top of fp16's
// range, and rounded to fp16: exact for fp16, and for bf16 down to 2^-32 of the largest
// element (smaller ones move by at most 2^-40 of it).  Both products run on the fp16
// matrix cores with fp32 accumulators; scales, softmax statistics and sums are fp32:
//   s_j = (Σ q·(u − z)2^-9)·(2^-6·scale·log2 e·sk_j),  p_j = exp2(C·(s_j − max) + e),
//   l = Σ p_j,  o = 2^9·Σ fp16(p_j·sv_j)·(u − z)2^-9 / l,
// C the row's power of two (so C·max is exact), e = 15 − log2(ref), ref
// a power of two above the scales sv of the values that the row has seen: the
// weights p·sv reach up to 2^15 and keep their 11 bits down to 2^-29 of that.  Rounding
// the weights to fp16 is what lets the matrix cores take them at speed (their fp32 rate is a
// sixteenth).  It moves a weight by at most 2^-11, which the last rounding of bf16 outputs
// covers; fp16 outputs end 3e-4 (relative) from the exact ones where 32-bit weights leave 2e-4.
// One pass over the keys: when the maximum or ref grows, the row's sums are
// scaled back.  Scales are the only numbers of the cache that can be NaN or
// infinite, and a key that a row does not see enters neither its maximum, its
// ref nor its sums.
#include <algorithm>

#include "grid8.hpp"
#include "kvcache.hpp"

namespace g2ptq {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileRows = 128;  // of a workgroup of attend_tiles_kernel
constexpr int kFewRows = 16;  // rows of a sequence and head up to which attend_rows_kernel runs

struct AttnArgs {
  KvCache c;
  const void* q;
  int64_t qt, qh;  // strides of query token and head
  void* out;       // T × Hq × D, contiguous
  int64_t ldt;
  const int32_t *table, *cu, *kv;
  int T, Hq, B, G, width;
  int dtype;
  bool vec;        // 16-byte loads of queries
  float scale;
  float kscale;    // |scale|·log2 e·2^(9 − 15): multiplies the keys' scales
  int tiles;       // row tiles a launch provides for a sequence and head (attend_tiles_kernel)
  int split, few_split;  // most shares of a sequence's keys (tiles; few rows)
  int share, few_share;  // keys of a share, unless a sequence needs larger ones
  bool by_rows, by_tiles;  // kernels that run; with both, sequences of at most kFewRows rows
                           // go to attend_rows_kernel
  float *part, *few_part;  // partial results of the shares, or null
  int64_t row0;            // first row of a launch of attend_join_kernel
};

// A sequence's rows of the query and its keys.
struct Span {
  int q0, qlen;  // first query row, query rows
  int pos0;      // position of the first new token (negative: queries without keys)
  int n;         // keys that the page table has
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  Span s;
  s.q0 = min(max(a.cu[b], 0), a.T);
  s.qlen = min(max(a.cu[b + 1], s.q0), a.T) - s.q0;
  const int kv = a.kv[b];
  s.pos0 = kv - s.qlen;
  const int64_t room = (int64_t)a.width << a.c.shift;
  s.n = a.c.pages == 0 ? 0 : (int)min<int64_t>(max(kv, 0), room);
  if (kv > s.n && s.qlen > 0 && threadIdx.x == 0) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);
  return s;
}

// The shares of n keys: of `share` keys each (a multiple of `step`; sequences of a batch
// differ in length, their shares do not), larger ones where `most` would not do.
struct Shares {
  int each, count;
};
__device__ __forceinline__ Shares shares_of(int n, int most, int share, int step) {
  const int each = max(share, ((n + most - 1) / most + step - 1) / step * step);
  return {each, max(1, (n + each - 1) / each)};
}

__device__ __forceinline__ f16x2 as_h2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }

// (u − z)·2^-9 of two codes held as 16-bit integers; zc = −z·2^-9 twice.
__device__ __forceinline__ f16x2 centred(uint32_t two, f16x2 zc) {
  const f16x2 up = {(_Float16)32768.f, (_Float16)32768.f};
  return __builtin_elementwise_fma(as_h2(two), up, zc);
}
// The same of 4-bit codes in the low (H = 0) or high half of the words' low bytes: 16u is as
// good a subnormal as u, and needs no shift.
template <int H>
__device__ __forceinline__ f16x2 centred4(uint32_t two, f16x2 zc) {
  const _Float16 f = (_Float16)(H ? 2048.f : 32768.f);
  const f16x2 up = {f, f};
  return __builtin_elementwise_fma(as_h2(two & (H ? 0x00f000f0u : 0x000f000fu)), up, zc);
}
__device__ __forceinline__ f16x2 centre(int z0, int z1) {
  return f16x2{(_Float16)((float)-z0 * 0x1p-9f), (_Float16)((float)-z1 * 0x1p-9f)};
}

// Eight channels of one key, in the order channel_of gives.
template <int BITS>
__device__ __forceinline__ f16x8 key_codes(const uint32_t* w, f16x2 zc) {
  f16x2 h[4];
  if constexpr (BITS == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[2 * i] = centred(__builtin_amdgcn_perm(0, w[i], 0x0c010c00), zc);
      h[2 * i + 1] = centred(__builtin_amdgcn_perm(0, w[i], 0x0c030c02), zc);
    }
  } else {
    h[0] = centred4<0>(w[0], zc), h[1] = centred4<1>(w[0], zc);
    h[2] = centred4<0>(w[0] >> 8, zc), h[3] = centred4<1>(w[0] >> 8, zc);
  }
  return f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}
// Position i of key_codes' eight channels (4-bit codes: i and i + 4 side by side).
template <int BITS>
__device__ __forceinline__ constexpr int channel_of(int i) {
  return BITS == 8 ? i : (i >> 1) + 4 * (i & 1);
}

// Channel e (of eight) of two tokens' values.
template <int BITS>
__device__ __forceinline__ f16x2 value_codes(const uint32_t* a, const uint32_t* b, int e,
                                             f16x2 zc) {
  if constexpr (BITS == 8) {
    const uint32_t k = e & 3;
    return centred(__builtin_amdgcn_perm(b[e >> 2], a[e >> 2], 0x0c000c00u | (4 + k) << 16 | k), zc);
  } else {
    const uint32_t k = e >> 1;
    const uint32_t two = __builtin_amdgcn_perm(b[0], a[0], 0x0c000c00u | (4 + k) << 16 | k);
    return e & 1 ? centred4<1>(two, zc) : centred4<0>(two, zc);
  }
}

// Power of two just above the finite scale x, from 2^-90 up.
__device__ __forceinline__ float above(float x) {
  const uint32_t e = (__float_as_uint(x) & 0x7f800000u) + 0x00800000u;
  return __uint_as_float(max(e, (uint32_t)(127 - 90) << 23));
}
__device__ __forceinline__ int exponent(float p) { return (int)(__float_as_uint(p) >> 23) - 127; }

// Power of two that brings a query row's largest |q| (16 bits of the query's type in the
// high half of m) into [2^15, 2^16), and 2^15 times its inverse.  Rows below 2^-112 stay
// below that (the power has to be a number).
struct RowScale {
  float down, up;
};
__device__ __forceinline__ RowScale row_scale(int dtype, uint32_t m) {
  const float x = dtype == 0 ? __uint_as_float(m)
                             : (float)__builtin_bit_cast(_Float16, (uint16_t)(m >> 16));
  uint32_t e = __float_as_uint(x) >> 23;
  // A NaN or an infinity makes every logit of the row NaN or infinite, and their softmax NaN
  // (also where all are -inf, which would look like a row without keys): NaN as the unit.
  if (e >= 255) return {1.f, __builtin_nanf("")};
  e = max(e, 15u);
  return {__uint_as_float((269 - e) << 23), __uint_as_float(e << 23)};
}

// Output row of sequence row r, or -1 past the sequence's rows.
struct RowAt {
  int token, head;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs& a, const Span& s, int h, int r) {
  const uint32_t t = (uint32_t)r / (uint32_t)a.G;
  return {s.q0 + (int)t, h * a.G + (r - (int)t * a.G)};
}

template <int N>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, const float (&y)[N]) {
  uint16_t w[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    w[i] = a.dtype == 0 ? __builtin_bit_cast(uint16_t, (__bf16)y[i])
                        : __builtin_bit_cast(uint16_t, (_Float16)y[i]);
  uint16_t* o = static_cast<uint16_t*>(a.out) + at;
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(o) = make_uint4(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16,
                                              w[4] | (uint32_t)w[5] << 16, w[6] | (uint32_t)w[7] << 16);
  else
    *reinterpret_cast<uint2*>(o) = make_uint2(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16);
}

// Pieces of eight channels of a query row as they are, piece s from channel
// channel(s) (zeros from channel D up).
template <int N, typename F>
__device__ __forceinline__ void load_query(const AttnArgs& a, int64_t at, uint4 (&raw)[N], int D,
                                           F channel) {
  const uint16_t* x = static_cast<const uint16_t*>(a.q) + at;
#pragma unroll
  for (int s = 0; s < N; ++s) raw[s] = make_uint4(0, 0, 0, 0);
  if (a.vec) {
#pragma unroll
    for (int s = 0; s < N; ++s)
      if (channel(s) < D) raw[s] = *reinterpret_cast<const uint4*>(x + channel(s));
  } else {
#pragma nounroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int s = 0; s < N; ++s)
        if (channel(s) < D) {
          const uint16_t* y = x + channel(s) + 2 * i;
          const uint32_t w = y[0] | (uint32_t)y[1] << 16;
          raw[s].x = i == 0 ? w : raw[s].x, raw[s].y = i == 1 ? w : raw[s].y;
          raw[s].z = i == 2 ? w : raw[s].z, raw[s].w = i == 3 ? w : raw[s].w;
        }
    }
  }
}

// Scaled (and negated for a negative scale of the logits) to fp16, in the order of
// key_codes.
template <int BITS>
__device__ __forceinline__ f16x8 scaled_query(const AttnArgs& a, uint4 raw, float down) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  const float f = a.scale < 0.f ? -down : down;
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (a.dtype == 0) {
      v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
      v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
    }
  }
  f16x8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (_Float16)(v[channel_of<BITS>(i)] * f);
  return h;
}

// A partial result: the row's output over a share of the keys (D floats), its
// maximum (log2 units) and its sum.
__device__ __forceinline__ int64_t part_size(const AttnArgs& a) { return a.c.D + 4; }

// Query rows outside every sequence.
__device__ void clear_outside(const AttnArgs& a) {
  const int lo = a.B ? min(max(a.cu[0], 0), a.T) : a.T;
  const int hi = a.B ? min(max(a.cu[a.B], 0), a.T) : a.T;
  const int64_t row = a.Hq * a.c.D / 8;
  uint4* o = static_cast<uint4*>(a.out);
  for (int64_t i = threadIdx.x; i < lo * row; i += blockDim.x) o[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = hi * row + threadIdx.x; i < a.T * row; i += blockDim.x)
    o[i] = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Few rows (decoding): the keys' and values' bytes are what counts.  A wave takes
// 32 keys at a time straight into registers, laid out so that neither operand
// needs a shuffle: with v_mfma_f32_16x16x32_f16,
//   S^T (16 keys × 16 rows) = K·Q^T: lane (key, g) loads a quarter g of the key's
//     channels in one piece, the query's channels are laid out alike;
//   O^T (channels × 16 rows) += V^T·P^T: lane (n, g) loads channels n·DV .. of the
//     eight tokens whose weights lie in its own registers after the softmax
//     (4g .. 4g + 3 and 16 + 4g ..), so P^T needs no exchange; channel n·DV + e is
//     row n of the e-th product.
// Row statistics are per lane (row = lane % 16).  Four waves interleave blocks of 32
// keys and join through LDS; `few_split` workgroups share a sequence's keys.
// DP: channels rounded up to 64, 128 or 256 (FULL: D == DP).
// Bound by the cache's bytes at 8 bits and by vector arithmetic (two to three
// instructions per two codes) and the loads a CU keeps under way about alike at 4, where heads
// of 128 also spill 13 of a lane's registers under the bound of three waves.  MI355X, back to
// back and with the join, heads 32 on 8 of 128, 8 bits: one query over 131072 keys 51 µs
// (5.4 TB/s), 64 over 4096 each 99 µs (5.6 TB/s); 4 bits: 64 over 4096 60 µs (4.8 TB/s); one
// over 4001 at 8 bits 12 µs, of which 8.3 here and 4 in the join, latency.  Up to 16 rows, one
// block of the product's columns: 32 uneven sequences with 2 tokens of 8 heads 38 µs, 74 by
// attend_tiles_kernel; 4 tokens over 8192 keys 14.4 against 24.6 µs.  More rows of one token
// (over 16 query heads on a head of the cache) go to attend_tiles_kernel unmeasured.
// ---------------------------------------------------------------------------
template <int BITS, int DP, bool FULL>
__global__ __launch_bounds__(256, DP == 64 ? 3 : DP == 128 ? (BITS == 4 ? 3 : 2) : 1) void
attend_rows_kernel(AttnArgs a) {
  constexpr int DG = DP / 4;                  // channels of a lane's share of a key
  constexpr int KW = DG * BITS / 32;          // its words
  constexpr int KS = DP / 32;                 // products of 32 channels
  constexpr int DV = DP / 16;                 // channels of a lane's share of a value
  constexpr int VW = (DV * BITS + 31) / 32;   // its words
  constexpr int PITCH = DP + 4;
  // a wave's steps: rows in the cache, scales, zero points (two buffers); then the join
  __shared__ uint32_t rowL[4][2][32], zkL[4][2][32];
  __shared__ __attribute__((aligned(16))) float skL[4][2][32], svL[4][2][32];
  __shared__ __attribute__((aligned(8))) _Float16 zvL[4][2][32];
  __shared__ __attribute__((aligned(16))) float oL[4][16 * PITCH];
  __shared__ float mL[4][16], lL[4][16];

  // Workgroups go round the 8 XCDs: the heads' shares of the same pages mostly meet on one,
  // and turned by the sequence, the last shares (short sequences have fewer) on all.
  const int b = blockIdx.z, h = blockIdx.y, split = (blockIdx.x + b) % gridDim.x;
  if (b == a.B) {
    if (h == 0 && split == 0) clear_outside(a);
    return;
  }
  const Span sp = span_of(a, b);
  const int rows = sp.qlen * a.G;
  if (rows == 0 || (a.by_tiles && rows > kFewRows)) return;
  const Shares sh = rows > kFewRows ? Shares{sp.n, 1}
                                    : shares_of(sp.n, a.few_split, a.few_share, 128);
  if (split >= sh.count) return;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int D = FULL ? DP : (int)a.c.D;
  const uint32_t rowb = D * BITS / 8;
  const int half = 1 << (BITS - 1);
  const int32_t* table = a.table + b * a.ldt;

  for (int r0 = 0; r0 < rows; r0 += 16) {
    const RowAt at = row_at(a, sp, h, min(r0 + n, rows - 1));
    // the last key that the lane's row sees; that every and that any of the block's rows sees
    const int last = min(sp.pos0 + (at.token - sp.q0), sp.n - 1);
    const int first_all = min(sp.pos0 + r0 / a.G, sp.n - 1);  // seen by every row of the block
    const int last_all = min(sp.pos0 + (min(r0 + 15, rows - 1)) / a.G, sp.n - 1);
    const int k0 = split * sh.each + 32 * wave, k1 = min(last_all + 1, (split + 1) * sh.each);
    const int steps = k1 > k0 ? (k1 - k0 + 127) / 128 : 0;  // blocks of 32 keys, every 128

    // A step's pages (P), rows and numbers (M, shown to the wave by S), codes (C): loaded
    // three, two and one step ahead of the arithmetic.  Lanes 0 .. 31 are for keys, the
    // others for values.
    const int kv = lane >> 5;
    int page = -1, sz = half, bad = 0;
    uint32_t srow = 0;
    float sc = 0.f;
    bool sok = false;
#define G2_P(step) page = table[max(min(k0 + (step) * 128 + (lane & 31), k1 - 1), 0) >> a.c.shift]
#define G2_M(step)                                                                           \
  do {                                                                                       \
    const int key_ = k0 + (step) * 128 + (lane & 31);                                        \
    sok = (key_ < k1) & ((uint32_t)page < (uint64_t)a.c.pages);                              \
    bad |= (key_ < k1) & !sok;                                                               \
    const int pg_ = sok ? page : 0, of_ = sok ? key_ & ((1 << a.c.shift) - 1) : 0;           \
    srow = ((uint32_t)(pg_ * (int)a.c.H + h) << a.c.shift) + of_;                            \
    sc = (kv ? a.c.scale[1] : a.c.scale[0])[srow];                                           \
    if (a.c.zero[0]) sz = (kv ? a.c.zero[1] : a.c.zero[0])[srow];                            \
  } while (0)
#define G2_S(buf, ok)                                                                        \
  do {                                                                                       \
    if (!sok) sc = 0.f;                                                                      \
    ok = __builtin_amdgcn_ballot_w64(sok && (!kv || sc < __builtin_inff()));                 \
    if (kv) {                                                                                \
      svL[wave][buf][lane - 32] = sc;                                                        \
      zvL[wave][buf][lane - 32] = centre(sz, sz)[0];                                         \
    } else {                                                                                 \
      rowL[wave][buf][lane] = srow;                                                          \
      skL[wave][buf][lane] = sc * a.kscale;                                                  \
      zkL[wave][buf][lane] = __builtin_bit_cast(uint32_t, centre(sz, sz));                   \
    }                                                                                        \
    __builtin_amdgcn_wave_barrier();                                                         \
  } while (0)
#define G2_C(buf, kw, vw)                                                                    \
  do {                                                                                       \
    _Pragma("unroll") for (int kb = 0; kb < 2; ++kb) {                                       \
      const uint8_t* p_ = a.c.codes[0] + (uint64_t)rowL[wave][buf][16 * kb + n] * rowb +     \
                          g * (DG * BITS / 8);                                               \
      if constexpr (FULL && KW % 4 == 0) {                                                   \
        _Pragma("unroll") for (int i = 0; i < KW / 4; ++i) {                                 \
          const uint4 v_ = reinterpret_cast<const uint4*>(p_)[i];                            \
          kw[kb][4 * i] = v_.x, kw[kb][4 * i + 1] = v_.y;                                    \
          kw[kb][4 * i + 2] = v_.z, kw[kb][4 * i + 3] = v_.w;                                \
        }                                                                                    \
      } else {                                                                               \
        _Pragma("unroll") for (int i = 0; i < KW / 2; ++i) { /* 8 or 16 channels */          \
          uint2 v_ = make_uint2(0, 0);                                                       \
          if (FULL || g * DG + i * (64 / BITS) < D)                                          \
            v_ = reinterpret_cast<const uint2*>(p_)[i];                                      \
          kw[kb][2 * i] = v_.x, kw[kb][2 * i + 1] = v_.y;                                    \
        }                                                                                    \
      }                                                                                      \
    }                                                                                        \
    _Pragma("unroll") for (int j = 0; j < 8; ++j) {                                          \
      const int t_ = (j < 4 ? 4 * g + j : 16 + 4 * g + j - 4);                               \
      uint64_t o_ = (uint64_t)rowL[wave][buf][t_] * rowb + n * (DV * BITS / 8);              \
      if (!FULL) o_ = n * DV < D ? o_ : 0;                                                   \
      const uint8_t* p_ = a.c.codes[1] + o_;                                                 \
      if constexpr (DV * BITS == 16) {                                                       \
        vw[j][0] = *reinterpret_cast<const uint16_t*>(p_);                                   \
      } else if constexpr (VW == 1) {                                                        \
        vw[j][0] = *reinterpret_cast<const uint32_t*>(p_);                                   \
      } else if constexpr (VW == 2) {                                                        \
        const uint2 v_ = *reinterpret_cast<const uint2*>(p_);                                \
        vw[j][0] = v_.x, vw[j][1] = v_.y;                                                    \
      } else {                                                                               \
        const uint4 v_ = *reinterpret_cast<const uint4*>(p_);                                \
        vw[j][0] = v_.x, vw[j][1] = v_.y, vw[j][2] = v_.z, vw[j][3] = v_.w;                  \
      }                                                                                      \
    }                                                                                        \
  } while (0)
    uint32_t ka[2][KW], va[8][VW], kb_[2][KW], vb[8][VW];
    // low half: keys that are there; high half: those whose value's scale is finite
    uint64_t oka = 0, okb = 0;
    if (steps > 0) {
      G2_P(0);
      G2_M(0);
      G2_P(1);
    }

    // query: channels g·DG + 8s .. of row n, scaled into fp16
    f16x8 qf[KS];
    float C;
    {
      uint4 raw[KS];
      uint32_t top = 0;
      load_query<KS>(a, at.token * a.qt + at.head * a.qh, raw, D,
                     [&](int s) { return g * DG + 8 * s; });
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t w[4] = {raw[s].x, raw[s].y, raw[s].z, raw[s].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = max(top, max(w[i] << 16 & 0x7fff0000u, w[i] & 0x7fff0000u));
      }
      top = max(top, __shfl_xor(top, 16));
      top = max(top, __shfl_xor(top, 32));
      const RowScale rs = row_scale(a.dtype, top);
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = scaled_query<BITS>(a, raw[s], rs.down);
      C = rs.up;
    }

    f32x4 acc[DV];
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[e] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f, ref = 0x1p-90f;

    auto arithmetic = [&](int j0, int buf, uint64_t ok, const uint32_t (&kw)[2][KW],
                          const uint32_t (&vw)[8][VW]) __attribute__((always_inline)) {
      float p[8], sv[8];
      float mx = m, vx = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const f16x2 zc = as_h2(zkL[wave][buf][16 * kb + n]);
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s)
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_codes<BITS>(&kw[kb][s * BITS / 4], zc),
                                                     qf[s], x, 0, 0, 0);
        const f32x4 sk = *reinterpret_cast<const f32x4*>(&skL[wave][buf][16 * kb + 4 * g]);
        const f32x4 s4 = *reinterpret_cast<const f32x4*>(&svL[wave][buf][16 * kb + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[4 * kb + i] = x[i] * sk[i], sv[4 * kb + i] = s4[i];
      }
      const bool whole = ok == ~0ull && j0 + 31 <= first_all;  // every row sees every key
      uint32_t see = 0;  // bit i: element i = 4kb + i%4 is key 16kb + 4g + i%4 of the step
      if (__builtin_expect(whole, 1)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, p[i]), vx = fmaxf(vx, sv[i]);
      } else {
        const int c = last - j0;  // the last key seen
        const uint32_t seen = (c < 0 ? 0u : (uint32_t)ok) & (~0u >> (31 - min(max(c, 0), 31)));
        see = (seen >> (4 * g) & 15u) | (seen >> (16 + 4 * g) & 15u) << 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool on = see >> i & 1;
          mx = fmaxf(mx, on ? p[i] : -INFINITY);
          vx = fmaxf(vx, on && sv[i] < __builtin_inff() ? sv[i] : 0.f);
        }
      }
      // ---- the row's units: m and ref are the same in its four lanes, and grow rarely ----
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx > m || vx >= ref) != 0, 0)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        vx = fmaxf(vx, __shfl_xor(vx, 16));
        vx = fmaxf(vx, __shfl_xor(vx, 32));
        const float nref = vx >= ref ? above(vx) : ref;
        float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * C);
        if (m == mx) f = 1.f;
        f = __builtin_amdgcn_ldexpf(f, exponent(ref) - exponent(nref));
        m = mx, ref = nref;
        l *= f;
#pragma unroll
        for (int e = 0; e < DV; ++e) acc[e] *= f;
      }
      asm volatile("" : "+v"(m), "+v"(ref));  // (as in attend_tiles_kernel)
      const float e0 = (float)(15 - exponent(ref)), m0 = m == -INFINITY ? 0.f : m;
      f16x8 w;
      if (__builtin_expect(whole, 1)) {
        asm volatile("");  // (keeps the branches apart: no selects here)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i] - m0, C, e0));
          l += x;
          w[i] = (_Float16)(x * sv[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool on = see >> i & 1;
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i] - m0, C, e0));
          l += on ? x : 0.f;
          w[i] = (_Float16)(on ? x * sv[i] : 0.f);
        }
      }
      // ---- values ----
      const f16x4 z0 = *reinterpret_cast<const f16x4*>(&zvL[wave][buf][4 * g]);
      const f16x4 z1 = *reinterpret_cast<const f16x4*>(&zvL[wave][buf][16 + 4 * g]);
      const f16x2 zc[4] = {{z0[0], z0[1]}, {z0[2], z0[3]}, {z1[0], z1[1]}, {z1[2], z1[3]}};
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        f16x2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = value_codes<BITS>(&vw[2 * i][e / 8 * (BITS / 4)],
                                   &vw[2 * i + 1][e / 8 * (BITS / 4)], e & 7, zc[i]);
        const f16x8 vf = {v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
        acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, w, acc[e], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();
    };
    if (steps > 0) {
      G2_S(0, oka);
      G2_C(0, ka, va);
      G2_M(1);
      G2_P(2);
    }
    for (int step = 0; step < steps; step += 2) {
      G2_S(1, okb);
      G2_C(1, kb_, vb);
      G2_M(step + 2);
      G2_P(step + 3);
      arithmetic(k0 + step * 128, 0, oka, ka, va);
      if (step + 1 == steps) break;
      G2_S(0, oka);
      G2_C(0, ka, va);
      G2_M(step + 3);
      G2_P(step + 4);
      arithmetic(k0 + step * 128 + 128, 1, okb, kb_, vb);
    }
#undef G2_P
#undef G2_M
#undef G2_S
#undef G2_C
    if (bad) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);

    // ---- join the four waves: units of the block's maximum, true scale ----
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    l = __builtin_amdgcn_ldexpf(l, exponent(ref) - 15);
    if (g == 0) mL[wave][n] = m, lL[wave][n] = l;
    __syncthreads();
    const float M = fmaxf(fmaxf(mL[0][n], mL[1][n]), fmaxf(mL[2][n], mL[3][n]));
    {
      // (a wave without keys has m = -inf and sums of zero)
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * C);
      const float back = __builtin_amdgcn_ldexpf(f, exponent(ref) - 15 + 9);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DV; ++e)
          oL[wave][n * PITCH + (4 * g + i) * DV + e] = acc[e][i] * back;
      if (g == 0) lL[wave][n] = l * f;
    }
    __syncthreads();
    const float MC = M * C;  // of row n, as every wave has it
    for (int i = threadIdx.x; i < 16 * (D / 8); i += 256) {
      // i % 16 == lane % 16: row n of this lane is row r
      const int r = i & 15, d = (i >> 4) * 8;
      if (r0 + r >= rows) continue;
      const float L = lL[0][r] + lL[1][r] + lL[2][r] + lL[3][r];
      const float inv = L == 0.f ? 0.f : 1.f / L;
      float y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        y[k] = (oL[0][r * PITCH + d + k] + oL[1][r * PITCH + d + k] + oL[2][r * PITCH + d + k] +
                oL[3][r * PITCH + d + k]) * inv;
      if (sh.count > 1) {
        float* o = a.few_part +
                   ((((int64_t)b * a.c.H + h) * kFewRows + r) * a.few_split + split) * part_size(a);
        *reinterpret_cast<float4*>(o + d) = make_float4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<float4*>(o + d + 4) = make_float4(y[4], y[5], y[6], y[7]);
        if (d == 0) o[D] = M == -INFINITY ? -INFINITY : MC, o[D + 1] = L;
      } else {
        const RowAt ra = row_at(a, sp, h, r0 + r);
        store_out(a, ((int64_t)ra.token * a.Hq + ra.head) * D + d, y);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Many rows (chunks of prompts): matrix cores.  A workgroup of four waves takes 128
// rows, 32 per wave, through 64 keys at a time.  The keys and values of a step are
// converted to fp16 once per workgroup and kept in LDS, keys as [key][channel], values
// transposed as [channel][key] (two buffers each); the codes after them are loaded
// meanwhile.  The first two waves look up pages, scales and zero points three steps
// ahead (a ring of four).  A step is softmax and staging, a barrier, and the products
// of its values and the next step's keys.  v_mfma_f32_32x32x16_f16:
//   S^T (32 keys × 32 rows) = K·Q^T, so that a lane holds one row's logits (row =
//     lane % 32, the other half of the keys in lane + 32) and its statistics;
//   O^T (channels × rows) += V^T·P^T with the weights as they lie: the eight keys of
//     a lane's operand are 16t + 4h .. and 16t + 8 + 4h .. (h = lane / 32), and V^T is
//     stored with its keys in that order.
// LDS rows are 16 bytes longer than their data, so that fragment reads (16 consecutive
// rows, one 16-byte chunk) touch all banks; values' rows also hold chunk c at
// c ^ (channel / 16), which spreads the writes (8 rows 8 channels apart, one chunk).
// Bound by the products, whose operands come from LDS at about the rate the matrix cores
// take them (a wave's 32 rows read all of a step's keys and values), and the softmax between
// them, which the two workgroups of a CU overlap only in part: MI355X, 2048 tokens over 16384
// keys, heads 32 on 8 of 128, 8 bits, back to back 654–668 µs, 770–790 TFLOP/s (the library's
// largest bf16 product: 1520; under the profiler, with the clocks of single launches, 689 at
// best and 746 on average).  Slower: waves in two groups that take turns at softmax and
// products (780 against 688 µs then), steps of 32 keys (915 against 795); both read as much
// from LDS for a product.  Heads of 129 to 256 channels put 20 bytes a lane into scratch.
// ---------------------------------------------------------------------------
// Largest of 64 lanes' non-negative x (rows of 16 lanes, then across rows, into lane 63).
__device__ __forceinline__ float wave_max(float x) {
#define G2_DPP(ctrl, rows)                                                                   \
  x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(                        \
                                             0, __builtin_bit_cast(int, x), ctrl, rows, 0xf, \
                                             false)))
  G2_DPP(0x111, 0xf);  // row_shr 1, 2, 4, 8
  G2_DPP(0x112, 0xf);
  G2_DPP(0x114, 0xf);
  G2_DPP(0x118, 0xf);
  G2_DPP(0x142, 0xa);  // row_bcast 15 into rows 1 and 3
  G2_DPP(0x143, 0xc);  // row_bcast 31 into rows 2 and 3
#undef G2_DPP
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

template <int BITS, int DP, bool FULL>
__global__ __launch_bounds__(2 * kTileRows, DP <= 128 ? 2 : 1) void
attend_tiles_kernel(AttnArgs a) {
  constexpr int NT = 2 * kTileRows, BM = kTileRows, BN = 64;
  constexpr int KC = BN * (DP / 16) / NT;                          // 16-channel pieces of keys
  constexpr int VP = BN / 4 * (DP / 8), VQ = (VP + NT - 1) / NT;   // 4-key × 8-channel of values
  constexpr int KW = BITS / 2, VW = BITS / 4;   // words of 16 and of 8 channels
  constexpr int KPITCH = DP * 2 + 16, VPITCH = BN * 2 + 16;  // bytes of an LDS row
  constexpr int KB = BN * KPITCH, VB = DP * VPITCH;          // of a step's keys and values
  __shared__ __attribute__((aligned(16))) char kL[2 * KB], vL[2 * VB];
  __shared__ __attribute__((aligned(16))) float skL[4][BN], svL[4][BN];
  __shared__ __attribute__((aligned(16))) uint32_t rowL[4][BN];
  __shared__ uint32_t zkL[4][BN];  // −z·2^-9 in fp16, twice
  __shared__ __attribute__((aligned(16))) _Float16 zvL[4][BN];
  __shared__ float vmaxL[4];
  __shared__ uint64_t okL[4];

  // Workgroups go round the 8 XCDs; number them so that an XCD takes a contiguous
  // range: the row tiles of one sequence and head share its keys in one L2.  (Heads last:
  // the sequences, which differ in length, are spread over the XCDs.)
  const int total = a.B * (int)a.c.H * a.split * a.tiles;
  if ((int)blockIdx.x == total) {
    clear_outside(a);
    return;
  }
  int id;
  {
    const int q8 = total >> 3, r8 = total & 7, xcd = blockIdx.x & 7;
    id = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
  }
  const int tile0 = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.split;
  id /= a.split;
  const int b = id % a.B, h = id / a.B;
  const Span sp = span_of(a, b);
  const int rows = sp.qlen * a.G;
  if (rows == 0 || (a.by_rows && rows <= kFewRows)) return;
  const Shares sh = shares_of(sp.n, a.split, a.share, BN);
  if (split >= sh.count) return;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = FULL ? DP : (int)a.c.D;
  const uint32_t rowb = D * BITS / 8;
  const int half = 1 << (BITS - 1);
  const int32_t* table = a.table + b * a.ldt;
  const int ntile = (rows + BM - 1) / BM;

  // Keys: piece p = tid + i·NT is 16 channels c of key p / (DP/16).  Values: bits of a
  // piece from low to high: 3 of the 8-channel group, 1 half of the chunk (8 keys), the
  // group's other bits, 3 of the chunk; with fewer pieces than threads the upper half
  // of the workgroup takes them.
  const int tv = VP < NT ? (tid + NT / 2) % NT : tid;
  const int first_v = VP < NT ? (wave * 64 + NT / 2) % NT : wave * 64;  // of the wave
  constexpr int OH = DP / 64;  // 8-channel groups over 8

  // the longest tiles (the last rows) first
  for (int tile = ntile - 1 - tile0; tile >= 0; tile -= a.tiles) {
    const int r0 = tile * BM, r = r0 + wave * 32 + lr;
    const RowAt at = row_at(a, sp, h, min(r, rows - 1));
    const int last = min(sp.pos0 + (at.token - sp.q0), sp.n - 1);
    const int first_all = min(sp.pos0 + r0 / a.G, sp.n - 1);  // seen by every row of the tile
    const int last_all = min(sp.pos0 + (min(r0 + BM, rows) - 1) / a.G, sp.n - 1);
    const int k0 = split * sh.each, k1 = min(last_all + 1, k0 + sh.each);
    const int steps = k1 > k0 ? (k1 - k0 + BN - 1) / BN : 0;

    // query fragments: chunk c = 2s + lh of keys' LDS rows holds channels 16c .. + 7
    // for c < DP/16 and 16(c − DP/16) + 8 .. above
    f16x8 qf[DP / 16];
    float C;
    {
      uint4 raw[DP / 16];
      uint32_t m = 0;
      load_query<DP / 16>(a, at.token * a.qt + at.head * a.qh, raw, D, [&](int s) {
        const int c = 2 * s + lh;
        return c < DP / 16 ? 16 * c : 16 * (c - DP / 16) + 8;
      });
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        const uint32_t w[4] = {raw[s].x, raw[s].y, raw[s].z, raw[s].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(w[i] << 16 & 0x7fff0000u, w[i] & 0x7fff0000u));
      }
      m = max(m, __shfl_xor(m, 32));
      const RowScale rs = row_scale(a.dtype, m);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) qf[s] = scaled_query<BITS>(a, raw[s], rs.down);
      C = rs.up;
    }

    f32x16 acc[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[e][v] = 0.f;
    float m = -INFINITY, l = 0.f, ref = 0x1p-90f;
    int bad = 0;

    // first wave (keys) and second (values): page of key `lane` of a step (−1: none),
    // then its row and numbers
    int page = -1;
#define G2_PAGE(step)                                                                        \
  do {                                                                                       \
    const int key_ = k0 + (step) * BN + lane;                                                \
    page = table[min(key_, k1 - 1) >> a.c.shift];                                            \
  } while (0)
    bool sok = false;
    uint32_t srow = 0;
    float sc = 0.f;
    int sz = half;
#define G2_META(step)                                                                        \
  do {                                                                                       \
    const int key_ = k0 + (step) * BN + lane;                                                \
    const int64_t pages_ = a.c.pages;                                                        \
    sok = (key_ < k1) & ((uint32_t)page < (uint64_t)pages_);                                 \
    bad |= (key_ < k1) & !sok;                                                               \
    const int pg_ = sok ? page : 0, of_ = sok ? key_ & ((1 << a.c.shift) - 1) : 0;           \
    srow = ((uint32_t)(pg_ * (int)a.c.H + h) << a.c.shift) + of_;                            \
    sc = a.c.scale[wave][srow];                                                              \
    if (a.c.zero[0]) sz = a.c.zero[wave][srow];                                              \
  } while (0)
#define G2_SHOW(at4)                                                                         \
  do {                                                                                       \
    if (!sok) sc = 0.f;                                                                      \
    if (wave == 0) {                                                                         \
      skL[at4][lane] = sc * a.kscale;                                                        \
      rowL[at4][lane] = srow;                                                                \
      zkL[at4][lane] = __builtin_bit_cast(uint32_t, centre(sz, sz));                         \
      const uint64_t ok_ = __builtin_amdgcn_ballot_w64(sok);                                 \
      okL[at4] = ok_;                                                                        \
    } else {                                                                                 \
      svL[at4][lane] = sc;                                                                   \
      zvL[at4][lane] = centre(sz, sz)[0];                                                    \
      const float vx_ = wave_max(sc < __builtin_inff() ? sc : 0.f);                          \
      vmaxL[at4] = vx_;                                                                      \
    }                                                                                        \
  } while (0)
    uint32_t kw[KC][KW], vw[VQ][4][VW];
#define G2_FETCH_K(at4)                                                                      \
  do {                                                                                       \
    _Pragma("unroll") for (int i = 0; i < KC; ++i) {                                         \
      const int p_ = tid + i * NT, c_ = p_ % (DP / 16);                                      \
      uint64_t o_ = (uint64_t)rowL[at4][p_ / (DP / 16)] * rowb + c_ * (2 * BITS);            \
      if (!FULL) o_ = c_ * 16 < D ? o_ : 0;                                                  \
      const uint8_t* s_ = a.c.codes[0] + o_;                                                 \
      if constexpr (BITS == 8) {                                                             \
        const uint4 v_ = *reinterpret_cast<const uint4*>(s_);                                \
        kw[i][0] = v_.x, kw[i][1] = v_.y, kw[i][2] = v_.z, kw[i][3] = v_.w;                  \
      } else {                                                                               \
        const uint2 v_ = *reinterpret_cast<const uint2*>(s_);                                \
        kw[i][0] = v_.x, kw[i][1] = v_.y;                                                    \
      }                                                                                      \
    }                                                                                        \
  } while (0)
#define G2_FETCH_V(at4)                                                                      \
  do {                                                                                       \
    _Pragma("unroll") for (int i = 0; i < VQ; ++i) {                                         \
      const int p_ = tv + i * NT, o_ = (p_ & 7) + 8 * ((p_ >> 4) % OH), ch_ = (p_ >> 4) / OH;\
      if (VP % NT && first_v + i * NT >= VP) break;                                          \
      const uint4 r_ = *reinterpret_cast<const uint4*>(                                      \
          &rowL[at4][16 * (ch_ >> 1) + 4 * (ch_ & 1) + 8 * ((p_ >> 3) & 1)]);                \
      const uint32_t row_[4] = {r_.x, r_.y, r_.z, r_.w};                                     \
      _Pragma("unroll") for (int t = 0; t < 4; ++t) {                                        \
        uint64_t at_ = (uint64_t)row_[t] * rowb + o_ * BITS;                                 \
        if (!FULL) at_ = o_ * 8 < D ? at_ : 0;                                               \
        const uint8_t* s_ = a.c.codes[1] + at_;                                              \
        if constexpr (BITS == 8) {                                                           \
          const uint2 v_ = *reinterpret_cast<const uint2*>(s_);                              \
          vw[i][t][0] = v_.x, vw[i][t][1] = v_.y;                                            \
        } else {                                                                             \
          vw[i][t][0] = *reinterpret_cast<const uint32_t*>(s_);                              \
        }                                                                                    \
      }                                                                                      \
    }                                                                                        \
  } while (0)
#define G2_PUT_K(step)                                                                       \
  do {                                                                                       \
    _Pragma("unroll") for (int i = 0; i < KC; ++i) {                                         \
      const int p_ = tid + i * NT, key_ = p_ / (DP / 16), c_ = p_ % (DP / 16);               \
      const f16x2 zc_ = as_h2(zkL[(step) & 3][key_]);                                        \
      char* at_ = kL + ((step) & 1) * KB + key_ * KPITCH + c_ * 16;                          \
      *reinterpret_cast<f16x8*>(at_) = key_codes<BITS>(&kw[i][0], zc_);                      \
      *reinterpret_cast<f16x8*>(at_ + DP) = key_codes<BITS>(&kw[i][KW / 2], zc_);            \
    }                                                                                        \
  } while (0)
#define G2_PUT_V(step)                                                                       \
  do {                                                                                       \
    _Pragma("unroll") for (int i = 0; i < VQ; ++i) {                                         \
      const int p_ = tv + i * NT, o_ = (p_ & 7) + 8 * ((p_ >> 4) % OH), ch_ = (p_ >> 4) / OH;\
      const int hf_ = (p_ >> 3) & 1;                                                         \
      if (VP % NT && first_v + i * NT >= VP) break;                                          \
      const f16x4 z_ = *reinterpret_cast<const f16x4*>(                                      \
          &zvL[(step) & 3][16 * (ch_ >> 1) + 4 * (ch_ & 1) + 8 * hf_]);                      \
      const f16x2 z0_ = {z_[0], z_[1]}, z1_ = {z_[2], z_[3]};                                \
      char* at_ = vL + ((step) & 1) * VB + o_ * (8 * VPITCH) +                               \
                  ((ch_ ^ (o_ >> 1 & 7)) << 4) + 8 * hf_;                                    \
      _Pragma("unroll") for (int e = 0; e < 8; ++e) {                                        \
        const f16x2 x_ = value_codes<BITS>(vw[i][0], vw[i][1], e, z0_);                      \
        const f16x2 y_ = value_codes<BITS>(vw[i][2], vw[i][3], e, z1_);                      \
        *reinterpret_cast<f16x4*>(at_ + e * VPITCH) = f16x4{x_[0], x_[1], y_[0], y_[1]};     \
      }                                                                                      \
    }                                                                                        \
  } while (0)
// The workgroup's next step: the codes loaded last go to LDS, the ones after them are loaded.
#define G2_STAGE()             \
  do {                         \
    G2_PUT_K(stage);           \
    G2_PUT_V(stage - 1);       \
    G2_FETCH_K((stage + 1) & 3); \
    G2_FETCH_V(stage & 3);     \
    ++stage;                   \
  } while (0)

    f32x16 x[2];
    f16x8 w[4];
    // Products of a step's keys and the query; element v of block kb: key
    // 32kb + 8(v/4) + 4lh + v%4.  Fragments are read one group of products ahead.
    auto logits = [&](int step) __attribute__((always_inline)) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) x[kb][v] = 0.f;
      const char* kp = kL + (step & 1) * KB + lr * KPITCH + lh * 16;
      f16x8 kf[2][2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
          kf[0][s][kb] = *reinterpret_cast<const f16x8*>(kp + kb * (32 * KPITCH) + s * 32);
#pragma unroll
      for (int g = 0; g < DP / 32; ++g) {
        if (g + 1 < DP / 32) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
              kf[(g + 1) & 1][s][kb] = *reinterpret_cast<const f16x8*>(
                  kp + kb * (32 * KPITCH) + (2 * g + 2 + s) * 32);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            x[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[g & 1][s][kb], qf[2 * g + s],
                                                           x[kb], 0, 0, 0);
      }
    };
    int stage = 1;
    if (steps > 0) {
      if (wave < 2) {  // three steps' pages, then their numbers, under way together
        int page0, page1, page2, page3, page4;
        G2_PAGE(0);
        page0 = page;
        G2_PAGE(1);
        page1 = page;
        G2_PAGE(2);
        page2 = page;
        G2_PAGE(3);
        page3 = page;
        G2_PAGE(4);
        page4 = page;
        page = page0;
        G2_META(0);
        const uint32_t row0 = srow;
        const float sc0 = sc;
        const int sz0 = sz;
        const bool ok0 = sok;
        page = page1;
        G2_META(1);
        const uint32_t row1 = srow;
        const float sc1 = sc;
        const int sz1 = sz;
        const bool ok1 = sok;
        page = page2;
        G2_META(2);
        const uint32_t row2 = srow;
        const float sc2 = sc;
        const int sz2 = sz;
        const bool ok2 = sok;
        page = page3;
        G2_META(3);
        const uint32_t row3 = srow;
        const float sc3 = sc;
        const int sz3 = sz;
        const bool ok3 = sok;
        srow = row0, sc = sc0, sz = sz0, sok = ok0;
        G2_SHOW(0);
        srow = row1, sc = sc1, sz = sz1, sok = ok1;
        G2_SHOW(1);
        srow = row2, sc = sc2, sz = sz2, sok = ok2;
        G2_SHOW(2);
        srow = row3, sc = sc3, sz = sz3, sok = ok3;
        page = page4;
      }
      __syncthreads();
      G2_FETCH_K(0);
      G2_PUT_K(0);
      G2_FETCH_K(1);
      G2_FETCH_V(0);
      __syncthreads();
      // (the logits past the last step are of finite numbers and not used)
      logits(0);
      for (int step = 0; step < steps; ++step) {
        // ---- softmax of the step; whole: every row sees every key ----
        const int at4 = step & 3, j0 = k0 + step * BN;
        const uint64_t ok_l = okL[at4];  // (the same in every lane: into scalar registers)
        const uint64_t ok = (uint64_t)__builtin_amdgcn_readfirstlane((int)(ok_l >> 32)) << 32 |
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)ok_l);
        const float* sk = &skL[at4][4 * lh];
        const float* sv = &svL[at4][4 * lh];
        const bool whole = ok == ~0ull && j0 + BN - 1 <= first_all;
        float mx = m, vx = vmaxL[at4];
        uint32_t see[2] = {~0u, ~0u};  // bit 8q + i of word kb: element 4q + i of block kb
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 s4 = *reinterpret_cast<const f32x4*>(sk + 32 * kb + 8 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[kb][4 * q + i] *= s4[i];
          }
        if (__builtin_expect(whole, 1)) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, x[kb][v]);
        } else {
          const int n = last - j0;  // the last key seen
          const uint64_t any = n < 0 ? 0 : ok;
          const uint64_t seen = any & (~0ull >> (63 - min(max(n, 0), 63)));
          see[0] = (uint32_t)seen >> (4 * lh);
          see[1] = (uint32_t)(seen >> 32) >> (4 * lh);
          vx = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int t = 8 * (v >> 2) + (v & 3);
              const float s1 = sv[32 * kb + t];
              const bool on = see[kb] >> t & 1;
              mx = fmaxf(mx, on ? x[kb][v] : -INFINITY);
              vx = fmaxf(vx, on && s1 < __builtin_inff() ? s1 : 0.f);
            }
        }
        // (m and ref are the same in a row's two lanes)
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx > m || vx >= ref) != 0, 0)) {
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          vx = fmaxf(vx, __shfl_xor(vx, 32));
          const float nref = vx >= ref ? above(vx) : ref;
          float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * C);
          if (m == mx) f = 1.f;
          f = __builtin_amdgcn_ldexpf(f, exponent(ref) - exponent(nref));
          m = mx, ref = nref;
          l *= f;
#pragma unroll
          for (int e = 0; e < DP / 32; ++e)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[e][v] *= f;
        }
        // (opaque: the rare branch stays a branch around, without a second copy of the sums)
        asm volatile("" : "+v"(m), "+v"(ref));
        const float off = (float)(15 - exponent(ref)) - (m == -INFINITY ? 0.f : m * C);
        if (__builtin_expect(whole, 1)) {
          asm volatile("");  // (keeps the branches apart: no selects here)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 s4 = *reinterpret_cast<const f32x4*>(sv + 32 * kb + 8 * q);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][4 * q + i], C, off));
                l += p;
                w[2 * kb + (q >> 1)][4 * (q & 1) + i] = (_Float16)(p * s4[i]);
              }
            }
        } else {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 s4 = *reinterpret_cast<const f32x4*>(sv + 32 * kb + 8 * q);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool on = see[kb] >> (8 * q + i) & 1;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[kb][4 * q + i], C, off));
                l += on ? p : 0.f;
                w[2 * kb + (q >> 1)][4 * (q & 1) + i] = (_Float16)(on ? p * s4[i] : 0.f);
              }
            }
        }
        // ---- the next steps' codes ----
        G2_STAGE();
        if (wave < 2) {
          G2_SHOW((step + 3) & 3);
          G2_META(step + 4);
          G2_PAGE(step + 5);
        }
        __syncthreads();
        // ---- products of this step's values and the next one's keys ----
        __builtin_amdgcn_sched_barrier(0);
        const char* vp = vL + (step & 1) * VB + lr * VPITCH;
        // chunk 2t + lh of row 32e + lr: vc ^ 32(t ^ e % 4)
        const int vc = (lh ^ (lr >> 4)) << 4;
        f16x8 vf[2][DP / 32];
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
          vf[0][e] =
              *reinterpret_cast<const f16x8*>(vp + e * (32 * VPITCH) + (vc ^ (32 * (e & 3))));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (t < 3) {
#pragma unroll
            for (int e = 0; e < DP / 32; ++e)
              vf[(t + 1) & 1][e] = *reinterpret_cast<const f16x8*>(
                  vp + e * (32 * VPITCH) + (vc ^ (32 * ((t + 1) ^ (e & 3)))));
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < DP / 32; ++e)
            acc[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t & 1][e], w[t], acc[e], 0, 0, 0);
        }
        logits(step + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#undef G2_FETCH_K
#undef G2_FETCH_V
#undef G2_PUT_K
#undef G2_PUT_V
#undef G2_STAGE
#undef G2_PAGE
#undef G2_META
#undef G2_SHOW
    if (bad) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);
    l += __shfl_xor(l, 32);
    const float inv = l == 0.f ? 0.f : 512.f / l;
    int r_end = r;
    asm volatile("" : "+v"(r_end));
    if (r_end < rows) {
      const RowAt at = row_at(a, sp, h, r_end);
      const int64_t row = (int64_t)at.token * a.Hq + at.head;
      float* o = a.part + (row * a.split + split) * part_size(a);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = e * 32 + 8 * q + 4 * lh;
          if (!FULL && d >= D) continue;
          const float y[4] = {acc[e][4 * q] * inv, acc[e][4 * q + 1] * inv,
                              acc[e][4 * q + 2] * inv, acc[e][4 * q + 3] * inv};
          if (sh.count > 1)
            *reinterpret_cast<float4*>(o + d) = make_float4(y[0], y[1], y[2], y[3]);
          else
            store_out(a, row * D + d, y);
        }
      if (sh.count > 1 && lh == 0) {
        o[D] = m == -INFINITY ? -INFINITY : m * C;
        o[D + 1] = __builtin_amdgcn_ldexpf(l, exponent(ref) - 15);
      }
    }
    __syncthreads();
  }
}

// Joins the shares of a query row (token, head): LW lanes of four channels each, with the
// shares' weights in LDS; sixteen shares' outputs are under way at a time.  Bound by
// latency (MI355X, one row of 16 shares 4 µs; 2048 rows of up to 8 of 128 channels 5.2 µs,
// 8400 of 64 channels 4.6; with a wave per row those took 5.4 and 8.4).
template <int LW>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a) {
  __shared__ float wL[256 / LW][64];  // (at most 64 shares)
  const int64_t rows_all = (int64_t)a.T * a.Hq;
  const int sub = threadIdx.x % LW, group = threadIdx.x / LW;
  const int64_t first = a.row0 + (int64_t)blockIdx.x * (256 / LW);
  const int64_t row = first + group;
  const int64_t row0 = first + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * (64 / LW);
  if (row0 >= rows_all) return;
  const int64_t near = KvCache::sequence_of_wave(a.cu, a.B, row0 / a.Hq);
  // from here on groups go their own ways
  if (row >= rows_all) return;
  const int t = (int)(row / a.Hq), hq = (int)(row % a.Hq);
  const int b = (int)KvCache::sequence_near(a.cu, a.B, t, near);
  if (b < 0) return;
  Span sp;
  sp.q0 = min(max(a.cu[b], 0), a.T);
  sp.qlen = min(max(a.cu[b + 1], sp.q0), a.T) - sp.q0;
  sp.n = a.c.pages == 0 ? 0 : (int)min<int64_t>(max(a.kv[b], 0), (int64_t)a.width << a.c.shift);
  const int rows = sp.qlen * a.G, h = hq / a.G;
  // which kernel had the row, and in how many shares
  const bool by_rows = a.by_rows && (rows <= kFewRows || !a.by_tiles);
  if (by_rows && rows > kFewRows) return;
  const int split = by_rows ? shares_of(sp.n, a.few_split, a.few_share, 128).count
                            : shares_of(sp.n, a.split, a.share, 64).count;
  if (split == 1) return;
  const int r = (t - sp.q0) * a.G + hq - h * a.G;
  const int64_t pitch = part_size(a);
  const float* p = by_rows
      ? a.few_part + (((int64_t)b * a.c.H + h) * kFewRows + r) * a.few_split * pitch
      : a.part + row * a.split * pitch;
  const int D = (int)a.c.D, d = sub * 4;
  const float* pd = p + (d < D ? d : 0);
  float4 o[2][8];
  // (before the weights are known)
#pragma unroll
  for (int s = 0; s < 8; ++s)
    o[0][s] = *reinterpret_cast<const float4*>(pd + min(s, split - 1) * pitch);
  // a share without keys has a maximum of -inf and adds nothing, unless its sum is NaN
  constexpr int J = 64 / LW;
  float m[J], w[J], M = -INFINITY, L = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int s = sub + j * LW;
    m[j] = -INFINITY, w[j] = 0.f;
    if (s < split) m[j] = p[s * pitch + D], w[j] = p[s * pitch + D + 1];
    M = fmaxf(M, m[j]);
  }
#pragma unroll
  for (int k = LW / 2; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (m[j] != -INFINITY) w[j] *= __builtin_amdgcn_exp2f(m[j] - M);
    L += w[j];
    wL[group][sub + j * LW] = m[j] == -INFINITY ? 0.f : w[j];
  }
#pragma unroll
  for (int k = LW / 2; k > 0; k >>= 1) L += __shfl_xor(L, k);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  float y[4] = {0, 0, 0, 0};
  for (int s0 = 0; s0 < split; s0 += 16) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = s0 + 8 * half;
      if (at + 8 < split) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          o[half ^ 1][s] =
              *reinterpret_cast<const float4*>(pd + min(at + 8 + s, split - 1) * pitch);
      }
      if (at >= split) break;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float ws = wL[group][at + s];  // (zero past the last share)
        if (ws != 0.f) {                     // (also where it is NaN)
          y[0] += ws * o[half][s].x, y[1] += ws * o[half][s].y;
          y[2] += ws * o[half][s].z, y[3] += ws * o[half][s].w;
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] *= inv;
  if (d < D) store_out(a, row * D + d, y);
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
constexpr int64_t kCUs = 256;

struct Plan {
  bool few, tiles;     // which kernels run
  int64_t ntiles, split, few_split, share, few_share;
  int64_t part, few_part;  // bytes of partial results
  Plan(int64_t T, int64_t Hq, int64_t H, int64_t D, int64_t B, int64_t max_q, int64_t max_kv) {
    const int64_t G = Hq / H, rows = max_q * G, pairs = std::max<int64_t>(1, B * H);
    tiles = rows > kFewRows;
    // a batch of chunks only has sequences of few rows if some are shorter than the rest
    few = !tiles || B > 1;
    const int64_t keys = std::min<int64_t>(std::max<int64_t>(1, max_kv), 1 << 30);
    // Few rows: shares of 1024 keys or more, up to sixteen workgroups per CU (sequences of a
    // batch differ in length, and the last ones to run should be short); smaller ones, from
    // 256 keys (two steps of every wave), for six per CU.  MI355X, heads 32 on 8 of 128:
    //   64 uneven sequences of up to 8192 keys, 4 bits: 72 µs in 8, 76 in 3, 91 unshared
    //   96 of them: 111 µs in 6 shares, 131 in 2
    //   16 uneven of up to 8192, 4 bits: 32 µs in 12, 36 in 4, 53 in 32
    //   one of 8192, 8 bits: 13.1 µs in shares of 256, 16.1 of 128, 14.1 of 512
    // None where two workgroups per CU are there without and short: 64 uneven sequences of up
    // to 4096 keys 55 µs, 57 in 4; 160 of up to 2048, 68 µs and 89 in 2.  At most 32: 8
    // sequences of 16384, two heads, 21 µs in 32 and 26 in 64, whose joining costs more; up
    // to 64 for a few heads, which are not enough otherwise.
    int64_t want = std::max(std::min(cdiv(16 * kCUs, pairs), keys / 1024),
                            std::min(cdiv(6 * kCUs, pairs), cdiv(keys, 256)));
    if (pairs >= 2 * kCUs && keys < 5120) want = 1;
    want = std::min<int64_t>(want, pairs > 4 ? 32 : 64);
    few_share = cdiv(cdiv(keys, want), 128) * 128;
    few_split = cdiv(keys, few_share);
    // 128 rows a workgroup, two workgroups to a CU.  (256 rows, one to a CU: MI355X, 2048
    // tokens over 16384 keys 714 against 702 µs, six uneven chunks 44 against 35 µs; 64 rows:
    // 1211 against 671 µs, and where that is all there are, 8 tokens of four heads over 4096
    // keys, 23.4 against 20.9.)
    // As many tiles as the largest sequence may have, unless the launch gets too large (many
    // sequences whose sizes are not given): workgroups then take further tiles in turn.
    ntiles = std::max<int64_t>(1, std::min(cdiv(rows, kTileRows), kMaxGroups / pairs));
    // Shares for two workgroups per CU, three in a batch (its sequences differ in length).
    // MI355X, heads 32 on 8 of 128, two / three / four: 512 tokens over 2048 keys 53.7 / 62.9
    // / 66.6 µs; four chunks of 300 over up to 4096 keys 158 / 116 / 123 µs; six of 100, 100 /
    // 71 / 84 µs.  Of 256 keys or more: 8 chunks of 16 tokens over 2048 keys 33 µs, 40 with 512.
    split = std::max<int64_t>(1, std::min((B > 1 ? 3 : 2) * kCUs / (pairs * ntiles), keys / 256));
    split = std::min<int64_t>(split, 32);
    // Every token has its partial results, also where more tokens than stated came: at most a
    // GiB of them (sizes stated right need a sixth of that at most).
    const int64_t one = T * Hq * (D + 4) * 4;
    split = std::min(split, std::max<int64_t>(1, (1 << 30) / std::max<int64_t>(1, one)));
    share = cdiv(cdiv(keys, split), 64) * 64;
    part = tiles && split > 1 ? cdiv(T * Hq * split * (D + 4) * 4, 256) * 256 : 0;
    few_part = few && few_split > 1
                   ? cdiv(B * H * kFewRows * few_split * (D + 4) * 4, 256) * 256 : 0;
  }
};

template <int BITS, int DP, bool FULL>
int launch(hipStream_t st, const AttnArgs& a, const Plan& p) {
  if (p.few) {
    hipLaunchKernelGGL((attend_rows_kernel<BITS, DP, FULL>),
                       dim3((unsigned)p.few_split, (unsigned)a.c.H, (unsigned)a.B + 1), dim3(256),
                       0, st, a);
    G2PTQ_LAUNCHED();
  }
  if (p.tiles) {
    hipLaunchKernelGGL((attend_tiles_kernel<BITS, DP, FULL>),
                       dim3((unsigned)(a.B * a.c.H * a.split * a.tiles + 1)), dim3(2 * kTileRows),
                       0, st, a);
    G2PTQ_LAUNCHED();
  }
  if (a.part || a.few_part) {
    constexpr int LW = DP / 4;
    const int64_t groups = cdiv((int64_t)a.T * a.Hq, 256 / LW);
    for (int64_t g = 0; g < groups; g += kMaxGroups) {
      AttnArgs part = a;
      part.row0 = g * (256 / LW);
      hipLaunchKernelGGL((attend_join_kernel<LW>), dim3((unsigned)std::min(groups - g, kMaxGroups)),
                         dim3(256), 0, st, part);
      G2PTQ_LAUNCHED();
    }
  }
  return G2PTQ_OK;
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_paged_attention_workspace(int64_t T, int64_t Hq, int64_t kv_heads, int64_t dim,
                                               int64_t B, int64_t max_q, int64_t max_kv,
                                               size_t* bytes) {
  G2PTQ_CHECK(bytes && T >= 0 && Hq >= 1 && kv_heads >= 1 && Hq % kv_heads == 0 && dim >= 16 &&
                  B >= 0 && max_q >= 0 && max_kv >= 0,
              "paged_attention_workspace: bad sizes");
  const Plan p(T, Hq, kv_heads, dim, B, max_q, max_kv);
  *bytes = (size_t)(p.part + p.few_part);
  return G2PTQ_OK;
}

extern "C" int g2ptq_paged_attention(void* stream, const g2ptq_kv_cache* cache, const void* q,
                                     int64_t q_token, int64_t q_head, int dtype, int64_t T,
                                     int64_t Hq, const int32_t* table, int64_t ldt, int64_t B,
                                     int64_t width, const int32_t* cu_q, const int32_t* kv_lens,
                                     int64_t max_q, int64_t max_kv, float scale, void* out,
                                     void* ws, size_t ws_bytes) {
  AttnArgs a;
  G2PTQ_TRY(check_cache("paged_attention", cache, a.c));
  G2PTQ_CHECK(dtype == 0 || dtype == 1, "paged_attention: dtype code %d (bf16 or fp16)", dtype);
  G2PTQ_CHECK(Hq >= 1 && Hq <= 65535 && Hq % a.c.H == 0,
              "paged_attention: %lld query heads over %lld heads of the cache", (long long)Hq,
              (long long)a.c.H);
  G2PTQ_CHECK(T >= 0 && T * Hq < (1ll << 31), "paged_attention: %lld tokens of %lld heads",
              (long long)T, (long long)Hq);
  G2PTQ_CHECK(B >= 0 && B < 65535 && width >= 0 && width < (1ll << 31) && ldt >= width &&
                  max_q >= 0 && max_q <= T && max_kv >= 0,
              "paged_attention: bad page table or sizes");
  if (T == 0) return G2PTQ_OK;
  G2PTQ_CHECK(width << a.c.shift <= 1ll << 30,
              "paged_attention: sequences of up to %lld keys (at most 2^30)",
              (long long)(width << a.c.shift));
  G2PTQ_CHECK(q && out && (B == 0 || (cu_q && kv_lens)) && (table || B * width == 0),
              "paged_attention: null pointer");
  G2PTQ_CHECK((reinterpret_cast<uintptr_t>(out) & 15) == 0,
              "paged_attention: output not 16-byte aligned");
  const Plan p(T, Hq, a.c.H, a.c.D, B, max_q, max_kv);
  G2PTQ_CHECK(!p.tiles || B * a.c.H * p.split * p.ntiles <= kMaxGroups,
              "paged_attention: %lld sequences of %lld heads (at most %lld in all)", (long long)B,
              (long long)a.c.H, (long long)kMaxGroups);
  const size_t need = (size_t)(p.part + p.few_part);
  if (need && (!ws || ws_bytes < need)) {
    set_error("paged_attention: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return G2PTQ_ERR_WORKSPACE;
  }
  G2PTQ_CHECK(!need || (reinterpret_cast<uintptr_t>(ws) & 15) == 0,
              "paged_attention: workspace not 16-byte aligned");
  a.q = q, a.qt = q_token, a.qh = q_head, a.out = out, a.ldt = ldt;
  a.table = table, a.cu = cu_q, a.kv = kv_lens;
  a.T = (int)T, a.Hq = (int)Hq, a.B = (int)B, a.G = (int)(Hq / a.c.H), a.width = (int)width;
  a.dtype = dtype;
  a.vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_token % 8 == 0 && q_head % 8 == 0;
  a.scale = scale, a.kscale = fabsf(scale) * 1.44269504088896340736f * 0x1p-6f;
  a.tiles = (int)p.ntiles, a.split = (int)p.split, a.few_split = (int)p.few_split;
  a.share = (int)p.share, a.few_share = (int)p.few_share;
  a.by_rows = p.few, a.by_tiles = p.tiles;
  a.part = p.part ? static_cast<float*>(ws) : nullptr;
  a.few_part = p.few_part ? reinterpret_cast<float*>(static_cast<char*>(ws) + p.part) : nullptr;
  hipStream_t st = as_stream(stream);
  const int64_t D = a.c.D;
#define G2_DIM(BITS)                                                                         \
  if (D == 64) return launch<BITS, 64, true>(st, a, p);                                      \
  if (D < 64) return launch<BITS, 64, false>(st, a, p);                                      \
  if (D == 128) return launch<BITS, 128, true>(st, a, p);                                    \
  if (D < 128) return launch<BITS, 128, false>(st, a, p);                                    \
  return launch<BITS, 256, false>(st, a, p)
  if (a.c.bits == 8) { G2_DIM(8); }
  G2_DIM(4);
#undef G2_DIM
}
