// Rotary positions of queries and keys.
//
//   pair i of a head, at position p:  (a, b) → m·(a·cos φ − b·sin φ, a·sin φ + b·cos φ),
//   φ = 2π·p·f_i,  f_i in turns per position
//   pairs are channels (i, i + n/2) or (2i, 2i + 1) of the first n; the others stay
//
// p·f_i is a product of 64 bits, of which whole turns are dropped exactly: a position of 2^31
// keeps 24 bits of a turn and more, where fp32 has none.  The angle's sine and cosine and the
// products are fp32, a result is rounded once to its type.
#include <algorithm>

#include "grid8.hpp"

namespace g2ptq {
namespace {

constexpr int kAngles = 1024;  // pairs of a workgroup's tokens
constexpr int kMaxTokens = 8;

struct RotaryArgs {
  const void* x[2];       // queries, keys
  int64_t st[2], sh[2];   // strides of token and head (elements)
  int heads[2];
  void* out[2];           // T × heads × dim
  int64_t T, first;       // tokens, and the launch's first
  int dim, n;
  const int64_t* positions;
  const double* freq;     // n / 2, turns a position
  float factor;
  int tokens;             // of a workgroup
};

// A workgroup takes `tokens` tokens: the sines and cosines of their pairs first, once for all
// heads, then pieces of eight pairs (half layout: sixteen channels) or eight channels.  Bound by
// the bytes: MI355X, 16384 tokens of 32 + 8 heads of 128, bf16, 66.6 µs (336 MB, 5.0 TB/s); one
// token 3.1–3.4 µs, a launch and the latencies of position, angle and channels.
template <int DT, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  __shared__ float cosL[kAngles], sinL[kAngles];
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.tokens;
  const int count = (int)min<int64_t>(a.tokens, a.T - t0);
  const int pairs = a.n / 2;
  for (int i = threadIdx.x; i < count * pairs; i += 256) {
    const int t = i / pairs, j = i - t * pairs;
    double turn = (double)a.positions[t0 + t] * a.freq[j];
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * (float)turn, &s, &c);
    cosL[i] = c * a.factor, sinL[i] = s * a.factor;
  }
  __syncthreads();
  const uint32_t turned = (uint32_t)(HALF ? (pairs + 7) / 8 : (a.n + 7) / 8);
  const uint32_t P = turned + (uint32_t)(a.dim - a.n + 7) / 8, H = a.heads[0] + a.heads[1];
  // item = (token t, head h, piece p), counted on by 256 in mixed radix
  const uint32_t q256 = 256 / P, dp = 256 - q256 * P, dt = q256 / H, dh = q256 - dt * H;
  const uint32_t q = threadIdx.x / P;
  uint32_t p = threadIdx.x - q * P, t = q / H, h = q - t * H;
  while (t < (uint32_t)count) {
    const int w = h >= (uint32_t)a.heads[0];
    const uint32_t hw = w ? h - a.heads[0] : h;
    const int64_t in = (t0 + t) * a.st[w] + hw * a.sh[w];
    const int64_t out = ((t0 + t) * a.heads[w] + hw) * a.dim;
    if (p < turned) {
      const float* cs = cosL + t * pairs;
      const float* sn = sinL + t * pairs;
      if constexpr (HALF) {
        const int j = p * 8, n = pairs - j;
        float u[8], v[8], x[8], y[8];
        load8_any<DT>(a.x[w], in + j, n, u);
        load8_any<DT>(a.x[w], in + j + pairs, n, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = i < n ? j + i : 0;
          x[i] = u[i] * cs[k] - v[i] * sn[k];
          y[i] = u[i] * sn[k] + v[i] * cs[k];
        }
        store8_any<DT>(a.out[w], out + j, n, x);
        store8_any<DT>(a.out[w], out + j + pairs, n, y);
      } else {
        const int j = p * 8, n = a.n - j;
        float u[8], x[8];
        load8_any<DT>(a.x[w], in + j, n, u);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int k = i < n ? (j + i) / 2 : 0;
          x[i] = u[i] * cs[k] - u[i + 1] * sn[k];
          x[i + 1] = u[i] * sn[k] + u[i + 1] * cs[k];
        }
        store8_any<DT>(a.out[w], out + j, n, x);
      }
    } else {
      const int j = a.n + (p - turned) * 8, n = a.dim - j;
      float u[8];
      load8_any<DT>(a.x[w], in + j, n, u);
      store8_any<DT>(a.out[w], out + j, n, u);
    }
    p += dp, h += dh, t += dt;
    if (p >= P) p -= P, ++h;
    if (h >= H) h -= H, ++t;
  }
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_rotary(void* stream, const void* q, int64_t q_token, int64_t q_head,
                            int64_t q_heads, const void* k, int64_t k_token, int64_t k_head,
                            int64_t k_heads, int dtype, int64_t T, int64_t dim, int64_t n,
                            int interleaved, const int64_t* positions, const double* freq,
                            float factor, void* q_out, void* k_out) {
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2, "rotary: dtype code %d", dtype);
  G2PTQ_CHECK(dim >= 2 && dim <= 1024 && n >= 2 && n <= dim && n % 2 == 0,
              "rotary: %lld of %lld channels turned (an even number, of at most 1024)",
              (long long)n, (long long)dim);
  G2PTQ_CHECK(q_heads >= 0 && k_heads >= 0 && q_heads <= 65535 && k_heads <= 65535,
              "rotary: %lld and %lld heads", (long long)q_heads, (long long)k_heads);
  G2PTQ_CHECK(T >= 0, "rotary: %lld tokens", (long long)T);
  if (T == 0 || q_heads + k_heads == 0) return G2PTQ_OK;
  G2PTQ_CHECK(positions && freq && (q_heads == 0 || (q && q_out)) &&
                  (k_heads == 0 || (k && k_out)), "rotary: null pointer");
  RotaryArgs a;
  a.x[0] = q, a.st[0] = q_token, a.sh[0] = q_head, a.heads[0] = (int)q_heads, a.out[0] = q_out;
  a.x[1] = k, a.st[1] = k_token, a.sh[1] = k_head, a.heads[1] = (int)k_heads, a.out[1] = k_out;
  a.T = T, a.dim = (int)dim, a.n = (int)n;
  a.positions = positions, a.freq = freq, a.factor = factor;
  // As many tokens as a workgroup has threads for, mostly one.  MI355X, one token of 40 heads
  // against eight: 16384 × 128 channels 66.7 and 67.7 µs, 2048 × 64 channels of which 32 turn 7.4
  // and 8.4; sixteen 82.8 at the first.
  const int64_t pieces = (interleaved ? cdiv(n, 8) : cdiv(n, 16)) + cdiv(dim - n, 8);
  const int64_t tokens = std::max<int64_t>(
      1, std::min<int64_t>(std::min<int64_t>(kMaxTokens, kAngles / (n / 2)),
                           256 / (pieces * (q_heads + k_heads))));
  a.tokens = (int)tokens;
  hipStream_t st = as_stream(stream);
  for (a.first = 0; a.first < T; a.first += kMaxGroups * tokens) {
    const dim3 grid((unsigned)std::min(cdiv(T - a.first, tokens), kMaxGroups));
#define G2_ROT(DT)                                                                             \
  do {                                                                                         \
    if (interleaved)                                                                           \
      hipLaunchKernelGGL((rotary_kernel<DT, false>), grid, dim3(256), 0, st, a);               \
    else                                                                                       \
      hipLaunchKernelGGL((rotary_kernel<DT, true>), grid, dim3(256), 0, st, a);                \
  } while (0)
    if (dtype == 0) G2_ROT(0);
    else if (dtype == 1) G2_ROT(1);
    else G2_ROT(2);
#undef G2_ROT
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}
