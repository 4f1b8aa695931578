// Causal attention of ragged chunks of new tokens over the paged cache.
//
//   o[i] = Σ_j p_ij·v̂_j / Σ_j p_ij,   p_ij = exp(c·q_i·k̂_j − max_j(c·q_i·k̂_j))
//
// over the keys j ≤ p_i of the query's sequence, p_i = kv_len − q_len + i the
// position of its i-th new token.  k̂ = s(u − z) and v̂ are what the cache holds
// (kvcache.hip).  A query without keys (kv_len < q_len) gets zeros.
#include <algorithm>

#include "grid8.hpp"
#include "kvcache.hpp"

namespace g2ptq {
namespace {

struct AttnArgs {
  KvCache c;
  const void* q;
  int64_t qt, qh;  // strides of query token and head
  void* out;       // T × Hq × D, contiguous
  int64_t T, Hq, B, ldt, width;
  const int32_t *table, *cu, *kv;
  float scale;
};

// One wave per (query token, head): lanes share a block of 64 keys for the
// products with the query, then the head's channels for the products with the
// values.
template <int DT>
__global__ __launch_bounds__(64) void attention_simple_kernel(AttnArgs a) {
  __shared__ float qs[256], ps[64];
  const int64_t t = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq;
  const int lane = threadIdx.x, D = (int)a.c.D;
  const int64_t h = hq / (a.Hq / a.c.H);
  const int64_t b = KvCache::sequence(a.cu, a.B, t);
  int64_t last = -1;  // the last key that the query sees
  if (b >= 0) last = (int64_t)a.kv[b] - (a.cu[b + 1] - t);
  const int half = 1 << (a.c.bits - 1), per = a.c.bits == 8 ? 1 : 2;
  for (int d = lane * 8; d < D; d += 512) {
    float v[8];
    load8<DT>(a.q, t * a.qt + hq * a.qh + d, false, 8, v);
    for (int i = 0; i < 8; ++i) qs[d + i] = v[i];
  }
  __syncthreads();
  float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.f;
  int bad = 0;
  const int32_t* table = a.table + (b < 0 ? 0 : b) * a.ldt;
  for (int64_t j0 = 0; j0 <= last; j0 += 64) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    int64_t at = -1;
    if (j <= last) {
      const int64_t slot = a.c.slot(table, a.width, j);
      if (slot >= 0) {
        at = a.c.row(slot, h);
        const uint8_t* k = a.c.codes[0] + at * (D / per);
        const int z = a.c.zero[0] ? a.c.zero[0][at] : half;
        float x = 0.f;
        for (int d = 0; d < D; ++d) {
          const int u = per == 1 ? k[d] : (k[d >> 1] >> (4 * (d & 1))) & 15;
          x += qs[d] * (float)(u - z);
        }
        s = x * a.c.scale[0][at] * a.scale;
      } else {
        bad = 1;
      }
    }
    float mj = s;
    for (int w = 32; w > 0; w >>= 1) mj = fmaxf(mj, __shfl_xor(mj, w));
    const float mn = fmaxf(m, mj);
    const float shift = mn == -INFINITY ? 0.f : mn;
    const float p = at >= 0 ? expf(s - shift) : 0.f, alpha = expf(m - shift);
    m = mn;
    float pl = p;
    for (int w = 32; w > 0; w >>= 1) pl += __shfl_xor(pl, w);
    l = l * alpha + pl;
    for (int r = 0; r < 4; ++r) o[r] *= alpha;
    const float pv = at >= 0 ? p * a.c.scale[1][at] : 0.f;
    for (int i = 0; i < 64; ++i) {
      const int64_t ai = __shfl(at, i);
      const float pi = __shfl(pv, i);
      if (ai < 0) continue;
      const uint8_t* v = a.c.codes[1] + ai * (D / per);
      const int z = a.c.zero[1] ? a.c.zero[1][ai] : half;
      for (int r = 0; r < 4; ++r) {
        const int d = lane + 64 * r;
        if (d >= D) break;
        const int u = per == 1 ? v[d] : (v[d >> 1] >> (4 * (d & 1))) & 15;
        o[r] += pi * (float)(u - z);
      }
    }
  }
  if (__any(bad) && lane == 0) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);
  for (int r = 0; r < 4; ++r) {
    const int d = lane + 64 * r;
    if (d >= D) break;
    const float y = l == 0.f ? 0.f : o[r] / l;
    const int64_t e = (t * a.Hq + hq) * D + d;
    if (DT == 0) static_cast<uint16_t*>(a.out)[e] = __builtin_bit_cast(uint16_t, (__bf16)y);
    else static_cast<_Float16*>(a.out)[e] = (_Float16)y;
  }
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
  *bytes = 0;
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
  G2PTQ_CHECK(B >= 0 && B <= 65535 && width >= 0 && ldt >= width && max_q >= 0 && max_kv >= 0,
              "paged_attention: bad page table");
  if (T == 0) return G2PTQ_OK;
  G2PTQ_CHECK(q && out && (B == 0 || (cu_q && kv_lens)) && (table || B * width == 0),
              "paged_attention: null pointer");
  a.q = q, a.qt = q_token, a.qh = q_head, a.out = out, a.T = T, a.Hq = Hq, a.B = B, a.ldt = ldt;
  a.width = width, a.table = table, a.cu = cu_q, a.kv = kv_lens, a.scale = scale;
  const dim3 grid((unsigned)(T * Hq));
  if (dtype == 0)
    hipLaunchKernelGGL(attention_simple_kernel<0>, grid, dim3(64), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(attention_simple_kernel<1>, grid, dim3(64), 0, as_stream(stream), a);
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}
