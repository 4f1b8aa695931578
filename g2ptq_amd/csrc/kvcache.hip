// Paged cache of quantized keys and values: writing and reading back.
//
// Layout (pages of `page` slots, H heads of D channels, b bits; keys and values
// apart):
//   codes  [pages][H][page][D·b/8] bytes: unsigned codes q + 2^(b−1), at 4 bits
//          two channels a byte, the first in the low half
//   scale  [pages][H][page] fp32
//   zero   [pages][H][page] bytes: z + 2^(b−1) (asymmetric grid only)
// A code u of a slot stands for scale·(u − zero), zero = 2^(b−1) in the
// symmetric grid.  A sequence's token p lives in slot p % page of page
// table[p / page].
#include <algorithm>

#include "grid8.hpp"
#include "kvcache.hpp"

namespace g2ptq {
namespace {

struct WriteArgs {
  const void* x[2];        // keys, values: T × H × D, channels contiguous
  int64_t st[2], sh[2];    // strides of token and head (elements)
  const int64_t* slots;    // page·(page size) + offset; negative: not written
  uint32_t items, first;   // T·H, and the launch's first of them
  KvCache c;
  bool vec[2];
};

// L lanes hold one token's head, sixteen channels each (lanes past D idle), and reduce
// it among themselves; a workgroup takes 256 / L consecutive heads of the T × H.  Sixteen
// channels are the largest store of a lane at 8 bits and leave few lanes to reduce over.
// A wave loads, then computes, then stores, once.  At 8 bits its waves wait for memory seven
// tenths of the time; at 4 bits asymmetric they execute 22 vector instructions a value (18 at
// 8 bits; range, corrected product, code, packing), 9 µs of the whole by themselves.  MI355X,
// 8192 tokens of 8 × 128 bf16, 8 bits 15–22 µs (bytes 10), 4 bits asymmetric 11–13 µs (bytes
// 8.3); 32 tokens 3.4 µs, a launch's latency.
// grid.y: 0 keys, 1 values.
template <int DT, bool SYM, int BITS, int L>
__global__ __launch_bounds__(256) void kv_write_kernel(WriteArgs a) {
  constexpr int OFF = 1 << (BITS - 1);
  const int w = blockIdx.y;
  const uint32_t item = a.first + blockIdx.x * (256 / L) + threadIdx.x / L;
  const int d = (threadIdx.x % L) * 16;
  if (item >= a.items) return;
  const uint32_t t = item / (uint32_t)a.c.H, h = item - t * (uint32_t)a.c.H;
  const int64_t slot = a.slots[t];
  const bool on = d < a.c.D;
  float v[2][8] = {};
  if (on) {
    const int64_t at = t * a.st[w] + h * a.sh[w] + d;
    load8<DT>(a.x[w], at, a.vec[w], 8, v[0]);
    load8<DT>(a.x[w], at + 8, a.vec[w], 8, v[1]);
  }
  if (slot < 0) return;
  if (slot >= a.c.pages << a.c.shift) {
    if (d == 0) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);
    return;
  }
  Range<SYM> r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r.add(v[i >> 3][i & 7]);
  reduce_range<L>(r);
  const Grid g = make_grid<SYM>(r, BITS);
  const int64_t at = a.c.row(slot, h);
  if (d == 0) {
    a.c.scale[w][at] = g.s;
    if (!SYM) a.c.zero[w][at] = (uint8_t)((int)g.z + OFF);
  }
  if (!on) return;
  uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t u = (uint32_t)(to_code(g, v[i >> 3][i & 7]) + OFF);
    if constexpr (BITS == 8) o[i >> 2] |= u << (8 * (i & 3));
    else o[i >> 3] |= u << (4 * (i & 7));
  }
  if constexpr (BITS == 8)
    *reinterpret_cast<uint4*>(a.c.codes[w] + at * a.c.D + d) = make_uint4(o[0], o[1], o[2], o[3]);
  else
    *reinterpret_cast<uint2*>(a.c.codes[w] + at * (a.c.D / 2) + d / 2) = make_uint2(o[0], o[1]);
}

struct ReadArgs {
  KvCache c;
  const int32_t* table;
  int64_t ldt, B, width;
  const int32_t* cu;  // B + 1 offsets of the sequences in the output
  int64_t total, first;  // rows, and the launch's first of them
  void* out[2];       // total × H × D
  int tokens;         // of a workgroup, at most kReadTokens
};

constexpr int kReadTokens = 64;

// A workgroup takes `tokens` consecutive output rows: their slots first (one thread each),
// then their pieces of 16 channels, consecutive threads consecutive pieces.  Output rows
// outside every sequence, and tokens whose page is not in the cache, are zero.  Bound by
// the bytes: MI355X, 131072 tokens of 8 × 128, 8 bits to bf16, 177 µs (4.6 TB/s); 8192 at 4
// bits 10.5–12 µs (3.5–4 TB/s); 512 tokens 4 µs, the latency of offset, page, scale and code.
template <int DT, int BITS>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
  __shared__ int64_t slotL[kReadTokens];
  const int w = blockIdx.y;
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.tokens;
  const int n = (int)min<int64_t>(a.tokens, a.total - t0);
  if (threadIdx.x < 64) {  // (one wave: n <= 64)
    const int64_t b = KvCache::sequence_of_wave(a.cu, a.B, t0);
    if ((int)threadIdx.x < n) {
      const int64_t slot = a.c.find(a.table, a.ldt, a.width, a.cu, a.B, t0 + threadIdx.x, b);
      if (slot == -2) atomicOr(a.c.flags, G2PTQ_FLAG_BAD_INDEX);
      slotL[threadIdx.x] = slot;
    }
  }
  __syncthreads();
  // piece = (token t, head h, 16 channels c), counted on by 256 in mixed radix
  const uint32_t C = (uint32_t)a.c.D / 16, H = (uint32_t)a.c.H, rest = 256 / C;
  const uint32_t dc = 256 - rest * C, dt = rest / H, dh = rest - dt * H;
  uint32_t q = threadIdx.x / C, c = threadIdx.x - q * C, t = q / H, h = q - t * H;
  const int64_t base = t0 * H * C;
  for (uint32_t piece = threadIdx.x; t < (uint32_t)n; piece += 256) {
    const int64_t slot = slotL[t];
    float lo[8] = {0, 0, 0, 0, 0, 0, 0, 0}, hi[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (slot >= 0) {
      const int64_t at = a.c.row(slot, h);
      const float s = a.c.scale[w][at];
      const int z = a.c.zero[w] ? a.c.zero[w][at] : 1 << (BITS - 1);
      uint32_t u[4];
      if constexpr (BITS == 8) {
        const uint4 o = *reinterpret_cast<const uint4*>(a.c.codes[w] + at * a.c.D + c * 16);
        u[0] = o.x, u[1] = o.y, u[2] = o.z, u[3] = o.w;
      } else {
        const uint2 o = *reinterpret_cast<const uint2*>(a.c.codes[w] + at * (a.c.D / 2) + c * 8);
        u[0] = o.x, u[1] = o.y, u[2] = u[3] = 0;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (BITS == 8) {
          lo[i] = s * (float)((int)(u[i >> 2] >> (8 * (i & 3)) & 0xffu) - z);
          hi[i] = s * (float)((int)(u[2 + (i >> 2)] >> (8 * (i & 3)) & 0xffu) - z);
        } else {
          lo[i] = s * (float)((int)(u[0] >> (4 * i) & 15u) - z);
          hi[i] = s * (float)((int)(u[1] >> (4 * i) & 15u) - z);
        }
      }
    }
    store8<DT>(a.out[w], (base + piece) * 16, true, 8, lo);
    store8<DT>(a.out[w], (base + piece) * 16 + 8, true, 8, hi);
    c += dc, h += dh, t += dt;
    if (c >= C) c -= C, ++h;
    if (h >= H) h -= H, ++t;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename F>
int by_lanes(int64_t D, F f) {
  if (D <= 16) return f(std::integral_constant<int, 1>());
  if (D <= 32) return f(std::integral_constant<int, 2>());
  if (D <= 64) return f(std::integral_constant<int, 4>());
  if (D <= 128) return f(std::integral_constant<int, 8>());
  return f(std::integral_constant<int, 16>());
}

}  // namespace

int check_cache(const char* who, const g2ptq_kv_cache* c, KvCache& k) {
  G2PTQ_CHECK(c, "%s: null cache", who);
  G2PTQ_CHECK(c->bits == 4 || c->bits == 8, "%s: %d bits (4 or 8)", who, c->bits);
  G2PTQ_CHECK(c->pages >= 0 && c->pages < (1ll << 31) && c->heads >= 1 && c->heads <= 65535,
              "%s: %lld pages of %lld heads", who, (long long)c->pages, (long long)c->heads);
  G2PTQ_CHECK(c->dim >= 16 && c->dim <= 256 && c->dim % 16 == 0,
              "%s: head dimension %lld (a multiple of 16 up to 256)", who, (long long)c->dim);
  G2PTQ_CHECK(c->page >= 1 && c->page <= 4096 && (c->page & (c->page - 1)) == 0,
              "%s: pages of %lld slots (a power of two up to 4096)", who, (long long)c->page);
  G2PTQ_CHECK(c->pages * c->heads * c->page < (1ll << 31),
              "%s: %lld pages of %lld heads of %lld slots (fewer than 2^31 in all)", who,
              (long long)c->pages, (long long)c->heads, (long long)c->page);
  G2PTQ_CHECK(c->flags, "%s: null flags", who);
  G2PTQ_CHECK(c->pages == 0 || (c->k_codes && c->v_codes && c->k_scale && c->v_scale),
              "%s: null cache buffer", who);
  G2PTQ_CHECK(aligned16(c->k_codes) && aligned16(c->v_codes),
              "%s: codes not 16-byte aligned", who);
  G2PTQ_CHECK(c->sym || c->pages == 0 || (c->k_zero && c->v_zero), "%s: null zero points", who);
  k.codes[0] = c->k_codes, k.codes[1] = c->v_codes;
  k.scale[0] = c->k_scale, k.scale[1] = c->v_scale;
  k.zero[0] = c->sym ? nullptr : c->k_zero, k.zero[1] = c->sym ? nullptr : c->v_zero;
  k.pages = c->pages, k.H = c->heads, k.D = c->dim;
  k.shift = __builtin_ctzll((unsigned long long)c->page);
  k.bits = c->bits;
  k.flags = c->flags;
  return G2PTQ_OK;
}

}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_kv_write(void* stream, const g2ptq_kv_cache* cache, const void* k,
                              int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                              int64_t v_head, int dtype, int64_t T, const int64_t* slots) {
  WriteArgs a;
  G2PTQ_TRY(check_cache("kv_write", cache, a.c));
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2, "kv_write: dtype code %d", dtype);
  G2PTQ_CHECK(T >= 0 && T * a.c.H < (1ll << 31), "kv_write: %lld tokens of %lld heads",
              (long long)T, (long long)a.c.H);
  if (T == 0) return G2PTQ_OK;
  G2PTQ_CHECK(k && v && slots, "kv_write: null pointer");
  const int e = dtype == 2 ? 4 : 2;
  a.x[0] = k, a.x[1] = v;
  a.st[0] = k_token, a.sh[0] = k_head, a.st[1] = v_token, a.sh[1] = v_head;
  a.vec[0] = aligned16(k) && k_token * e % 16 == 0 && k_head * e % 16 == 0;
  a.vec[1] = aligned16(v) && v_token * e % 16 == 0 && v_head * e % 16 == 0;
  a.slots = slots;
  a.items = (uint32_t)(T * a.c.H);
  hipStream_t st = as_stream(stream);
  const bool sym = cache->sym != 0;
  return by_lanes(a.c.D, [&](auto lanes) -> int {
    constexpr int L = decltype(lanes)::value;
#define G2_WR(DT, SYM)                                                                      \
  do {                                                                                      \
    if (a.c.bits == 8)                                                                      \
      hipLaunchKernelGGL((kv_write_kernel<DT, SYM, 8, L>), grid, dim3(256), 0, st, a);      \
    else                                                                                    \
      hipLaunchKernelGGL((kv_write_kernel<DT, SYM, 4, L>), grid, dim3(256), 0, st, a);      \
  } while (0)
    for (int64_t first = 0; first < a.items; first += kMaxGroups * (256 / L)) {
      a.first = (uint32_t)first;
      const dim3 grid((unsigned)std::min(cdiv(a.items - first, 256 / L), kMaxGroups), 2);
      if (dtype == 0) { if (sym) G2_WR(0, true); else G2_WR(0, false); }
      else if (dtype == 1) { if (sym) G2_WR(1, true); else G2_WR(1, false); }
      else { if (sym) G2_WR(2, true); else G2_WR(2, false); }
      G2PTQ_LAUNCHED();
    }
#undef G2_WR
    return G2PTQ_OK;
  });
}

extern "C" int g2ptq_kv_read(void* stream, const g2ptq_kv_cache* cache, const int32_t* table,
                             int64_t ldt, int64_t B, int64_t width, const int32_t* cu,
                             int64_t total, void* k, void* v, int dtype) {
  ReadArgs a;
  G2PTQ_TRY(check_cache("kv_read", cache, a.c));
  G2PTQ_CHECK(dtype >= 0 && dtype <= 2, "kv_read: dtype code %d", dtype);
  G2PTQ_CHECK(B >= 0 && width >= 0 && ldt >= width, "kv_read: bad page table");
  G2PTQ_CHECK(total >= 0 && total * a.c.H < (1ll << 31), "kv_read: %lld tokens of %lld heads",
              (long long)total, (long long)a.c.H);
  if (total == 0) return G2PTQ_OK;
  G2PTQ_CHECK(k && v && cu && (table || B * width == 0), "kv_read: null pointer");
  G2PTQ_CHECK(aligned16(k) && aligned16(v), "kv_read: outputs not 16-byte aligned");
  a.table = table, a.ldt = ldt, a.B = B, a.width = width, a.cu = cu, a.total = total;
  a.out[0] = k, a.out[1] = v;
  // Some four pieces per thread, fewer where that leaves CUs idle: one number for both widths.
  // MI355X, 8 bits, 131072 tokens of 8 × 128: 177 µs, 191 with eight.  Two take 158 there, but
  // lose at 4 bits (65536 tokens of 8 × 64 35 against 31.6 µs).
  const int64_t pieces = a.c.H * a.c.D / 16;
  int64_t tokens = std::max<int64_t>(1, std::min<int64_t>(kReadTokens, 1024 / pieces));
  while (tokens > 1 && cdiv(total, tokens) < 256) tokens /= 2;
  a.tokens = (int)tokens;
  hipStream_t st = as_stream(stream);
  for (a.first = 0; a.first < total; a.first += kMaxGroups * tokens) {
    const dim3 grid((unsigned)std::min(cdiv(total - a.first, tokens), kMaxGroups), 2);
#define G2_RD(DT)                                                                          \
  do {                                                                                     \
    if (a.c.bits == 8)                                                                     \
      hipLaunchKernelGGL((kv_read_kernel<DT, 8>), grid, dim3(256), 0, st, a);              \
    else                                                                                   \
      hipLaunchKernelGGL((kv_read_kernel<DT, 4>), grid, dim3(256), 0, st, a);              \
  } while (0)
    if (dtype == 0) G2_RD(0);
    else if (dtype == 1) G2_RD(1);
    else G2_RD(2);
    G2PTQ_LAUNCHED();
  }
#undef G2_RD
  return G2PTQ_OK;
}
