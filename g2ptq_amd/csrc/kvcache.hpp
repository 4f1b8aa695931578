// The paged cache as the kernels see it (layout: kvcache.hip).
#pragma once
#include "common.hpp"

namespace g2ptq {

struct KvCache {
  uint8_t* codes[2];  // keys, values
  float* scale[2];
  uint8_t* zero[2];   // null in the symmetric grid
  int64_t pages, H, D;
  int shift, bits;    // log2 of the slots of a page
  int* flags;

  // Row (slot, head) of scale and zero, and of codes in units of a head's bytes.
  __device__ __forceinline__ int64_t row(int64_t slot, int64_t h) const {
    const int64_t p = slot >> shift;
    return (((p * H + h) << shift) | (slot & ((1 << shift) - 1)));
  }

  // Slot of position p of the sequence with page table row `table` (width
  // entries), or -2 where that names no page of the cache.
  __device__ __forceinline__ int64_t slot(const int32_t* table, int64_t width, int64_t p) const {
    const int64_t i = p >> shift;
    if (i >= width) return -2;
    const int64_t g = table[i];
    if (g < 0 || g >= pages) return -2;
    return (g << shift) | (p & ((1 << shift) - 1));
  }

  // The sequence of row t of a ragged batch (cu: B + 1 offsets), or -1.
  static __device__ __forceinline__ int64_t sequence(const int32_t* cu, int64_t B, int64_t t) {
    if (B == 0 || t < cu[0] || t >= cu[B]) return -1;
    int64_t lo = 0, hi = B;  // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
      const int64_t m = (lo + hi) >> 1;
      if (cu[m] <= t) lo = m;
      else hi = m;
    }
    return lo;
  }

  // The same where a whole wave looks for one t: 64 offsets at a time, so that up to 64
  // sequences cost one load's latency and 4096 two.
  static __device__ __forceinline__ int64_t sequence_of_wave(const int32_t* cu, int64_t B,
                                                             int64_t t) {
    if (B == 0) return -1;
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, n = B;  // cu[i + 1] <= t for i < lo, and for none from lo + n up
    while (n > 0) {
      const int64_t step = (n + 63) >> 6, i = (lane + 1) * step - 1;
      const uint64_t before = __builtin_amdgcn_ballot_w64(i < n && cu[lo + min(i, n - 1) + 1] <= t);
      const int64_t next = lo + __builtin_popcountll(before) * step;
      n = min(step - 1, lo + n - next);
      lo = next;
    }
    return lo < B && cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
  }

  // The same where `near` is likely the one (or -1).
  static __device__ __forceinline__ int64_t sequence_near(const int32_t* cu, int64_t B, int64_t t,
                                                          int64_t near) {
    return near >= 0 && t >= cu[near] && t < cu[near + 1] ? near : sequence(cu, B, t);
  }

  // Slot of row t of a ragged batch; -1 outside every sequence.
  __device__ __forceinline__ int64_t find(const int32_t* table, int64_t ldt, int64_t width,
                                          const int32_t* cu, int64_t B, int64_t t,
                                          int64_t near) const {
    const int64_t b = sequence_near(cu, B, t, near);
    if (b < 0) return -1;
    return slot(table + b * ldt, width, t - cu[b]);
  }
};

// Checks the caller's description of a cache and lays it out for kernels.
int check_cache(const char* who, const g2ptq_kv_cache* c, KvCache& k);

}  // namespace g2ptq
