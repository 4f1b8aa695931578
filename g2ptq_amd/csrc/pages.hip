// Page tables and slot maps of a paged cache, from request lengths.
//
// State (g2ptq_page_tables): a row of page numbers and a length per request, and a stack of
// free pages, free_pages[0 .. free_count − 1], the last on top.  With c(n) = ceil(n / page):
//
//   extend:  request i of the batch, with ℓ tokens and n new ones, takes c(ℓ + n) − c(ℓ) pages
//            off the top, request by request; its token ℓ + j lives in slot
//            row[(ℓ + j) / page]·page + (ℓ + j) mod page
//   release: request i, cut to m tokens, gives its pages c(m) .. c(ℓ) − 1 back so that the
//            first request's first page ends on top: releasing what an extend took, in the same
//            order, restores the stack
//
// Everything is whole numbers.  A request whose demand does not fit is left as it was, and
// flagged.
//
// One workgroup plans (duplicates, sums over the requests, state), many fill the tables and the
// tokens' slots.  Bound by latency: MI355X, under the profiler, 32 requests of one token each in
// one launch 5.7–5.9 µs and 3.4–3.6 for its release; 700 requests of 717000 tokens in all 4.6–5.3
// to plan and 6.9–8.5 to fill (11.5 MB of slots and positions: 2.3 µs at a copy's rate), their
// release 2.8–2.9 and 3.1–3.4.
#include <algorithm>

#include "common.hpp"

namespace g2ptq {
namespace {

constexpr int kPlan = 1024;  // threads of the planning workgroup, and requests of a round
// Places in LDS of the rows of up to kPlan and of up to kMany requests.
constexpr int kMany = 4096, kHash = 4 * kPlan, kLargeHash = 2 * kMany;
// Requests, and tables' entries and tokens, that the planning workgroup fills by itself.
constexpr int kFew = 64;
constexpr int64_t kSmall = 16384;

struct Tables {
  int32_t *table, *lengths, *free_pages, *free_count, *mark;
  int* flags;
  int64_t seqs, width, pages;
  int shift;  // log2 of the slots of a page
};

// What a plan says of a request: its row (−1: none), its length before (−1: its tokens are
// not placed), its pages before and after, the stack's place of its first page to move.
struct Plan {
  int32_t row, before, had, need, place;
};

struct StepArgs {
  Tables s;
  const int32_t *rows, *counts;  // B; counts: new tokens, or tokens to keep (null: none)
  int64_t B, total;
  Plan* plan;                    // B
  int32_t* table;                // B × width
  int32_t *cu, *kv_lens;         // B + 1, B
  int64_t *slots, *positions;    // total
  int token_blocks;              // of the filling launch
};

// Sums that stay at 2^32 − 1 once they reach it: beyond every count and total, which are below
// 2^31.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
  return add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
// Inclusive sums over the wave: within 16 lanes, then the rows before.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = scan_step<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
  return scan_step<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
}

struct Sums {
  uint32_t v[2];
};
// Inclusive sums over the planning workgroup of two numbers each, on top of `before`; returns
// the totals.
__device__ __forceinline__ Sums group_scan(Sums& s, const Sums& before,
                                           uint32_t (*lds)[kPlan / 64]) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  Sums all;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s.v[i] = wave_scan(s.v[i]);
    if (lane == 63) lds[i][wave] = s.v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // (every wave sums the waves' totals: lane w has those up to wave w)
    const uint32_t sums = wave_scan(lane < kPlan / 64 ? lds[i][lane] : 0u);
    all.v[i] = add_sat(before.v[i],
                       (uint32_t)__builtin_amdgcn_readlane((int)sums, kPlan / 64 - 1));
    const uint32_t ahead =
        wave ? (uint32_t)__builtin_amdgcn_readlane((int)sums, max(wave - 1, 0)) : 0u;
    s.v[i] = add_sat(add_sat(s.v[i], ahead), before.v[i]);
  }
  return all;
}

// A row named twice counts once, for the first request of the batch.  Up to kMany requests meet
// in LDS (HASH places); more leave the lowest request that names a row in its mark
// (0x7fffffff between calls; HASH = 0).
template <int HASH>
struct Rows {
  int32_t key[HASH ? HASH : 1], first[HASH ? HASH : 1];
};
template <int HASH>
__device__ __forceinline__ void clear_rows(Rows<HASH>& r) {
  for (int i = threadIdx.x; i < HASH; i += kPlan) r.key[i] = -1, r.first[i] = 0x7fffffff;
}
// The row's place.  (Ends: there are more places than rows.)
template <int HASH>
__device__ __forceinline__ int enter_row(Rows<HASH>& r, int32_t row, int32_t i) {
  static_assert((HASH & (HASH - 1)) == 0, "a power of two");
  uint32_t h = ((uint32_t)row * 2654435761u >> 8) & (HASH - 1);
  for (;;) {
    const int32_t was = atomicCAS(&r.key[h], -1, row);
    if (was == -1 || was == row) break;
    h = (h + 1) & (HASH - 1);
  }
  atomicMin(&r.first[h], i);
  return (int)h;
}
__device__ __forceinline__ bool is_row(const StepArgs& a, int32_t row) {
  return row >= 0 && row < a.s.seqs;
}
// (the state is the caller's memory: within its bounds whatever was written there)
__device__ __forceinline__ int32_t free_pages(const StepArgs& a) {
  return (int32_t)min<int64_t>(max(*a.s.free_count, 0), a.s.pages);
}
__device__ __forceinline__ int32_t length_of(const StepArgs& a, int32_t row) {
  return (int32_t)min<int64_t>(max(a.s.lengths[row], 0), a.s.width << a.s.shift);
}
__device__ __forceinline__ void mark_rows(const StepArgs& a) {
  for (int64_t i = threadIdx.x; i < a.B; i += kPlan)
    if (is_row(a, a.rows[i])) atomicMin(a.s.mark + a.rows[i], (int32_t)i);
  __threadfence();
  __syncthreads();
}
__device__ __forceinline__ bool first_of_row(const StepArgs& a, int32_t row, int64_t i) {
  return __hip_atomic_load(a.s.mark + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
         (int32_t)i;
}
__device__ __forceinline__ void unmark_rows(const StepArgs& a) {
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.B; i += kPlan)
    if (is_row(a, a.rows[i]))
      __hip_atomic_store(a.s.mark + a.rows[i], 0x7fffffff, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ int64_t pages_of(const Tables& s, int64_t n) {
  return (n + (1 << s.shift) - 1) >> s.shift;
}

// The request's page of column c.
__device__ __forceinline__ int32_t page_of(const StepArgs& a, const Plan& p, int64_t c) {
  return c < p.had ? a.s.table[p.row * a.s.width + c] : a.s.free_pages[p.place - (c - p.had)];
}

// A wave's part of request b's row of the batch's tables, and its new pages into its own row.
__device__ __forceinline__ void extend_row(const StepArgs& a, int64_t b, const Plan& p, int lane) {
  int32_t* out = a.table + b * a.s.width;
  const int64_t end = p.row < 0 ? 0 : p.need;
#pragma unroll 4
  for (int64_t c = lane; c < a.s.width; c += 64) {
    const int32_t page = c < end ? page_of(a, p, c) : -1;
    if (c >= p.had && c < end) a.s.table[p.row * a.s.width + c] = page;
    out[c] = page;
  }
}

// Token t's slot and position.  cu: the requests' offsets; the batch's tokens end at `end`; its
// request is one of lo .. hi.
__device__ __forceinline__ void extend_token(const StepArgs& a, int64_t t, const int32_t* cu,
                                             const Plan* plan, int32_t end, int lo, int hi) {
  int64_t slot = -1, position = 0;
  if (t < end) {
    while (lo < hi) {  // cu[lo] <= t < cu[lo + 1]
      const int mid = (lo + hi) >> 1;
      if (cu[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    const Plan p = plan[lo];
    if (p.row >= 0 && p.before >= 0) {
      position = p.before + (t - cu[lo]);
      slot = ((int64_t)page_of(a, p, position >> a.s.shift) << a.s.shift) +
             (position & ((1 << a.s.shift) - 1));
    }
  }
  a.slots[t] = slot;
  a.positions[t] = position;
}

// One workgroup: rows and counts to plans.  FILL: up to kFew requests, whose plans stay in LDS and
// whose entries the workgroup fills too.  A step of few requests is a chain of four memory
// latencies and a launch.
template <int HASH, bool FILL>
__global__ __launch_bounds__(kPlan) void extend_plan_kernel(StepArgs a) {
  static_assert(HASH || !FILL, "plans in LDS are of one round");
  __shared__ uint32_t lds[2][kPlan / 64];
  __shared__ Rows<HASH> hashed;
  __shared__ Plan planL[FILL ? kFew : 1];
  __shared__ int32_t cuL[FILL ? kFew + 1 : 1];
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  const int32_t count = free_pages(a);
  if (HASH) clear_rows(hashed);
  else mark_rows(a);
  Sums before_all = {{0, 0}};  // tokens and pages of the rounds before
  for (int64_t b0 = 0; b0 < a.B; b0 += kPlan) {
    const int64_t b = b0 + threadIdx.x;
    const bool on = b < a.B;
    const int32_t row = on ? a.rows[b] : -1;
    int64_t n = on ? a.counts[b] : 0;
    const bool inside = is_row(a, row);
    const int32_t held = inside ? length_of(a, row) : 0;
    bool known = inside, bad = n < 0 || row >= a.s.seqs;
    if constexpr (HASH > 0) {
      __syncthreads();
      int place = 0;
      if (inside) place = enter_row(hashed, row, (int32_t)b);
      __syncthreads();
      if (inside) known = hashed.first[place] == (int32_t)b;
    } else if (inside) {
      known = first_of_row(a, row, b);
    }
    bad |= inside && !known;
    n = n < 0 ? 0 : n;
    const int64_t before = known ? held : 0;
    const int64_t had = pages_of(a.s, before), need = pages_of(a.s, before + n);
    const bool wide = known && n > 0 && need > a.s.width;
    // A request whose tokens end past total is refused, and so are all later ones that have
    // any: that their pages are counted changes nothing for those before.
    Sums s = {{(uint32_t)n, known && n > 0 && !wide ? (uint32_t)(need - had) : 0u}};
    const uint32_t mine = s.v[1];
    const Sums all = group_scan(s, before_all, lds);
    const bool past = n > 0 && s.v[0] > (uint32_t)a.total;
    bool ok = known && n > 0 && !wide && !past;
    const bool short_of = ok && mine > 0 && s.v[1] > (uint32_t)count;
    ok = ok && !short_of;
    if (on) {
      const int32_t start = (int32_t)min(s.v[0] - (uint32_t)n, (uint32_t)a.total);
      a.cu[b] = start;
      a.kv_lens[b] = known ? (int32_t)(before + (ok ? n : 0)) : 0;
      Plan p;
      p.row = known ? row : -1;
      p.before = known && n > 0 && !ok ? -1 : (int32_t)before;
      p.had = (int32_t)had, p.need = (int32_t)(ok ? need : had);
      p.place = (int32_t)(count - 1 - (int64_t)(s.v[1] - mine));
      if (FILL) planL[threadIdx.x] = p, cuL[threadIdx.x] = start;
      else a.plan[b] = p;
      if (ok) a.s.lengths[row] = (int32_t)(before + n);
      // (those that get pages are the first that need any)
      if (ok && mine) atomicMax(&taken, (int)s.v[1]);
      const int flag = (bad || past ? G2PTQ_FLAG_BAD_INDEX : 0) |
                       (short_of || (wide && !past) ? G2PTQ_FLAG_NO_ROOM : 0);
      if (flag) atomicOr(a.s.flags, flag);
    }
    before_all = all;
  }
  __syncthreads();
  const int32_t tokens = (int32_t)min(before_all.v[0], (uint32_t)a.total);
  if (threadIdx.x == 0) {
    a.cu[a.B] = tokens;
    *a.s.free_count = count - taken;
  }
  if (!HASH) unmark_rows(a);
  if constexpr (FILL) {
    if (threadIdx.x == 0) cuL[a.B] = tokens;
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t t = threadIdx.x; t < a.total; t += kPlan)
      extend_token(a, t, cuL, planL, tokens, 0, (int)a.B - 1);
    for (int64_t b = wave; b < a.B; b += kPlan / 64) extend_row(a, b, planL[b], lane);
  }
}

constexpr int kFillTokens = 1024;  // of a filling workgroup
constexpr int kSpan = 256;         // of one of its waves

// The first request b of B with cu[b + 1] > t, by the whole wave: 64 ranges a step.
__device__ __forceinline__ int request_of(const int32_t* cu, int B, int64_t t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B;
  while (n > 1) {
    const int stride = (n + 63) / 64;
    const uint64_t past = __ballot(cu[lo + min((lane + 1) * stride, n)] > t);
    const int k = past ? __builtin_ctzll(past) : (n - 1) / stride;
    lo += k * stride, n = min(stride, n - k * stride);
  }
  return lo;
}

// A wave's tokens from t0 on: the requests of the first and the last are looked up by the wave,
// then each token's between them.  cu: the offsets of the batch.
__device__ __forceinline__ void extend_span(const StepArgs& a, int64_t t0, int32_t end,
                                            const int32_t* cu) {
  const int lane = threadIdx.x & 63;
  int lo = 0, more = 0;  // the first token's request, and how many further ones there are
  if (t0 < end) {
    lo = request_of(cu, (int)a.B, t0);
    more = request_of(cu + lo, (int)a.B - lo, min<int64_t>(t0 + kSpan, end) - 1);
  }
#pragma unroll
  for (int i = 0; i < kSpan / 64; ++i) {
    const int64_t t = t0 + i * 64 + lane;
    if (t < a.total) extend_token(a, t, cu + lo, a.plan + lo, end, 0, more);
  }
}

// The first token_blocks workgroups take tokens, the others four rows each.  Offsets of up to
// kPlan requests come into LDS, where they are looked through in a fraction of a memory's
// latency.
__global__ __launch_bounds__(256) void extend_fill_kernel(StepArgs a) {
  __shared__ int32_t cuL[kPlan + 1];
  const int64_t block = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (block >= a.token_blocks) {
    const int64_t b = (block - a.token_blocks) * 4 + wave;
    if (b < a.B) extend_row(a, b, a.plan[b], lane);
    return;
  }
  const int64_t t0 = block * kFillTokens + wave * kSpan;
  if (a.B <= kPlan) {
#pragma unroll
    for (int i = 0; i < kPlan; i += 256)
      if (i + (int)threadIdx.x <= a.B) cuL[i + threadIdx.x] = a.cu[i + threadIdx.x];
    if (a.B == kPlan && threadIdx.x == 0) cuL[kPlan] = a.cu[kPlan];
    __syncthreads();
    extend_span(a, t0, cuL[a.B], cuL);
  } else {
    extend_span(a, t0, a.cu[a.B], a.cu);
  }
}

// A wave's part of what request b gives back.
__device__ __forceinline__ void release_row(const StepArgs& a, const Plan& p, int lane) {
  if (p.row < 0) return;
#pragma unroll 4
  for (int64_t c = p.need + lane; c < p.had; c += 64) {
    int32_t* entry = a.s.table + p.row * a.s.width + c;
    const int64_t place = p.place - (c - p.need);
    if (place >= 0 && place < a.s.pages) a.s.free_pages[place] = *entry;
    *entry = -1;
  }
}

template <int HASH, bool FILL>
__global__ __launch_bounds__(kPlan) void release_plan_kernel(StepArgs a) {
  static_assert(HASH || !FILL, "plans in LDS are of one round");
  __shared__ uint32_t lds[2][kPlan / 64];
  __shared__ Rows<HASH> hashed;
  __shared__ Plan planL[FILL ? kFew : 1];
  const int32_t count = free_pages(a);
  if (HASH) clear_rows(hashed);
  else mark_rows(a);
  Sums whole = {{0, 0}};
  // the number of all pages first, then the requests' places (both known at once in one round)
  const bool one = a.B <= kPlan;
  for (int pass = one ? 1 : 0; pass < 2; ++pass) {
    Sums before_all = {{0, 0}};
    for (int64_t b0 = 0; b0 < a.B; b0 += kPlan) {
      const int64_t b = b0 + threadIdx.x;
      const bool on = b < a.B;
      const int32_t row = on ? a.rows[b] : -1;
      const int32_t keep = on && a.counts ? a.counts[b] : 0;
      const bool inside = is_row(a, row);
      const int32_t held = inside ? length_of(a, row) : 0;
      bool known = inside;
      if constexpr (HASH > 0) {
        __syncthreads();
        int place = 0;
        if (inside) place = enter_row(hashed, row, (int32_t)b);
        __syncthreads();
        if (inside) known = hashed.first[place] == (int32_t)b;
      } else if (inside) {
        known = first_of_row(a, row, b);
      }
      const bool bad = row >= a.s.seqs || (inside && !known) ||
                       (known && (keep < 0 || keep > held));
      known = known && !bad;
      const int32_t had = known ? (int32_t)pages_of(a.s, held) : 0;
      const int32_t kept = known ? (int32_t)pages_of(a.s, keep) : 0;
      Sums s = {{(uint32_t)(had - kept), 0}};
      const Sums all = group_scan(s, before_all, lds);
      if (one) whole = all;
      if (pass == 1 && on) {
        Plan p;
        p.row = known ? row : -1;
        p.before = held, p.had = had, p.need = kept;
        p.place = (int32_t)((int64_t)count + whole.v[0] - 1 - (s.v[0] - (had - kept)));
        if (FILL) planL[threadIdx.x] = p;
        else a.plan[b] = p;
        if (bad) atomicOr(a.s.flags, G2PTQ_FLAG_BAD_INDEX);
        if (known) a.s.lengths[row] = keep;
      }
      before_all = all;
    }
    if (pass == 0) whole = before_all;
  }
  if (threadIdx.x == 0) *a.s.free_count = (int32_t)(count + whole.v[0]);
  if (!HASH) unmark_rows(a);
  if constexpr (FILL) {
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t b = wave; b < a.B; b += kPlan / 64) release_row(a, planL[b], lane);
  }
}

__global__ __launch_bounds__(256) void release_fill_kernel(StepArgs a) {
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b < a.B) release_row(a, a.plan[b], threadIdx.x & 63);
}

// Whether the planning workgroup fills the entries too, which saves a launch.  MI355X, a step and
// its release, one launch each against two: 32 requests of 129 pages 9.1 and 10.7 µs, 8 with
// 2000 tokens each 8.5 and 9.8, 64 of 256 pages 12.8 and 12.1, 200 of 20 pages with 60 tokens
// each 28.9 and 14.7.
bool few(int64_t B, int64_t entries) { return B <= kFew && entries <= kSmall; }

int check_tables(const char* who, const g2ptq_page_tables* t, int64_t B, const void* rows,
                 const void* ws, size_t ws_bytes, StepArgs& a) {
  G2PTQ_CHECK(t, "%s: null tables", who);
  G2PTQ_CHECK(t->seqs >= 1 && t->seqs < (1ll << 31) && t->width >= 1 && t->width < (1ll << 31) &&
                  t->pages >= 0 && t->pages < (1ll << 31),
              "%s: %lld rows of %lld of %lld pages", who, (long long)t->seqs, (long long)t->width,
              (long long)t->pages);
  G2PTQ_CHECK(t->page >= 1 && t->page <= 4096 && (t->page & (t->page - 1)) == 0,
              "%s: pages of %lld slots (a power of two up to 4096)", who, (long long)t->page);
  G2PTQ_CHECK(t->width * t->page < (1ll << 31), "%s: %lld pages of %lld slots in a row", who,
              (long long)t->width, (long long)t->page);
  G2PTQ_CHECK(t->table && t->lengths && t->free_count && t->mark && t->flags &&
                  (t->free_pages || t->pages == 0), "%s: null table", who);
  G2PTQ_CHECK(B >= 0 && B <= 1 << 20, "%s: %lld requests (at most 1048576)", who, (long long)B);
  G2PTQ_CHECK(B == 0 || rows, "%s: null rows", who);
  if (B && (!ws || ws_bytes < sizeof(Plan) * (size_t)B)) {
    set_error("%s: workspace of %zu bytes, %zu needed", who, ws_bytes, sizeof(Plan) * (size_t)B);
    return G2PTQ_ERR_WORKSPACE;
  }
  G2PTQ_CHECK((reinterpret_cast<uintptr_t>(ws) & 3) == 0, "%s: workspace not 4-byte aligned", who);
  a.s = {t->table, t->lengths, t->free_pages, t->free_count, t->mark, t->flags,
         t->seqs, t->width, t->pages, __builtin_ctzll((unsigned long long)t->page)};
  a.B = B;
  a.plan = static_cast<Plan*>(const_cast<void*>(ws));
  return G2PTQ_OK;
}

}  // namespace
}  // namespace g2ptq

using namespace g2ptq;

extern "C" int g2ptq_pages_workspace(int64_t B, size_t* bytes) {
  G2PTQ_CHECK(bytes && B >= 0 && B <= 1 << 20, "pages_workspace: bad size");
  *bytes = sizeof(Plan) * (size_t)B;
  return G2PTQ_OK;
}

extern "C" int g2ptq_pages_extend(void* stream, const g2ptq_page_tables* tables,
                                  const int32_t* rows, const int32_t* counts, int64_t B,
                                  int64_t total, int32_t* table, int32_t* cu, int32_t* kv_lens,
                                  int64_t* slots, int64_t* positions, void* ws, size_t ws_bytes) {
  StepArgs a{};
  G2PTQ_TRY(check_tables("pages_extend", tables, B, rows, ws, ws_bytes, a));
  G2PTQ_CHECK(total >= 0 && total < (1ll << 31), "pages_extend: %lld tokens", (long long)total);
  G2PTQ_CHECK(cu && (B == 0 || (counts && table && kv_lens)) &&
                  (total == 0 || (slots && positions)), "pages_extend: null pointer");
  a.rows = rows, a.counts = counts, a.total = total;
  a.table = table, a.cu = cu, a.kv_lens = kv_lens, a.slots = slots, a.positions = positions;
  hipStream_t st = as_stream(stream);
  if (few(B, B * a.s.width + total)) {
    hipLaunchKernelGGL((extend_plan_kernel<kHash, true>), dim3(1), dim3(kPlan), 0, st, a);
    G2PTQ_LAUNCHED();
    return G2PTQ_OK;
  }
  if (B <= kPlan)
    hipLaunchKernelGGL((extend_plan_kernel<kHash, false>), dim3(1), dim3(kPlan), 0, st, a);
  else if (B <= kMany)
    hipLaunchKernelGGL((extend_plan_kernel<kLargeHash, false>), dim3(1), dim3(kPlan), 0, st, a);
  else
    hipLaunchKernelGGL((extend_plan_kernel<0, false>), dim3(1), dim3(kPlan), 0, st, a);
  G2PTQ_LAUNCHED();
  a.token_blocks = (int)cdiv(total, kFillTokens);
  hipLaunchKernelGGL(extend_fill_kernel, dim3((unsigned)(a.token_blocks + cdiv(B, 4))), dim3(256),
                     0, st, a);
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}

extern "C" int g2ptq_pages_release(void* stream, const g2ptq_page_tables* tables,
                                   const int32_t* rows, const int32_t* keep, int64_t B, void* ws,
                                   size_t ws_bytes) {
  StepArgs a{};
  G2PTQ_TRY(check_tables("pages_release", tables, B, rows, ws, ws_bytes, a));
  if (B == 0) return G2PTQ_OK;
  a.rows = rows, a.counts = keep;
  hipStream_t st = as_stream(stream);
  if (few(B, B * a.s.width)) {
    hipLaunchKernelGGL((release_plan_kernel<kHash, true>), dim3(1), dim3(kPlan), 0, st, a);
    G2PTQ_LAUNCHED();
    return G2PTQ_OK;
  }
  if (B <= kPlan)
    hipLaunchKernelGGL((release_plan_kernel<kHash, false>), dim3(1), dim3(kPlan), 0, st, a);
  else if (B <= kMany)
    hipLaunchKernelGGL((release_plan_kernel<kLargeHash, false>), dim3(1), dim3(kPlan), 0, st, a);
  else
    hipLaunchKernelGGL((release_plan_kernel<0, false>), dim3(1), dim3(kPlan), 0, st, a);
  G2PTQ_LAUNCHED();
  hipLaunchKernelGGL(release_fill_kernel, dim3((unsigned)cdiv(B, 4)), dim3(256), 0, st, a);
  G2PTQ_LAUNCHED();
  return G2PTQ_OK;
}
