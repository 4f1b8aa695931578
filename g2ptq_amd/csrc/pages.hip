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
// Everything is whole numbers; sums are 64 bits.  A request whose demand does not fit is left
// as it was, and flagged.
#include <algorithm>

#include "common.hpp"

namespace g2ptq {
namespace {

constexpr int kPlan = 1024;  // threads of the planning workgroup
// Entries (tables' and tokens') that the planning workgroup fills by itself.
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
  int32_t row, before;
  int64_t place;
  int32_t had, need;
};

struct StepArgs {
  Tables s;
  const int32_t *rows, *counts;  // B; counts: new tokens, or tokens to keep (null: none)
  int64_t B, total;
  Plan* plan;                    // B
  int32_t* table;                // B × width
  int32_t *cu, *kv_lens;         // B + 1, B
  int64_t *slots, *positions;    // total
  bool fill;                     // the planning workgroup fills too
};

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int64_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Inclusive sums over the planning workgroup of two numbers each; all: their totals.
__device__ __forceinline__ void group_scan(int64_t (&v)[2], int64_t (&all)[2],
                                           int64_t (*lds)[kPlan / 64]) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = wave_scan(v[i]);
    if ((threadIdx.x & 63) == 63) lds[i][wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int64_t sum = 0;
    for (int w = 0; w < kPlan / 64; ++w) {
      if (w == wave) v[i] += sum;
      sum += lds[i][w];
    }
    all[i] = sum;
  }
  __syncthreads();
}

// Marks rows with the lowest request that names them, so that a row named twice counts once.
// Marks are INT_MAX between calls.
__device__ __forceinline__ void mark_rows(const StepArgs& a) {
  for (int64_t i = threadIdx.x; i < a.B; i += kPlan) {
    const int32_t row = a.rows[i];
    if (row >= 0 && row < a.s.seqs) atomicMin(a.s.mark + row, (int32_t)i);
  }
  __threadfence();
  __syncthreads();
}
__device__ __forceinline__ bool first_of_row(const StepArgs& a, int32_t row, int64_t i) {
  return __hip_atomic_load(a.s.mark + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
         (int32_t)i;
}
__device__ __forceinline__ void unmark_rows(const StepArgs& a) {
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.B; i += kPlan) {
    const int32_t row = a.rows[i];
    if (row >= 0 && row < a.s.seqs)
      __hip_atomic_store(a.s.mark + row, 0x7fffffff, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

__device__ __forceinline__ int64_t pages_of(const Tables& s, int64_t n) {
  return (n + (1 << s.shift) - 1) >> s.shift;
}

// Entry `at` of the batch's tables.
__device__ __forceinline__ void extend_entry(const StepArgs& a, int64_t at) {
  const int64_t b = at / a.s.width, c = at - b * a.s.width;
  const Plan p = a.plan[b];
  int32_t page = -1;
  if (p.row >= 0) {
    if (c < p.had) page = a.s.table[p.row * a.s.width + c];
    else if (c < p.need) {
      page = a.s.free_pages[p.place - (c - p.had)];
      a.s.table[p.row * a.s.width + c] = page;
    }
  }
  a.table[at] = page;
}

// Token t's slot and position.
__device__ __forceinline__ void extend_token(const StepArgs& a, int64_t t) {
  int64_t slot = -1, position = 0;
  if (t < a.cu[a.B]) {
    int64_t lo = 0, hi = a.B - 1;  // the request with cu[b] <= t < cu[b + 1]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.cu[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    const Plan p = a.plan[lo];
    if (p.row >= 0 && p.before >= 0) {
      position = p.before + (t - a.cu[lo]);
      const int64_t c = position >> a.s.shift;
      const int32_t page = c < p.had ? a.s.table[p.row * a.s.width + c]
                                     : a.s.free_pages[p.place - (c - p.had)];
      slot = ((int64_t)page << a.s.shift) + (position & ((1 << a.s.shift) - 1));
    }
  }
  a.slots[t] = slot;
  a.positions[t] = position;
}

__global__ __launch_bounds__(kPlan) void extend_plan_kernel(StepArgs a) {
  __shared__ int64_t lds[2][kPlan / 64];
  mark_rows(a);
  const int64_t count = *a.s.free_count;
  int64_t tokens = 0, pages = 0, taken = 0;  // of the requests before this round's
  for (int64_t b0 = 0; b0 < a.B; b0 += kPlan) {
    const int64_t b = b0 + threadIdx.x;
    int32_t row = -1, before = 0;
    int64_t n = 0;
    bool known = false, bad = false, full = false;
    if (b < a.B) {
      row = a.rows[b];
      n = a.counts[b];
      if (n < 0) n = 0, bad = true;
      if (row >= a.s.seqs) bad = true;
      else if (row >= 0) {
        known = first_of_row(a, row, b);
        bad |= !known;
      }
      if (known) before = a.s.lengths[row];
    }
    const int64_t had = pages_of(a.s, before), need = pages_of(a.s, before + n);
    int64_t v[2] = {n, 0}, all[2];
    group_scan(v, all, lds);
    const int64_t start = tokens + v[0] - n;
    // what the step's tokens or its own row have no room for is refused before pages are counted
    const bool past = start + n > a.total && n > 0;
    full = known && n > 0 && !past && need > a.s.width;
    bool ok = known && n > 0 && !full && !past;
    const int64_t last = tokens + all[0];
    v[0] = 0, v[1] = ok ? need - had : 0;
    group_scan(v, all, lds);
    const int64_t before_pages = pages + v[1] - (ok ? need - had : 0);
    if (ok && need > had && pages + v[1] > count) ok = false, full = true;
    if (b < a.B) {
      a.cu[b] = (int32_t)min(start, a.total);
      a.kv_lens[b] = known ? (int32_t)(before + (ok ? n : 0)) : 0;
      Plan p;
      p.row = known ? row : -1;
      p.before = before;
      p.place = count - 1 - before_pages;
      p.had = (int32_t)had, p.need = (int32_t)(ok ? need : had);
      if (known && n > 0 && !ok) p.before = -1;
      a.plan[b] = p;
      if (ok) a.s.lengths[row] = (int32_t)(before + n);
      if (bad || past) atomicOr(a.s.flags, G2PTQ_FLAG_BAD_INDEX);
      if (full) atomicOr(a.s.flags, G2PTQ_FLAG_NO_ROOM);
    }
    tokens = last;
    pages += all[1];
    v[0] = 0, v[1] = ok ? need - had : 0;
    group_scan(v, all, lds);
    taken += all[1];
  }
  if (threadIdx.x == 0) {
    a.cu[a.B] = (int32_t)min(tokens, a.total);
    *a.s.free_count = (int32_t)(count - taken);
  }
  unmark_rows(a);
  if (a.fill) {
    __syncthreads();
    for (int64_t i = threadIdx.x; i < a.B * a.s.width; i += kPlan) extend_entry(a, i);
    for (int64_t t = threadIdx.x; t < a.total; t += kPlan) extend_token(a, t);
  }
}

__global__ __launch_bounds__(256) void extend_fill_kernel(StepArgs a, int64_t first) {
  const int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x, entries = a.B * a.s.width;
  if (i < entries) extend_entry(a, i);
  else if (i < entries + a.total) extend_token(a, i - entries);
}

// Column c of request b's row, where its page goes back.
__device__ __forceinline__ void release_entry(const StepArgs& a, int64_t at) {
  const int64_t b = at / a.s.width, c = at - b * a.s.width;
  const Plan p = a.plan[b];
  if (p.row < 0 || c < p.need || c >= p.had) return;
  int32_t* entry = a.s.table + p.row * a.s.width + c;
  const int64_t place = p.place - (c - p.need);
  if (place >= 0 && place < a.s.pages) a.s.free_pages[place] = *entry;
  *entry = -1;
}

__global__ __launch_bounds__(kPlan) void release_plan_kernel(StepArgs a) {
  __shared__ int64_t lds[2][kPlan / 64];
  mark_rows(a);
  const int64_t count = *a.s.free_count;
  int64_t pages = 0;  // of the requests before this round's
  for (int round = 0; round < 2; ++round) {  // the number of all, then their places
    const int64_t whole = pages;
    pages = 0;
    for (int64_t b0 = 0; b0 < a.B; b0 += kPlan) {
      const int64_t b = b0 + threadIdx.x;
      int32_t row = -1, before = 0;
      int64_t keep = 0;
      bool known = false, bad = false;
      if (b < a.B) {
        row = a.rows[b];
        keep = a.counts ? a.counts[b] : 0;
        if (row >= a.s.seqs) bad = true;
        else if (row >= 0) {
          known = first_of_row(a, row, b);
          bad |= !known;
        }
        if (known) before = a.s.lengths[row];
        if (known && (keep < 0 || keep > before)) known = false, bad = true;
      }
      const int64_t had = known ? pages_of(a.s, before) : 0, kept = known ? pages_of(a.s, keep) : 0;
      int64_t v[2] = {had - kept, 0}, all[2];
      group_scan(v, all, lds);
      if (round == 1 && b < a.B) {
        Plan p;
        p.row = known ? row : -1;
        p.before = before;
        p.had = (int32_t)had, p.need = (int32_t)kept;
        p.place = count + whole - 1 - (pages + v[0] - (had - kept));
        a.plan[b] = p;
        if (bad) atomicOr(a.s.flags, G2PTQ_FLAG_BAD_INDEX);
        if (known) a.s.lengths[row] = (int32_t)keep;
      }
      pages += all[0];
    }
  }
  if (threadIdx.x == 0) *a.s.free_count = (int32_t)(count + pages);
  unmark_rows(a);
  if (a.fill) {
    __syncthreads();
    for (int64_t i = threadIdx.x; i < a.B * a.s.width; i += kPlan) release_entry(a, i);
  }
}

__global__ __launch_bounds__(256) void release_fill_kernel(StepArgs a, int64_t first) {
  const int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < a.B * a.s.width) release_entry(a, i);
}

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
  G2PTQ_CHECK((reinterpret_cast<uintptr_t>(ws) & 7) == 0, "%s: workspace not 8-byte aligned", who);
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
  G2PTQ_CHECK(cu && (B == 0 || (counts && table && kv_lens)) && (total == 0 || (slots && positions)),
              "pages_extend: null pointer");
  a.rows = rows, a.counts = counts, a.total = total;
  a.table = table, a.cu = cu, a.kv_lens = kv_lens, a.slots = slots, a.positions = positions;
  const int64_t all = B * a.s.width + total;
  a.fill = all <= kSmall;
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(extend_plan_kernel, dim3(1), dim3(kPlan), 0, st, a);
  G2PTQ_LAUNCHED();
  for (int64_t first = 0; !a.fill && first < all; first += kMaxGroups * 256) {
    hipLaunchKernelGGL(extend_fill_kernel,
                       dim3((unsigned)std::min(cdiv(all - first, 256), kMaxGroups)), dim3(256), 0,
                       st, a, first);
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}

extern "C" int g2ptq_pages_release(void* stream, const g2ptq_page_tables* tables,
                                   const int32_t* rows, const int32_t* keep, int64_t B, void* ws,
                                   size_t ws_bytes) {
  StepArgs a{};
  G2PTQ_TRY(check_tables("pages_release", tables, B, rows, ws, ws_bytes, a));
  if (B == 0) return G2PTQ_OK;
  a.rows = rows, a.counts = keep;
  const int64_t all = B * a.s.width;
  a.fill = all <= kSmall;
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(release_plan_kernel, dim3(1), dim3(kPlan), 0, st, a);
  G2PTQ_LAUNCHED();
  for (int64_t first = 0; !a.fill && first < all; first += kMaxGroups * 256) {
    hipLaunchKernelGGL(release_fill_kernel,
                       dim3((unsigned)std::min(cdiv(all - first, 256), kMaxGroups)), dim3(256), 0,
                       st, a, first);
    G2PTQ_LAUNCHED();
  }
  return G2PTQ_OK;
}
