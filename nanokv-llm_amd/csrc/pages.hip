// Pages of a paged K/V cache shared between sequences: taking pages for new tokens, freeing them,
// forking sequences and closing up the pool. No counterpart in the reference's device code: it
// keeps blocks' reference counts and free lists on the host (nanokvllm/engine/block_manager.py:
// 13-138), where a fork, a rollback or a defragmentation means a host loop, a synchronisation and
// copies for every layer's K and V.
//
// The state is three int32 arrays: a reference count per page (0: free), a length per row
// (sequence) and a block table per row. A row's last page, where it is filled in part, belongs to
// that row alone (the operators keep it so), so that new tokens never land in a page that another
// row reads. A call takes the lowest free pages, in the order of its list, as far as they go; every
// decision is by the state before the call, so that results do not depend on timing.
//
// MI355X design: an operator is a plan of one workgroup of 1024 threads (prefix sums over the list,
// one walk over the counts for the free pages) and, where pages are copied or many table entries
// change, a second launch of up to kCopyGroups workgroups that reads the plan from the workspace.
// A copy is bound by HBM: rows are read once and written once, 16 bytes a lane, kCopyUnroll of them
// in flight; the grid's y runs over the 2 * layers planes of the pool. 50 pages of 512 KiB in each
// of 32 planes: 333 us, 5.0 TB/s read and written together (a copy of 2 GiB: 4.8); twice or half
// the loads in flight or the workgroups within 1.5%; loads that bypass the caches 4% faster there,
// but 32% slower where four beams of one sequence copy the same rows (24.4 -> 32.1 us).
// compact walks whole tables, empty rows' too: eight pages moved behind a copy of the state, in a
// graph, take 21 us over 64 rows of 64 entries (the copy alone 17.6), 62 over 2048 of 1024
// (17.5), 366 over 8192 of 2048 (25). Kernel times: one token each for 64 rows 3.5 us; 33 rows
// rolled back 6.0 + 3.7.
#include "nkv_common.h"

#include <algorithm>

namespace nkv {

constexpr int kPlan = 1024;        // threads of a plan
constexpr int kPlanWaves = kPlan / 64;
constexpr int kWalk = 16;          // counts a thread of a walk reads at once
constexpr int kMaxList = 8192;     // rows, and entries of a list: one LDS word each
constexpr int kMaxPages = 1 << 20; // prefix sums of needed pages fit 32 bits
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyBytes = kCopyThreads * 16 * kCopyUnroll;  // of a page, one workgroup's
constexpr int kCopyGroups = 4096;
constexpr int kBookGroups = 64;

typedef int32_t i32x2_t __attribute__((ext_vector_type(2)));
typedef int32_t i32x4w_t __attribute__((ext_vector_type(4)));

// Workspace: a header, a record for each entry of the list, {source, destination, rows} of each
// copy, and page ids.
struct PlanHeader {
  int32_t n_copies;
  int32_t n_live;  // compact: pages in use
};
constexpr size_t kHeaderBytes = 64;
static size_t pages_ws_bytes(int64_t n_pages) {
  return kHeaderBytes + sizeof(i32x4w_t) * (kMaxList + (size_t)n_pages) +
         2 * sizeof(int32_t) * (size_t)n_pages;
}

struct PagesArgs {
  char* kv;
  int32_t n_planes, n_pages, B, row_bytes;
  int32_t* refs;
  int32_t* lens;
  int32_t* tables;
  int64_t bt_stride;
  int32_t max_blocks, n_rows;
  PlanHeader* head;
  i32x4w_t* items;
  i32x4w_t* copies;
  int32_t* ids;  // a plan's free pages
  int32_t* map;  // compact: a moved page's new place
};

__device__ __forceinline__ int32_t* table_of(const PagesArgs& a, int row) {
  return a.tables + (int64_t)row * a.bt_stride;
}
__device__ __forceinline__ bool page_ok(const PagesArgs& a, int id) {
  NKV_DBG(id < 0 || id >= a.n_pages, NKV_DEBUG_BLOCK);
  return id >= 0 && id < a.n_pages;
}
__device__ __forceinline__ int pages_of(const PagesArgs& a, int tokens) {
  return tokens / a.B + (tokens % a.B != 0);
}

// Exclusive prefix of v over the workgroup, and the total.
__device__ __forceinline__ int plan_scan(int v, int& total) {
  __shared__ int wave_sums[kPlanWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_incl_scan(v);
  if (lane == 63) wave_sums[wave] = incl;
  __syncthreads();
  const int s = lane < kPlanWaves ? wave_sums[lane] : 0;
  const int sums = wave_incl_scan(s);
  total = __builtin_amdgcn_readlane(sums, kPlanWaves - 1);
  const int before = __shfl(sums - s, wave, 64);
  __syncthreads();
  return before + incl - v;
}

// marks[row]: the first entry of the list that names the row.
__device__ __forceinline__ void mark_first(const PagesArgs& a, const int32_t* rows, int n,
                                           int* marks) {
  for (int r = threadIdx.x; r < a.n_rows; r += kPlan) marks[r] = INT32_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int r = rows[i];
    NKV_DBG(r < -1 || r >= a.n_rows, NKV_DEBUG_BLOCK);
    if (r >= 0 && r < a.n_rows) atomicMin(&marks[r], i);
  }
  __syncthreads();
}

// Counts [i0, i0 + kWalk) of [0, n): a bit for each that is zero (ZERO) or positive.
template <bool ZERO>
__device__ __forceinline__ uint32_t count_bits(const int32_t* refs, int i0, int n) {
  i32x4w_t v[kWalk / 4];
#pragma unroll
  for (int k = 0; k < kWalk / 4; ++k) {
    const int i = i0 + 4 * k;
    if (i + 4 <= n) {
      v[k] = *reinterpret_cast<const i32x4w_t*>(refs + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = i + e < n ? refs[i + e] : (ZERO ? 1 : 0);
    }
  }
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < kWalk; ++k) {
    const int c = v[k / 4][k % 4];
    bits |= (uint32_t)(ZERO ? c == 0 : c > 0) << k;
  }
  return bits;
}

// The lowest `want` free pages of [0, n) into ids; how many there are.
__device__ __forceinline__ int find_free(const int32_t* refs, int n, int want, int32_t* ids) {
  int found = 0;
  for (int base = 0; base < n && found < want; base += kPlan * kWalk) {  // uniform
    const int i0 = base + (int)threadIdx.x * kWalk;
    uint32_t bits = count_bits<true>(refs, i0, n);
    int total;
    int at = found + plan_scan(__popc(bits), total);
    for (; bits && at < want; bits &= bits - 1) ids[at++] = i0 + __builtin_ctz(bits);
    found += total;
  }
  return min(found, want);
}

// Pages that entry i of the list needs, in the list's order: what stands before it. An entry that
// does not fit needs none. Sums stop at n_pages + 1, which is more than there can be.
struct Needs {
  int before = 0;
  __device__ __forceinline__ int add(const PagesArgs& a, int need) {
    int total;
    const int excl = before + plan_scan(min(need, a.n_pages + 1), total);
    before = min(before + total, a.n_pages + 1);
    return excl;
  }
};

// The entry whose pages hold the k-th granted one: the last with before[i] <= k.
__device__ __forceinline__ int entry_of(const int* before, int n, int k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (before[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One reference less, never below zero: the outcome is max(0, count - drops) in any order.
__device__ __forceinline__ void drop_ref(const PagesArgs& a, int id) {
  if (!page_ok(a, id)) return;
  int c = __hip_atomic_load(&a.refs[id], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  while (c > 0 && !__hip_atomic_compare_exchange_strong(&a.refs[id], &c, c - 1, __ATOMIC_RELAXED,
                                                        __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT)) {
  }
  NKV_DBG(c <= 0, NKV_DEBUG_BLOCK);
}

// ---------------------------------------------------------------- append
__global__ __launch_bounds__(kPlan) void pages_append_kernel(
    const PagesArgs a, const int32_t* __restrict__ rows, int n, const int32_t* __restrict__ cu,
    int64_t n_tokens, int32_t* __restrict__ slots, int32_t* __restrict__ status) {
  extern __shared__ int lds[];
  int bad = 0;
  if (cu) {
    for (int i = threadIdx.x; i < n; i += kPlan)
      bad |= cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > n_tokens;
    NKV_DBG(bad, NKV_DEBUG_LENGTH);
    bad = __syncthreads_or(bad);
  }
  mark_first(a, rows, n, lds);
  Needs needs;
  for (int base = 0; base < n; base += kPlan) {  // uniform
    const int i = base + (int)threadIdx.x;
    int row = -1, len = 0, add = 0, need = 0;
    if (i < n) {
      const int r = rows[i];
      if (!bad && r >= 0 && r < a.n_rows && lds[r] == i) {
        len = a.lens[r];
        add = cu ? cu[i + 1] - cu[i] : 1;
        const int64_t want = ((int64_t)len + add + a.B - 1) / a.B;
        NKV_DBG(len < 0, NKV_DEBUG_LENGTH);
        if (len >= 0 && want <= a.max_blocks) {
          row = r;
          need = (int)want - pages_of(a, len);
        }
      }
    }
    const int before = needs.add(a, need);
    if (i < n) a.items[i] = i32x4w_t{row, len, add, before};
  }
  const int n_free = needs.before ? find_free(a.refs, a.n_pages, min(needs.before, a.n_pages),
                                              a.ids)
                                  : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    i32x4w_t it = a.items[i];
    const int have = it[0] < 0 ? 0 : pages_of(a, it[1]);
    const int need = it[0] < 0 ? 0 : pages_of(a, it[1] + it[2]) - have;
    const bool ok = it[0] >= 0 && (need == 0 || it[3] + need <= n_free);
    status[i] = ok;
    if (ok) a.lens[it[0]] = it[1] + it[2];
    if (cu) {  // pages_slots_kernel gives the tokens their pages
      if (!ok) a.items[i] = i32x4w_t{-1, 0, 0, 0};
    } else {  // one token: its page and its slot
      int slot = -1;
      if (ok) {
        int32_t* bt = table_of(a, it[0]);
        const int page = need ? a.ids[it[3]] : bt[it[1] / a.B];
        if (need) {
          bt[have] = page;
          a.refs[page] = 1;
        }
        if (page_ok(a, page)) slot = page * a.B + it[1] % a.B;
      }
      slots[i] = slot;
    }
  }
}

// The slots of the tokens that a call with cu appended, one a thread; the first token of a new page
// enters it in the table.
__global__ __launch_bounds__(256) void pages_slots_kernel(const PagesArgs a, int n,
                                                          const int32_t* __restrict__ cu,
                                                          int64_t n_tokens,
                                                          int32_t* __restrict__ slots) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= n_tokens) return;
  int slot = -1;
  if (n > 0 && t >= cu[0] && t < cu[n]) {
    const int i = entry_of(cu, n, (int)t);
    const i32x4w_t it = a.items[i];  // {row, length before, tokens, pages before its own}
    const int j = (int)t - cu[i];
    if (it[0] >= 0 && j < it[2]) {
      const int pos = it[1] + j, k = pos / a.B - pages_of(a, it[1]);
      int32_t* entry = table_of(a, it[0]) + pos / a.B;
      const int page = k >= 0 ? a.ids[it[3] + k] : *entry;
      if (k >= 0 && pos % a.B == 0) {
        *entry = page;
        a.refs[page] = 1;
      }
      if (page_ok(a, page)) slot = page * a.B + pos % a.B;
    }
  }
  slots[t] = slot;
}

// ---------------------------------------------------------------- truncate
__global__ __launch_bounds__(kPlan) void pages_truncate_kernel(
    const PagesArgs a, const int32_t* __restrict__ rows, const int32_t* __restrict__ keep_lens,
    int n, int32_t* __restrict__ status) {
  extern __shared__ int lds[];
  __shared__ int granted;
  mark_first(a, rows, n, lds);
  if (threadIdx.x == 0) granted = 0;
  Needs needs;
  for (int base = 0; base < n; base += kPlan) {  // uniform
    const int i = base + (int)threadIdx.x;
    int row = -1, keep = 0, now = 0, own = 0;
    if (i < n) {
      const int r = rows[i];
      if (r >= 0 && r < a.n_rows && lds[r] == i) {
        keep = keep_lens[i];
        now = a.lens[r];
        NKV_DBG(keep < 0 || keep > now || pages_of(a, max(now, 0)) > a.max_blocks,
                NKV_DEBUG_LENGTH);
        if (keep >= 0 && keep <= now && pages_of(a, now) <= a.max_blocks) {
          row = r;
          if (keep < now && keep % a.B) {  // a page that stays in part: shared?
            const int id = table_of(a, r)[keep / a.B];
            own = page_ok(a, id) && a.refs[id] > 1;
          }
        }
      }
    }
    const int before = needs.add(a, own);
    if (i < n) a.items[i] = i32x4w_t{row, keep, now, own ? before : -1};
  }
  const int n_free = needs.before ? find_free(a.refs, a.n_pages, min(needs.before, a.n_pages),
                                              a.ids)
                                  : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const i32x4w_t it = a.items[i];
    const int row = it[0], keep = it[1], k = it[3];
    const bool ok = row >= 0 && (k < 0 || k < n_free);
    status[i] = ok;
    a.items[i] = i32x4w_t{ok ? row : -1, pages_of(a, keep), pages_of(a, it[2]), 0};
    if (!ok) continue;
    a.lens[row] = keep;
    if (k >= 0) {
      int32_t* e = table_of(a, row) + keep / a.B;
      a.copies[k] = i32x4w_t{*e, a.ids[k], keep % a.B, 0};
      *e = a.ids[k];
      a.refs[a.ids[k]] = 1;
      atomicMax(&granted, k + 1);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) *a.head = PlanHeader{granted, 0};
}

// ---------------------------------------------------------------- fork
__global__ __launch_bounds__(kPlan) void pages_fork_kernel(
    const PagesArgs a, const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
    int n, int share, int32_t* __restrict__ status) {
  extern __shared__ int lds[];
  __shared__ int granted;
  mark_first(a, children, n, lds);
  if (threadIdx.x == 0) granted = 0;
  Needs needs;
  for (int base = 0; base < n; base += kPlan) {  // uniform
    const int i = base + (int)threadIdx.x;
    int parent = -1, child = 0, len = 0, need = 0;
    if (i < n) {
      const int p = parents[i];
      child = children[i];
      NKV_DBG(p < -1 || p >= a.n_rows, NKV_DEBUG_BLOCK);
      if (p >= 0 && p < a.n_rows && child >= 0 && child < a.n_rows && lds[child] == i) {
        len = a.lens[p];
        NKV_DBG(len < 0 || pages_of(a, max(len, 0)) > a.max_blocks, NKV_DEBUG_LENGTH);
        if (a.lens[child] == 0 && len >= 0 && pages_of(a, len) <= a.max_blocks) {
          parent = p;
          need = pages_of(a, len) - (share ? len / a.B : 0);
        }
      }
    }
    const int before = needs.add(a, need);
    if (i < n) a.items[i] = i32x4w_t{parent, child, len, before};
  }
  const int n_free = needs.before ? find_free(a.refs, a.n_pages, min(needs.before, a.n_pages),
                                              a.ids)
                                  : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const i32x4w_t it = a.items[i];
    const int full = share ? it[2] / a.B : 0;
    const int need = it[0] < 0 ? 0 : pages_of(a, it[2]) - full;
    const bool ok = it[0] >= 0 && (need == 0 || it[3] + need <= n_free);
    status[i] = ok;
    lds[i] = it[3];
    if (ok) a.lens[it[1]] = it[2];
    else a.items[i] = i32x4w_t{-1, 0, 0, 0};
    if (ok && need) atomicMax(&granted, it[3] + need);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < granted; k += kPlan) {
    const int i = entry_of(lds, n, k);
    const i32x4w_t it = a.items[i];
    const int j = (share ? it[2] / a.B : 0) + k - lds[i];  // the page's place in the table
    const int page = a.ids[k];
    a.copies[k] = i32x4w_t{table_of(a, it[0])[j], page, min(a.B, it[2] - j * a.B), 0};
    table_of(a, it[1])[j] = page;
    a.refs[page] = 1;
  }
  if (threadIdx.x == 0) *a.head = PlanHeader{granted, 0};
}

// ---------------------------------------------------------------- compact
__global__ __launch_bounds__(kPlan) void pages_compact_kernel(const PagesArgs a, int max_moves,
                                                              int32_t* __restrict__ info,
                                                              i32x2_t* __restrict__ moves) {
  // The k-th lowest hole takes the k-th highest page in use; as many of those are at n_live and
  // above as there are holes below. `rank`: the page's, from below, among those.
  int n_live = 0, n_holes = 0, n = 0;
  auto place = [&](int id, bool live, int rank) {
    const int k = n_holes - 1 - rank;
    const bool moved = live && k >= 0 && k < n;
    const int to = moved ? a.ids[k] : id;
    a.map[id] = to;
    if (moved) {
      a.copies[k] = i32x4w_t{id, to, a.B, 0};
      moves[k] = i32x2_t{id, to};
      a.refs[to] = a.refs[id];
      a.refs[id] = 0;
    }
  };
  if (a.n_pages <= kPlan * kWalk) {  // one step of a walk: the counts are read once
    const int i0 = (int)threadIdx.x * kWalk;
    const uint32_t live = count_bits<false>(a.refs, i0, a.n_pages);
    int rank = plan_scan(__popc(live), n_live);
    const int below = max(0, min(n_live - i0, kWalk));  // of the thread's pages, below n_live
    uint32_t holes = ~live & ((1u << below) - 1u);
    int at = plan_scan(__popc(holes), n_holes);
    for (; holes; holes &= holes - 1) a.ids[at++] = i0 + __builtin_ctz(holes);
    n = min(n_holes, max_moves);
    __syncthreads();
    rank += __popc(live & ((1u << below) - 1u)) - (n_live - n_holes);
    for (int e = below; e < min(kWalk, a.n_pages - i0); ++e) {
      const bool l = live >> e & 1u;
      place(i0 + e, l, rank);
      rank += l;
    }
  } else {
    for (int base = 0; base < a.n_pages; base += kPlan * kWalk) {  // uniform
      int total;
      plan_scan(__popc(count_bits<false>(a.refs, base + (int)threadIdx.x * kWalk, a.n_pages)),
                total);
      n_live += total;
    }
    n_holes = find_free(a.refs, n_live, n_live, a.ids);
    n = min(n_holes, max_moves);
    __syncthreads();
    int before = 0;
    for (int base = n_live / kWalk * kWalk; base < a.n_pages; base += kPlan * kWalk) {  // uniform
      const int i0 = base + (int)threadIdx.x * kWalk;
      uint32_t bits = count_bits<false>(a.refs, i0, a.n_pages);
      if (i0 < n_live) bits &= ~((1u << (n_live - i0)) - 1u);
      int total;
      int rank = before + plan_scan(__popc(bits), total);
      for (int id = max(i0, n_live); id < min(i0 + kWalk, a.n_pages); ++id) {
        const bool l = bits >> (id - i0) & 1u;
        place(id, l, rank);
        rank += l;
      }
      before += total;
    }
  }
  for (int k = n + (int)threadIdx.x; k < max_moves; k += kPlan) moves[k] = i32x2_t{-1, -1};
  if (threadIdx.x == 0) {
    *a.head = PlanHeader{n, n_live};
    info[0] = n_live;
    info[1] = n;
  }
}

// ---------------------------------------------------------------- the second launch
enum { kTruncate, kFork, kCompact };

// Whether page id is a copy's destination, and so free before the call: they ascend, as the plan
// found them.
__device__ __forceinline__ bool copied_to(const PagesArgs& a, int n_copies, int id) {
  int lo = 0, hi = n_copies;  // the first destination from id on
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.copies[mid][1] < id) lo = mid + 1;
    else hi = mid;
  }
  return lo < n_copies && a.copies[lo][1] == id;
}

// Workgroups x < books of plane 0 change counts and tables; the others copy rows.
template <int OP>
__global__ __launch_bounds__(kCopyThreads) void pages_apply_kernel(
    const PagesArgs a, int n, const int32_t* __restrict__ loose, int n_loose, int share,
    int books) {
  const int n_copies = a.head->n_copies;
  const int x = blockIdx.x;
  if (x < books) {
    if (blockIdx.y) return;
    const int lane = threadIdx.x & 63;
    const int waves = books * (kCopyThreads / 64);
    const int w0 = __builtin_amdgcn_readfirstlane(x * (kCopyThreads / 64) + (threadIdx.x >> 6));
    const int t0 = x * kCopyThreads + threadIdx.x, threads = books * kCopyThreads;
    if constexpr (OP == kTruncate) {
      for (int i = w0; i < n; i += waves) {
        const i32x4w_t it = a.items[i];  // {row, pages that stay, pages before}
        if (it[0] < 0) continue;
        int32_t* bt = table_of(a, it[0]);
        for (int j = it[1] + lane; j < it[2]; j += 64) {
          drop_ref(a, bt[j]);
          bt[j] = -1;
        }
      }
      for (int k = t0; k < n_copies; k += threads) drop_ref(a, a.copies[k][0]);
      for (int k = t0; k < n_loose; k += threads)
        if (loose[k] != -1 && !copied_to(a, n_copies, loose[k])) drop_ref(a, loose[k]);
    } else if constexpr (OP == kFork) {
      if (!share) return;
      for (int i = w0; i < n; i += waves) {
        const i32x4w_t it = a.items[i];  // {parent, child, length}
        if (it[0] < 0) continue;
        const int32_t* from = table_of(a, it[0]);
        int32_t* to = table_of(a, it[1]);
        for (int j = lane; j < it[2] / a.B; j += 64) {
          const int id = from[j];
          to[j] = id;
          if (page_ok(a, id)) atomicAdd(&a.refs[id], 1);
        }
      }
    } else {
      const int n_live = a.head->n_live;
      if (n_copies == 0) return;
      for (int r = w0; r < a.n_rows; r += waves) {
        int32_t* bt = table_of(a, r);
        for (int j = lane; j < a.max_blocks; j += 64) {
          const int id = bt[j];
          if (id >= n_live && id < a.n_pages) {
            const int to = a.map[id];
            if (to != id) bt[j] = to;
          }
        }
      }
    }
    return;
  }
  const int64_t page_bytes = (int64_t)a.B * a.row_bytes;
  const int chunks = (int)((page_bytes + kCopyBytes - 1) / kCopyBytes);
  char* plane = a.kv + (int64_t)blockIdx.y * a.n_pages * page_bytes;
  const int64_t units = (int64_t)n_copies * chunks;
  for (int64_t u = x - books; u < units; u += (int)gridDim.x - books) {
    const int k = (int)(u / chunks);
    const i32x4w_t c = a.copies[k];
    if (!page_ok(a, c[0])) continue;
    const int64_t at = (u - (int64_t)k * chunks) * kCopyBytes + (int)threadIdx.x * 16;
    const int64_t bytes = (int64_t)c[2] * a.row_bytes;
    const char* src = plane + c[0] * page_bytes;
    char* dst = plane + c[1] * page_bytes;
    u32x4_t v[kCopyUnroll];
#pragma unroll
    for (int e = 0; e < kCopyUnroll; ++e) {
      const int64_t o = at + e * (kCopyThreads * 16);
      if (o < bytes) v[e] = *reinterpret_cast<const u32x4_t*>(src + o);
    }
#pragma unroll
    for (int e = 0; e < kCopyUnroll; ++e) {
      const int64_t o = at + e * (kCopyThreads * 16);
      if (o < bytes) __builtin_nontemporal_store(v[e], reinterpret_cast<u32x4_t*>(dst + o));
    }
  }
}

static int pages_check(const nkv_pages* p, const char* what, PagesArgs& a) {
  NKV_REQUIRE(p, NKV_EINVAL, "%s: null arguments", what);
  NKV_REQUIRE(p->n_planes > 0 && p->n_pages > 0 && p->block_size > 0 && p->row_bytes > 0 &&
                  p->max_blocks > 0 && p->n_rows > 0 && p->bt_row_stride >= p->max_blocks,
              NKV_EINVAL, "%s: bad sizes", what);
  NKV_REQUIRE(p->row_bytes % 16 == 0, NKV_EUNSUPPORTED,
              "%s: rows must be a multiple of 16 bytes (got %lld)", what,
              (long long)p->row_bytes);
  NKV_REQUIRE(p->n_rows <= kMaxList && p->n_pages <= kMaxPages && p->n_planes <= 65535,
              NKV_EUNSUPPORTED, "%s: at most %d rows, %d pages and 65535 planes", what, kMaxList,
              kMaxPages);
  NKV_REQUIRE(p->block_size <= INT32_MAX / p->n_pages && p->max_blocks <= INT32_MAX &&
                  p->block_size <= INT32_MAX / p->max_blocks && p->row_bytes <= INT32_MAX,
              NKV_EUNSUPPORTED, "%s: slots and lengths must fit 32 bits", what);
  NKV_REQUIRE(p->kv_cache && p->ref_counts && p->context_lens && p->block_tables, NKV_EINVAL,
              "%s: null pointer", what);
  NKV_REQUIRE(aligned16(p->kv_cache) && aligned16(p->ref_counts), NKV_EINVAL,
              "%s: kv_cache and ref_counts must be 16-byte aligned", what);
  const size_t need = pages_ws_bytes(p->n_pages);
  NKV_REQUIRE(p->workspace && aligned16(p->workspace) && p->workspace_bytes >= (int64_t)need,
              NKV_EWORKSPACE, "%s: workspace needs %zu bytes, 16-byte aligned", what, need);
  char* ws = static_cast<char*>(p->workspace);
  a.kv = static_cast<char*>(p->kv_cache);
  a.n_planes = (int32_t)p->n_planes;
  a.n_pages = (int32_t)p->n_pages;
  a.B = (int32_t)p->block_size;
  a.row_bytes = (int32_t)p->row_bytes;
  a.refs = p->ref_counts;
  a.lens = p->context_lens;
  a.tables = p->block_tables;
  a.bt_stride = p->bt_row_stride;
  a.max_blocks = (int32_t)p->max_blocks;
  a.n_rows = (int32_t)p->n_rows;
  a.head = reinterpret_cast<PlanHeader*>(ws);
  a.items = reinterpret_cast<i32x4w_t*>(ws + kHeaderBytes);
  a.copies = a.items + kMaxList;
  a.ids = reinterpret_cast<int32_t*>(a.copies + p->n_pages);
  a.map = a.ids + p->n_pages;
  return NKV_OK;
}

static size_t plan_lds(const PagesArgs& a, int32_t n) {
  return sizeof(int) * (size_t)std::max(a.n_rows, n);
}

// The second launch: at most `copies` pages, the bookkeeping of `entries` rows or list entries.
template <int OP>
static int pages_apply(const PagesArgs& a, int32_t n, const int32_t* loose, int32_t n_loose,
                       int32_t share, int64_t entries, int64_t copies, void* stream) {
  const int books = (int)std::min<int64_t>(kBookGroups, (entries + 3) / 4);
  const int64_t page_bytes = (int64_t)a.B * a.row_bytes;
  const int64_t units = copies * ((page_bytes + kCopyBytes - 1) / kCopyBytes);
  const int64_t groups = std::max<int64_t>(
      1, std::min<int64_t>(units, std::max(1, kCopyGroups / a.n_planes)));
  hipLaunchKernelGGL((pages_apply_kernel<OP>),
                     dim3((unsigned)(books + groups), (unsigned)a.n_planes), dim3(kCopyThreads),
                     0, as_stream(stream), a, n, loose, n_loose, share, books);
  return check_launch("nkv_pages");
}

}  // namespace nkv

extern "C" size_t nkv_pages_workspace_bytes(int64_t n_pages) {
  return n_pages > 0 && n_pages <= nkv::kMaxPages ? nkv::pages_ws_bytes(n_pages) : 0;
}

extern "C" int nkv_pages_append(const nkv_pages* pages, const int32_t* rows, int32_t n,
                                const int32_t* cu_seqlens_q, int64_t n_tokens,
                                int32_t* slot_mapping, int32_t* status, void* stream) {
  using namespace nkv;
  clear_error();
  PagesArgs a;
  int rc = pages_check(pages, "pages_append", a);
  if (rc) return rc;
  NKV_REQUIRE(n >= 0 && n <= kMaxList && n_tokens >= 0 && n_tokens < (1ll << 31), NKV_EINVAL,
              "pages_append: 0 to %d rows and fewer than 2^31 tokens (got %d, %lld)", kMaxList, n,
              (long long)n_tokens);
  NKV_REQUIRE(cu_seqlens_q || n_tokens == n, NKV_EINVAL,
              "pages_append: without cu_seqlens_q one token a row (%d rows, %lld tokens)", n,
              (long long)n_tokens);
  NKV_REQUIRE((n == 0 || (rows && status)) && (n_tokens == 0 || slot_mapping), NKV_EINVAL,
              "pages_append: null pointer");
  if (n > 0) {
    hipLaunchKernelGGL(pages_append_kernel, dim3(1), dim3(kPlan), plan_lds(a, n),
                       as_stream(stream), a, rows, n, cu_seqlens_q, n_tokens, slot_mapping,
                       status);
    rc = check_launch("nkv_pages_append");
    if (rc) return rc;
  }
  if (cu_seqlens_q && n_tokens > 0) {
    hipLaunchKernelGGL(pages_slots_kernel, dim3((unsigned)((n_tokens + 255) / 256)), dim3(256), 0,
                       as_stream(stream), a, n, cu_seqlens_q, n_tokens, slot_mapping);
    rc = check_launch("nkv_pages_append");
  }
  return rc;
}

extern "C" int nkv_pages_truncate(const nkv_pages* pages, const int32_t* rows,
                                  const int32_t* keep_lens, int32_t n, const int32_t* page_ids,
                                  int64_t n_page_ids, int32_t* status, void* stream) {
  using namespace nkv;
  clear_error();
  PagesArgs a;
  int rc = pages_check(pages, "pages_truncate", a);
  if (rc) return rc;
  NKV_REQUIRE(n >= 0 && n <= kMaxList && n_page_ids >= 0 && n_page_ids < (1 << 30), NKV_EINVAL,
              "pages_truncate: 0 to %d rows (got %d) and fewer than 2^30 page ids", kMaxList, n);
  NKV_REQUIRE((n == 0 || (rows && keep_lens && status)) && (n_page_ids == 0 || page_ids),
              NKV_EINVAL, "pages_truncate: null pointer");
  if (n == 0 && n_page_ids == 0) return NKV_OK;
  hipLaunchKernelGGL(pages_truncate_kernel, dim3(1), dim3(kPlan), plan_lds(a, n),
                     as_stream(stream), a, rows, keep_lens, n, status);
  rc = check_launch("nkv_pages_truncate");
  if (rc) return rc;
  return pages_apply<kTruncate>(a, n, page_ids, (int32_t)n_page_ids, 0,
                                std::max<int64_t>(n, (n_page_ids + 63) / 64), n, stream);
}

extern "C" int nkv_pages_fork(const nkv_pages* pages, const int32_t* parents,
                              const int32_t* children, int32_t n, int32_t share_pages,
                              int32_t* status, void* stream) {
  using namespace nkv;
  clear_error();
  PagesArgs a;
  int rc = pages_check(pages, "pages_fork", a);
  if (rc) return rc;
  NKV_REQUIRE(n >= 0 && n <= kMaxList, NKV_EINVAL, "pages_fork: 0 to %d rows (got %d)", kMaxList,
              n);
  if (n == 0) return NKV_OK;
  NKV_REQUIRE(parents && children && status, NKV_EINVAL, "pages_fork: null pointer");
  hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(kPlan), plan_lds(a, n), as_stream(stream),
                     a, parents, children, n, share_pages ? 1 : 0, status);
  rc = check_launch("nkv_pages_fork");
  if (rc) return rc;
  return pages_apply<kFork>(a, n, nullptr, 0, share_pages ? 1 : 0, n,
                            share_pages ? n
                                        : std::min<int64_t>(a.n_pages, (int64_t)n * a.max_blocks),
                            stream);
}

extern "C" int nkv_pages_compact(const nkv_pages* pages, int32_t max_moves, int32_t* info,
                                 int32_t* moves, void* stream) {
  using namespace nkv;
  clear_error();
  PagesArgs a;
  int rc = pages_check(pages, "pages_compact", a);
  if (rc) return rc;
  // the loop that pads the list counts in 32 bits
  NKV_REQUIRE(max_moves >= 0 && max_moves <= kMaxPages, NKV_EINVAL,
              "pages_compact: max_moves must be 0 to %d (got %d)", kMaxPages, max_moves);
  NKV_REQUIRE(info && (max_moves == 0 || moves) &&
                  (reinterpret_cast<uintptr_t>(moves) & 7u) == 0,
              NKV_EINVAL, "pages_compact: info and 8-byte aligned moves are needed");
  hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kPlan), 0, as_stream(stream), a,
                     max_moves, info, reinterpret_cast<i32x2_t*>(moves));
  rc = check_launch("nkv_pages_compact");
  if (rc) return rc;
  return pages_apply<kCompact>(a, a.n_rows, nullptr, 0, 0, a.n_rows,
                               std::min(max_moves, a.n_pages), stream);
}
