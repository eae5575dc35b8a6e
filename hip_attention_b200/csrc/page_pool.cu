// The pages of a pool: writing new keys and values into them, dealing them out, sharing, freeing and moving them.
//
// Which pages are free is read off the reference counts themselves: there is no list beside them that could disagree, and
// "the lowest free pages in the order of the entries" does not depend on how threads are scheduled.  A call is planned by one
// CTA, or a cluster (the counts are cut into runs, whose sums its CTAs exchange through distributed shared memory), which
// also changes the tables; pages are copied by a second launch over the whole GPU that the plan is handed to in device memory.
#include "in_turn.cuh"

namespace hipattn {
namespace {

constexpr int kSMs = 148;
constexpr int kPlanCtas = 8;           // of a cluster; one CTA plans for pools of up to kSmallPool pages (a few sequences freed and dealt out of 4096
constexpr int kSmallPool = 8192;       // pages: 7.1 us, 8.6 by a cluster; of 8192 7.7 and 8.6; of 16000 8.5 and 7.7, of 30000 11.0 and 7.7)
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kMaxCachesPerLaunch = 128;

struct Pool {
  int32_t* refs;
  int32_t* lens;
  int32_t* table;
  uint32_t* status;
  int32_t* grown;      // extend, or null: its rows, -1 where nothing grew
  int n_pages, page_size, n_seqs, width;
};
// (not n + P - 1 over P: the longest length and a page of more than 65537 tokens pass 2^31)
__device__ __forceinline__ int pages_of(int n, int P) { return n / P + (n % P != 0); }
struct CacheList {
  char* at[kMaxCachesPerLaunch];
  int n;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void plan_sync(int ctas) {
  if (ctas > 1) cluster_sync();
  else __syncthreads();
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int ld_cluster_int(const int* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Sums over the threads of a CTA: those before this thread (returned) and all (`all`).  s: kPlanWarps words.
template <typename N>
__device__ __forceinline__ N scan_block(N x, N* s, N& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  __syncthreads();
  if (lane == 31) s[warp] = sum;
  __syncthreads();
  N w = lane < kPlanWarps ? s[lane] : 0, ws = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, ws, o);
    if (lane >= o) ws += y;
  }
  all = __shfl_sync(0xffffffffu, ws, 31);
  return sum - x + __shfl_sync(0xffffffffu, ws - w, warp);
}

// The reference counts are cut into runs of `loads` times 128 consecutive pages, at most kMaxRuns, which the warps of the cluster take in
// turn (run q: CTA q % ctas), so that the pages dealt out, which lie at the front, are spread over all of them.  A lane reads four
// consecutive pages at a time.
constexpr int kMaxRuns = 2048;
struct Runs {
  int n_pages, loads, count;
};
__device__ __forceinline__ Runs runs_of(int n_pages) {
  Runs r;
  r.n_pages = n_pages;
  r.loads = (int)(((int64_t)n_pages + 128 * kMaxRuns - 1) / (128 * kMaxRuns));
  r.count = (int)(((int64_t)n_pages + 128 * r.loads - 1) / (128 * r.loads));
  return r;
}
// bit i: page `at` + i is in use / is there
__device__ __forceinline__ uint32_t live_pages(const int32_t* refs, int64_t at, int n) {
  if (at + 4 <= n && ((uintptr_t)(refs + at) & 15) == 0) {
    const int4 r = *reinterpret_cast<const int4*>(refs + at);
    return (uint32_t)((r.x > 0) | (r.y > 0) << 1 | (r.z > 0) << 2 | (r.w > 0) << 3);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < n && refs[at + i] > 0) m |= 1u << i;
  return m;
}
__device__ __forceinline__ uint32_t there_pages(int64_t at, int64_t n) { return at >= n ? 0u : (at + 4 <= n ? 15u : (1u << (int)(n - at)) - 1u); }

// Live pages of this warp's runs into s_count
__device__ __forceinline__ void count_runs(const int32_t* refs, const Runs& runs, int rank, int ctas, int* s_count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int q = rank + warp * ctas; q < runs.count; q += ctas * kPlanWarps) {
    int n = 0;
    for (int j = 0; j < runs.loads; ++j) n += __popc(live_pages(refs, ((int64_t)q * runs.loads + j) * 128 + lane * 4, runs.n_pages));
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_count[q / ctas] = n;
  }
}
// Between two barriers (the counts are written; nobody leaves before they are read): the live pages before every run, and in all
__device__ __forceinline__ int gather_runs(const Runs& runs, int ctas, const int* s_count, int* s_before, int* s_scan) {
  const int q = threadIdx.x * 2;
  auto count = [&](int i) { return i >= runs.count ? 0 : (ctas > 1 ? ld_cluster_int(s_count + i / ctas, i % ctas) : s_count[i]); };
  const int x = count(q), y = count(q + 1);
  int all;
  const int before = scan_block(x + y, s_scan, all);
  s_before[q] = before;
  s_before[q + 1] = before + x;
  __syncthreads();
  return all;
}
static_assert(kMaxRuns == 2 * kPlanThreads, "two runs to a thread");
static_assert(kSmallPool / 128 <= kMaxRuns / kPlanCtas, "the runs of a small pool fit into one CTA's counts");

// Sum over the lanes before this one
__device__ __forceinline__ int scan_warp(int x) {
  int sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) >= o) sum += y;
  }
  return sum - x;
}

// ---------------------------------------------------------------------------------------------------
// extend and fork
// ---------------------------------------------------------------------------------------------------
// A copied page: source, destination, tokens
struct PageCopy {
  int src, dst, tokens;
};

// extend: a[i] = row, b[i] (b null: every) = tokens that it grows by.  fork: a[i] = parent, b[i] = child.
// plan (fork): [0] = number of copies, then PageCopy[].
template <bool FORK>
__global__ void __launch_bounds__(kPlanThreads, 1)
    deal_pages_kernel(const Pool pool, const int32_t* a, const int32_t* b, int every, int n, int32_t* plan, int ctas) {
  extern __shared__ __align__(16) unsigned char smem[];
  int* s_row = reinterpret_cast<int*>(smem);        // row that gets pages, -1: none
  int* s_had = s_row + n;                           // pages that it has (fork: full pages of the parent)
  int* s_new = s_had + n;                           // its new length
  int* s_before = s_new + n;                        // pages that the entries before it get
  uint32_t* s_named = reinterpret_cast<uint32_t*>(s_before + n);   // rows that the call names
  __shared__ long long s_scan64[kPlanWarps];
  __shared__ int s_scan[kPlanWarps];
  __shared__ int s_longest, s_count[kMaxRuns / kPlanCtas], s_live[kMaxRuns], s_dealt[kPlanWarps][128];
  const int tid = threadIdx.x, rank = blockIdx.x, P = pool.page_size;
  in_turn();

  const Runs runs = runs_of(pool.n_pages);
  const int per = (n + kPlanThreads - 1) / kPlanThreads;   // consecutive entries of a thread
  const int x0 = tid * per < n ? a[tid * per] : -1, y0 = tid * per < n && b ? b[tid * per] : every;     // (on their way with the counts)
  for (int i = tid; i < (pool.n_seqs + 31) / 32; i += kPlanThreads) s_named[i] = 0;
  if (tid == 0) s_longest = 0;
  count_runs(pool.refs, runs, rank, ctas, s_count);
  __syncthreads();
  // ---- the entries: every CTA goes through all of them ----
  bool bad = false;
  long long mine = 0;
  for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) {
    const int x = i == tid * per ? x0 : a[i], y = i == tid * per ? y0 : (b ? b[i] : every), row = FORK ? y : x;
    int had = 0, len = 0, need = 0, at = -1;
    if (x >= 0 && row >= 0) {
      if (x >= pool.n_seqs || row >= pool.n_seqs || (!FORK && y < 0) || (atomicOr(&s_named[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u)) {
        bad = true;
      } else {
        const int old = pool.lens[x];
        const long long now = FORK ? old : (long long)old + y;
        if (old < 0 || now > 0x7fff0000LL || (FORK && pool.lens[row] != 0) || pages_of((int)now, P) > pool.width) {
          bad = true;
        } else {
          len = (int)now;
          had = FORK ? len / P : pages_of(old, P);
          need = pages_of(len, P) - had;
          at = row;
          if (FORK) atomicMax(&s_longest, had);
        }
      }
    }
    s_row[i] = at;
    s_had[i] = had;
    s_new[i] = len;
    s_before[i] = need;
    mine += need;
  }
  long long total;
  long long before = scan_block(mine, s_scan64, total);
  for (int i = tid * per; i < min(n, (tid + 1) * per); ++i) {
    const int need = s_before[i];
    s_before[i] = (int)min(before, (long long)0x7fffffff);
    before += need;
  }
  bad = __syncthreads_or(bad);

  // ---- free pages, and those before every run ----
  plan_sync(ctas);
  const int free_pages = pool.n_pages - gather_runs(runs, ctas, s_count, s_live, s_scan);
  plan_sync(ctas);   // (everybody has read the lengths and the sums: from here on they may change, and CTAs may leave)
  if (bad || total > free_pages) {
    if (rank == 0 && tid == 0) {
      atomicOr(pool.status, bad ? HIPATTN_STATUS_SEQUENCE : HIPATTN_STATUS_NO_PAGES);
      if (FORK) plan[0] = 0;
    }
    if (!FORK && rank == 0 && pool.grown)
      for (int i = tid; i < n; i += kPlanThreads) pool.grown[i] = -1;
    return;
  }

  // ---- deal out the free pages of the runs: a warp brings 128 pages' free ones into order, then consecutive lanes take consecutive ones.
  // (a million pages of which 36000 are dealt out: 325 us, frees included, with a thread to consecutive pages, 24 so) ----
  const int warp = tid >> 5, lane = tid & 31;
  for (int q = rank + warp * ctas; q < runs.count; q += ctas * kPlanWarps) {
    int64_t at = (int64_t)q * runs.loads * 128;
    int64_t nth = at - s_live[q];             // free pages before
    for (int j = 0; j < runs.loads && nth < total; ++j, at += 128) {
      uint32_t f = ~live_pages(pool.refs, at + lane * 4, pool.n_pages) & there_pages(at + lane * 4, pool.n_pages);
      int k = scan_warp(__popc(f));
      const int found = __shfl_sync(0xffffffffu, k + __popc(f), 31), count = (int)min((long long)found, total - (long long)nth);
      for (; f; f &= f - 1) s_dealt[warp][k++] = (int)at + lane * 4 + __ffs(f) - 1;
      __syncwarp();
      int entry = 0, end = 0;                 // the entry of the warp's last page, and where it ends: the next pages are most often its too
      for (int i = lane; i < count; i += 32) {
        const int page = s_dealt[warp][i], to = (int)nth + i;
        if (to >= end) {
          int lo = entry, hi = n - 1;         // the last entry that begins at or before `to`
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_before[mid] <= to) lo = mid;
            else hi = mid - 1;
          }
          entry = lo;
          end = lo + 1 < n ? s_before[lo + 1] : 0x7fffffff;
        }
        pool.refs[page] = 1;
        pool.table[(int64_t)s_row[entry] * pool.width + s_had[entry] + (to - s_before[entry])] = page;
        if (FORK) {
          int src = pool.table[(int64_t)a[entry] * pool.width + s_had[entry]];
          int tokens = s_new[entry] - s_had[entry] * P;
          if (src < 0 || src >= pool.n_pages) {
            atomicOr(pool.status, HIPATTN_STATUS_PAGE_RANGE);
            src = page;
            tokens = 0;
          }
          reinterpret_cast<PageCopy*>(plan + 1)[to] = PageCopy{src, page, tokens};
        }
      }
      __syncwarp();
      nth += found;
    }
  }
  if (FORK) {
    // ---- full pages are shared: 128 entries of a table at a time ----
    const int chunks = (s_longest + 127) / 128;
    for (int64_t it = rank * kPlanWarps + warp; it < (int64_t)chunks * n; it += ctas * kPlanWarps) {
      const int i = (int)(it % n), j0 = (int)(it / n) * 128 + lane;
      if (s_row[i] < 0) continue;
      const int32_t* from = pool.table + (int64_t)a[i] * pool.width;
      int32_t* to = pool.table + (int64_t)s_row[i] * pool.width;
      int page[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) page[k] = j0 + k * 32 < s_had[i] ? from[j0 + k * 32] : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (j0 + k * 32 < s_had[i]) {
          to[j0 + k * 32] = page[k];
          if (page[k] >= 0 && page[k] < pool.n_pages) atomicAdd(pool.refs + page[k], 1);
          else atomicOr(pool.status, HIPATTN_STATUS_PAGE_RANGE);
        }
      }
    }
  }
  if (rank == 0) {
    for (int i = tid; i < n; i += kPlanThreads) {
      if (s_row[i] >= 0) pool.lens[s_row[i]] = s_new[i];
      if (!FORK && pool.grown) pool.grown[i] = s_row[i];
    }
    if (FORK && tid == 0) plan[0] = (int)total;
  }
}

// ---------------------------------------------------------------------------------------------------
// copies of pages
// ---------------------------------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 16384;     // of a page, to a CTA at a time: four 16-byte pieces a thread in flight (begun pages of 96 beams in
                                      // 32 caches, 768 MB in and out: 121 us, 6.35 TB/s; 398 MB moved: 137 us, 5.8)

__device__ __forceinline__ void copy_piece(const char* src, char* dst, int64_t bytes) {
  uint4 v[kCopyBytes / 16 / kCopyThreads];
#pragma unroll
  for (int k = 0; k < kCopyBytes / 16 / kCopyThreads; ++k) {
    const int o = (k * kCopyThreads + threadIdx.x) * 16;
    if (o < bytes) v[k] = *reinterpret_cast<const uint4*>(src + o);
  }
#pragma unroll
  for (int k = 0; k < kCopyBytes / 16 / kCopyThreads; ++k) {
    const int o = (k * kCopyThreads + threadIdx.x) * 16;
    if (o < bytes) *reinterpret_cast<uint4*>(dst + o) = v[k];
  }
}

// The begun pages of a fork
__global__ void __launch_bounds__(kCopyThreads) copy_begun_pages_kernel(const CacheList caches, const int32_t* plan, int64_t page_stride, int64_t token_bytes,
                                                                        int pieces) {
  in_turn();
  const int count = plan[0];
  const PageCopy* copies = reinterpret_cast<const PageCopy*>(plan + 1);
  for (int64_t it = blockIdx.x; it < (int64_t)count * caches.n * pieces; it += gridDim.x) {
    const int piece = (int)(it % pieces);
    const int cache = (int)(it / pieces % caches.n);
    const PageCopy c = copies[it / pieces / caches.n];
    const int64_t at = (int64_t)piece * kCopyBytes, bytes = c.tokens * token_bytes - at;
    if (bytes > 0) copy_piece(caches.at[cache] + c.src * page_stride + at, caches.at[cache] + c.dst * page_stride + at, bytes);
  }
}

// ---------------------------------------------------------------------------------------------------
// free
// ---------------------------------------------------------------------------------------------------
// One cluster per row.  Its first CTA takes the length and leaves 0, so that a row that is named twice is freed once.
__global__ void __launch_bounds__(256) free_rows_kernel(const Pool pool, const int32_t* rows, int ctas) {
  __shared__ int s_len;
  in_turn();
  const int rank = ctas > 1 ? cluster_rank() : 0;
  const int row = rows[blockIdx.x / ctas];
  const bool there = row >= 0 && row < pool.n_seqs;
  if (threadIdx.x == 0 && rank == 0) {
    s_len = there ? atomicExch(pool.lens + row, 0) : 0;
    if (row >= pool.n_seqs) atomicOr(pool.status, HIPATTN_STATUS_SEQUENCE);
  }
  int len;
  if (ctas > 1) {
    cluster_sync();
    len = ld_cluster_int(&s_len, 0);
    cluster_sync();
  } else {
    __syncthreads();
    len = s_len;
  }
  const int64_t pages = min(((int64_t)max(len, 0) + pool.page_size - 1) / pool.page_size, (int64_t)pool.width);
  for (int64_t i = (int64_t)rank * 256 + threadIdx.x; i < pages; i += 256 * ctas) {
    const int page = pool.table[(int64_t)row * pool.width + i];
    if (page < 0 || page >= pool.n_pages) atomicOr(pool.status, HIPATTN_STATUS_PAGE_RANGE);
    else atomicSub(pool.refs + page, 1);
  }
}

// ---------------------------------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------------------------------
// plan: [0] = pages that move, [1] = pages in use, then holes [half], movers [half], nth [n_pages] (which mover a page is)
struct CompactPlan {
  int32_t *count, *holes, *movers, *nth;
};
__host__ __device__ __forceinline__ int64_t half_of(int64_t n) { return n / 2 + 1; }
__host__ __device__ __forceinline__ CompactPlan compact_plan(int32_t* scratch, int n_pages) {
  CompactPlan c;
  c.count = scratch;
  c.holes = scratch + 2;
  c.movers = c.holes + half_of(n_pages);
  c.nth = c.movers + half_of(n_pages);
  return c;
}

__global__ void __launch_bounds__(kPlanThreads, 1) plan_compact_kernel(const Pool pool, int32_t* scratch, int32_t* in_use, int ctas) {
  __shared__ int s_scan[kPlanWarps];
  __shared__ int s_count[kMaxRuns / kPlanCtas], s_live[kMaxRuns], s_part;
  in_turn();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x;
  const CompactPlan plan = compact_plan(scratch, pool.n_pages);
  const Runs runs = runs_of(pool.n_pages);
  count_runs(pool.refs, runs, rank, ctas, s_count);
  plan_sync(ctas);
  const int m = gather_runs(runs, ctas, s_count, s_live, s_scan);     // pages in use
  plan_sync(ctas);
  // ---- of them, numbered below m: those before m's run, and those of the run ----
  const int run_pages = runs.loads * 128, qm = min(m / run_pages, runs.count - 1);
  if (warp == 0) {
    int n = 0;
    for (int j = 0; j < runs.loads; ++j) {
      const int64_t at = (int64_t)qm * run_pages + j * 128 + lane * 4;
      n += __popc(live_pages(pool.refs, at, pool.n_pages) & there_pages(at, m));
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_part = n;
  }
  __syncthreads();
  const int stay = s_live[qm] + s_part;
  if (rank == 0 && tid == 0) {
    plan.count[0] = m - stay;
    plan.count[1] = m;
    if (in_use) *in_use = m;
  }
  if (stay == m) return;
  for (int q = rank + warp * ctas; q < runs.count; q += ctas * kPlanWarps) {
    int lower = s_live[q];           // pages in use below the next 128
    for (int j = 0; j < runs.loads; ++j) {
      const int64_t at = (int64_t)q * run_pages + j * 128 + lane * 4;
      const uint32_t live = live_pages(pool.refs, at, pool.n_pages), below = there_pages(at, m);
      const int before = lower + scan_warp(__popc(live));
      // holes below m: the page's number less the pages in use below it; movers at m and beyond: that less those that stay
      for (uint32_t pick = (~live & below) | (live & ~below); pick; pick &= pick - 1) {
        const int i = __ffs(pick) - 1, page = (int)at + i, k = before + __popc(live & ((1u << i) - 1u));
        if (page < m) {
          plan.holes[page - k] = page;
        } else {
          plan.movers[k - stay] = page;
          plan.nth[page] = k - stay;
        }
      }
      lower += __reduce_add_sync(0xffffffffu, __popc(live));
    }
  }
}

// Pages, counts and (first launch) tables
__global__ void __launch_bounds__(kCopyThreads) move_pages_kernel(const Pool pool, const CacheList caches, int32_t* scratch, int64_t page_stride, int64_t page_bytes,
                                                                  int pieces, int tables) {
  in_turn();
  const CompactPlan plan = compact_plan(scratch, pool.n_pages);
  const int moves = plan.count[0], m = plan.count[1];
  if (moves == 0) return;
  if (tables) {
    const int64_t thread = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x, threads = (int64_t)gridDim.x * kCopyThreads;
    for (int64_t i = thread; i < moves; i += threads) {
      pool.refs[plan.holes[i]] = pool.refs[plan.movers[i]];
      pool.refs[plan.movers[i]] = 0;
    }
    // a warp takes 32 entries of a row
    const int chunks = (pool.width + 31) / 32, lane = threadIdx.x & 31;
    for (int64_t it = thread >> 5; it < (int64_t)pool.n_seqs * chunks; it += threads >> 5) {
      const int row = (int)(it / chunks), j = (int)(it % chunks) * 32 + lane;
      const int64_t pages = ((int64_t)max(pool.lens[row], 0) + pool.page_size - 1) / pool.page_size;
      if (j >= pool.width || j >= pages) continue;
      int32_t* e = pool.table + (int64_t)row * pool.width + j;
      const int page = *e;
      if (page < 0 || page >= pool.n_pages) {
        atomicOr(pool.status, HIPATTN_STATUS_PAGE_RANGE);
      } else if (page >= m) {
        // (a table that names a page which the counts call free: the list of the movers does not have it)
        const int k = plan.nth[page];
        if (k >= 0 && k < moves && plan.movers[k] == page) *e = plan.holes[k];
        else atomicOr(pool.status, HIPATTN_STATUS_PAGE_RANGE);
      }
    }
  }
  for (int64_t it = blockIdx.x; it < (int64_t)moves * caches.n * pieces; it += gridDim.x) {
    const int piece = (int)(it % pieces);
    const int cache = (int)(it / pieces % caches.n);
    const int64_t i = it / pieces / caches.n, at = (int64_t)piece * kCopyBytes;
    copy_piece(caches.at[cache] + plan.movers[i] * page_stride + at, caches.at[cache] + plan.holes[i] * page_stride + at, page_bytes - at);
  }
}

// ---------------------------------------------------------------------------------------------------
// new keys and values
// ---------------------------------------------------------------------------------------------------
// Eight 16-bit values as e5m2, nearest, ties to even.  An e5m2 number is the upper byte of a half-precision one, so what is dropped
// is rounded in integers: half a step less one, and one more where the byte is odd.  Subnormal numbers and the step to infinity
// need nothing of their own; NaN keeps its top bit.  A bfloat16 value goes through half precision unharmed: that rounds only values
// below 2^-17, which e5m2 makes zero either way (2^-17 itself is a tie), and those beyond 65504, which are infinite either way.
template <int DT>
__device__ __forceinline__ uint2 narrow_e5m2(const uint4& w) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h = v[i];
    if (DT == HIPATTN_BF16) h = pack2<HIPATTN_F16>(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
    const __half2 x = *reinterpret_cast<const __half2*>(&h);
    const uint32_t nan = __hneu2_mask(x, x);
    h = (h & ~nan) | (nan & 0x7e007e00u);
    o[i] = h + 0x007f007fu + ((h >> 8) & 0x00010001u);
  }
  return make_uint2(__byte_perm(o[0], o[1], 0x7531), __byte_perm(o[2], o[3], 0x7531));
}

// A CTA writes `span` consecutive tokens: their slots are looked up once, by one thread each, while the first rows are on their way.  A
// thread keeps its place in the row (keys or values, head, elements) and goes from token to token, `lanes` threads to a token.
// Bound: HBM; 17600 tokens of 8 KV heads into an fp8 pool (108 MB): 109 us with a thread to a piece, which looked everything up for itself
// and rounded by way of the library's conversion, 22 so.  A step's 32 tokens: 2.6 us.
constexpr int kWriteThreads = 256;
constexpr int kMaxSpan = 32;
constexpr int kWriteAhead = 4;    // 16-byte pieces of a thread in flight
template <int DT, bool F8>
__global__ void __launch_bounds__(kWriteThreads) write_kv_kernel(const hipattn_write_kv_params_t p, int span, int lanes) {
  constexpr int EB = Elem<DT>::bytes, VEC = 16 / EB, CB = F8 ? 1 : EB;
  __shared__ int s_page[kMaxSpan], s_off[kMaxSpan];
  in_turn();
  const int row_pieces = p.D / VEC, pieces = p.HKV * row_pieces;       // of a token, keys or values
  const int64_t tok0 = (int64_t)blockIdx.x * span;
  const int tokens = (int)min((int64_t)span, p.N - tok0);
  const int groups = kWriteThreads / lanes, group = threadIdx.x / lanes;
  int i = threadIdx.x % lanes;      // piece of a token: keys, then values
  const char* src = nullptr;
  char* dst = nullptr;
  int64_t step = 0, page_step = 0, off_step = 0;      // bytes
  auto place = [&]() {
    const int which = i >= pieces, pc = i - which * pieces, h = pc / row_pieces, d = (pc - h * row_pieces) * VEC;
    const hipattn_tokens_t& pool = which ? p.v_pool : p.k_pool;
    step = (which ? p.v_stride_t : p.k_stride_t) * EB;
    src = (const char*)(which ? p.v : p.k) + ((int64_t)h * (which ? p.v_stride_h : p.k_stride_h) + d) * EB + tok0 * step;
    dst = (char*)pool.cache + ((int64_t)h * pool.stride_ch + d) * CB;
    page_step = pool.stride_page * CB;
    off_step = pool.stride_off * CB;
  };
  uint4 x[kWriteAhead];
  auto load = [&](int tok, uint4& to) {
    if (i < 2 * pieces && tok < tokens) to = __ldcs(reinterpret_cast<const uint4*>(src + tok * step));
  };
  if (i < 2 * pieces) place();
#pragma unroll
  for (int k = 0; k < kWriteAhead; ++k) load(group + k * groups, x[k]);

  if (threadIdx.x < tokens) {
    auto index = [](const void* q, int is64, int64_t i) { return is64 ? (int64_t)__ldcg((const long long*)q + i) : (int64_t)__ldcg((const int*)q + i); };
    const int64_t tok = tok0 + threadIdx.x;
    int page = -1, off = 0;                  // -1: not written
    // the token's sequence and place in it
    int64_t first = 0, count = 0;
    int b = -1;
    if (p.offsets) {
      int lo = 0, hi = p.B;                  // the first b with tok < offsets[b + 1]
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (index(p.offsets, p.offsets_is_i64, mid + 1) <= tok) lo = mid + 1;
        else hi = mid;
      }
      if (lo < p.B) {                        // (else: behind the last sequence)
        first = index(p.offsets, p.offsets_is_i64, lo);
        count = index(p.offsets, p.offsets_is_i64, lo + 1) - first;
        if (tok >= first) b = lo;            // (else: before the first)
      }
    } else {
      count = p.N / p.B;
      b = (int)(tok / count);
      first = b * count;
    }
    const int64_t row = b < 0 ? -1 : (p.rows ? index(p.rows, p.rows_is_i64, b) : b);
    if (row >= p.n_rows) {
      atomicOr(p.status, HIPATTN_STATUS_SEQUENCE);
    } else if (row >= 0) {
      const int64_t t = index(p.k_pool.cache_seq_lens, p.k_pool.seq_lens_is_i64, row) - count + (tok - first);
      if (t < 0 || t >= (int64_t)p.k_pool.table_width * p.k_pool.page_size || t > 0x7fffffff) {
        atomicOr(p.status, HIPATTN_STATUS_TOKEN_RANGE);
      } else {
        const int pi = (int)t / p.k_pool.page_size;
        const int64_t pg = index(p.k_pool.block_table, p.k_pool.table_is_i64, row * p.k_pool.table_stride_b + pi);
        if (pg < 0 || pg >= p.k_pool.n_pages) {
          atomicOr(p.status, HIPATTN_STATUS_PAGE_RANGE);
        } else {
          page = (int)pg;
          off = (int)t - pi * p.k_pool.page_size;
        }
      }
    }
    s_page[threadIdx.x] = page;
    s_off[threadIdx.x] = off;
  }
  __syncthreads();
  for (;;) {
    for (int t0 = group; t0 < tokens; t0 += kWriteAhead * groups) {
      uint4 now[kWriteAhead];
#pragma unroll
      for (int k = 0; k < kWriteAhead; ++k) now[k] = x[k];
#pragma unroll
      for (int k = 0; k < kWriteAhead; ++k) load(t0 + (kWriteAhead + k) * groups, x[k]);
#pragma unroll
      for (int k = 0; k < kWriteAhead; ++k) {
        const int tok = t0 + k * groups;
        if (i >= 2 * pieces || tok >= tokens) break;
        const int page = s_page[tok];
        if (page < 0) continue;
        char* to = dst + page * page_step + s_off[tok] * off_step;
        if constexpr (F8) *reinterpret_cast<uint2*>(to) = narrow_e5m2<DT>(now[k]);
        else *reinterpret_cast<uint4*>(to) = now[k];
      }
    }
    i += lanes;                       // (tokens of more pieces than a CTA has threads)
    if (i >= 2 * pieces) break;
    place();
#pragma unroll
    for (int k = 0; k < kWriteAhead; ++k) load(group + k * groups, x[k]);
  }
}

int validate_pool(const hipattn_page_pool_t* p, const char* what, bool caches) {
  HIPATTN_REQUIRE(p != nullptr, HIPATTN_ERR_INVALID, "%s: the pool is null", what);
  HIPATTN_REQUIRE(p->ref_counts && p->seq_lens && p->block_table && p->status, HIPATTN_ERR_INVALID, "%s: ref_counts, seq_lens, block_table and status are required", what);
  HIPATTN_REQUIRE(p->n_pages > 0 && p->page_size > 0 && p->n_sequences > 0 && p->table_width > 0, HIPATTN_ERR_INVALID,
                  "%s: n_pages %d, page_size %d, n_sequences %d, table_width %d must be positive", what, p->n_pages, p->page_size, p->n_sequences, p->table_width);
  HIPATTN_REQUIRE(p->n_pages <= 0x7fff0000 && p->n_sequences <= HIPATTN_POOL_MAX_SEQUENCES, HIPATTN_ERR_UNSUPPORTED, "%s: %d pages, %d sequences are too many",
                  what, p->n_pages, p->n_sequences);
  if (!caches) return HIPATTN_OK;
  HIPATTN_REQUIRE(p->caches && p->n_caches > 0 && p->n_caches <= HIPATTN_POOL_MAX_CACHES, HIPATTN_ERR_INVALID, "%s: %d caches outside [1, %d]", what, p->n_caches,
                  HIPATTN_POOL_MAX_CACHES);
  HIPATTN_REQUIRE(p->page_bytes > 0 && p->page_bytes % ((int64_t)p->page_size * 16) == 0 && p->page_stride >= p->page_bytes && p->page_stride % 16 == 0,
                  HIPATTN_ERR_INVALID, "%s: pages of %lld bytes, %lld apart: tokens must be multiples of 16 bytes", what, (long long)p->page_bytes, (long long)p->page_stride);
  for (int i = 0; i < p->n_caches; ++i)
    HIPATTN_REQUIRE(p->caches[i] && (uintptr_t)p->caches[i] % 16 == 0, HIPATTN_ERR_INVALID, "%s: cache %d is null or not 16-byte aligned", what, i);
  return HIPATTN_OK;
}
Pool device_pool(const hipattn_page_pool_t& p) {
  return Pool{p.ref_counts, p.seq_lens, p.block_table, p.status, p.grown, p.n_pages, p.page_size, p.n_sequences, p.table_width};
}

int plan_ctas(const hipattn_page_pool_t& p) { return p.n_pages <= kSmallPool ? 1 : kPlanCtas; }

template <bool FORK>
int deal_pages(const hipattn_page_pool_t& p, const int32_t* a, const int32_t* b, int every, int n, int32_t* plan, cudaStream_t stream, const char* what) {
  HIPATTN_REQUIRE(n > 0 && n <= HIPATTN_POOL_MAX_ENTRIES, HIPATTN_ERR_INVALID, "%s: %d entries outside [1, %d]", what, n, HIPATTN_POOL_MAX_ENTRIES);
  HIPATTN_REQUIRE(a && (b || !FORK), HIPATTN_ERR_INVALID, "%s: null pointer", what);
  const size_t smem = 4 * sizeof(int) * (size_t)n + sizeof(uint32_t) * (size_t)((p.n_sequences + 31) / 32);
  HIPATTN_CUDA_OK(allow_smem((const void*)deal_pages_kernel<FORK>, smem));
  const int ctas = plan_ctas(p);
  InTurn launch(ctas, kPlanThreads, smem, stream, ctas);
  HIPATTN_CUDA_OK(cudaLaunchKernelEx(&launch.cfg, deal_pages_kernel<FORK>, device_pool(p), a, b, every, n, plan, ctas));
  return check_launch("deal_pages_kernel");
}

int64_t copy_grid(int64_t items) {
  const int64_t most = kSMs * 8;
  return items < 1 ? 1 : (items < most ? items : most);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" int64_t hipattn_pool_scratch(const hipattn_page_pool_t* p, int32_t n) {
  if (p == nullptr || n < 0) return 0;
  if (n > 0) return 16 + (int64_t)n * (int64_t)sizeof(PageCopy);
  return (2 + 2 * half_of(p->n_pages) + (int64_t)p->n_pages) * 4;
}

extern "C" int hipattn_pool_extend(const hipattn_page_pool_t* p, const int32_t* rows, const int32_t* n_tokens, int32_t every, int32_t n, void* stream) {
  const int rc = validate_pool(p, "pool_extend", false);
  return rc ? rc : deal_pages<false>(*p, rows, n_tokens, every, n, nullptr, (cudaStream_t)stream, "pool_extend");
}

extern "C" int hipattn_pool_fork(const hipattn_page_pool_t* p, const int32_t* parents, const int32_t* children, int32_t n, void* stream) {
  int rc = validate_pool(p, "pool_fork", true);
  if (rc) return rc;
  HIPATTN_REQUIRE(p->scratch != nullptr, HIPATTN_ERR_INVALID, "pool_fork: scratch is null");
  rc = deal_pages<true>(*p, parents, children, 0, n, (int32_t*)p->scratch, (cudaStream_t)stream, "pool_fork");
  if (rc) return rc;
  const int pieces = (int)((p->page_bytes + kCopyBytes - 1) / kCopyBytes);
  for (int c0 = 0; c0 < p->n_caches; c0 += kMaxCachesPerLaunch) {
    CacheList list;
    list.n = p->n_caches - c0 < kMaxCachesPerLaunch ? p->n_caches - c0 : kMaxCachesPerLaunch;
    for (int i = 0; i < list.n; ++i) list.at[i] = (char*)p->caches[c0 + i];
    InTurn launch(copy_grid((int64_t)n * list.n * pieces), kCopyThreads, 0, (cudaStream_t)stream);
    HIPATTN_CUDA_OK(cudaLaunchKernelEx(&launch.cfg, copy_begun_pages_kernel, list, (const int32_t*)p->scratch, p->page_stride, p->page_bytes / p->page_size, pieces));
    rc = check_launch("copy_begun_pages_kernel");
    if (rc) return rc;
  }
  return HIPATTN_OK;
}

extern "C" int hipattn_pool_free(const hipattn_page_pool_t* p, const int32_t* rows, int32_t n, void* stream) {
  const int rc = validate_pool(p, "pool_free", false);
  if (rc) return rc;
  HIPATTN_REQUIRE(n > 0 && n <= HIPATTN_POOL_MAX_ENTRIES, HIPATTN_ERR_INVALID, "pool_free: %d entries outside [1, %d]", n, HIPATTN_POOL_MAX_ENTRIES);
  HIPATTN_REQUIRE(rows != nullptr, HIPATTN_ERR_INVALID, "pool_free: null pointer");
  // rows of 512 pages: 3.0 us with a CTA each, 3.7 with a cluster; of 1024 3.4 and 3.6; of 2048 4.2 and 3.8; of 8192 8.7 and 4.3
  const int ctas = p->table_width > 1024 ? 8 : 1;
  InTurn launch((int64_t)n * ctas, 256, 0, (cudaStream_t)stream, ctas);
  HIPATTN_CUDA_OK(cudaLaunchKernelEx(&launch.cfg, free_rows_kernel, device_pool(*p), rows, ctas));
  return check_launch("free_rows_kernel");
}

extern "C" int hipattn_pool_compact(const hipattn_page_pool_t* p, int32_t* pages_in_use, void* stream) {
  int rc = validate_pool(p, "pool_compact", true);
  if (rc) return rc;
  HIPATTN_REQUIRE(p->scratch != nullptr, HIPATTN_ERR_INVALID, "pool_compact: scratch is null");
  const int ctas = plan_ctas(*p);
  InTurn plan(ctas, kPlanThreads, 0, (cudaStream_t)stream, ctas);
  HIPATTN_CUDA_OK(cudaLaunchKernelEx(&plan.cfg, plan_compact_kernel, device_pool(*p), (int32_t*)p->scratch, pages_in_use, ctas));
  rc = check_launch("plan_compact_kernel");
  if (rc) return rc;
  const int pieces = (int)((p->page_bytes + kCopyBytes - 1) / kCopyBytes);
  for (int c0 = 0; c0 < p->n_caches; c0 += kMaxCachesPerLaunch) {
    CacheList list;
    list.n = p->n_caches - c0 < kMaxCachesPerLaunch ? p->n_caches - c0 : kMaxCachesPerLaunch;
    for (int i = 0; i < list.n; ++i) list.at[i] = (char*)p->caches[c0 + i];
    InTurn launch(copy_grid((int64_t)half_of(p->n_pages) * list.n * pieces + (int64_t)p->n_sequences * ((p->table_width + 31) / 32) / 8), kCopyThreads, 0, (cudaStream_t)stream);
    HIPATTN_CUDA_OK(cudaLaunchKernelEx(&launch.cfg, move_pages_kernel, device_pool(*p), list, (int32_t*)p->scratch, p->page_stride, p->page_bytes, pieces, c0 == 0 ? 1 : 0));
    rc = check_launch("move_pages_kernel");
    if (rc) return rc;
  }
  return HIPATTN_OK;
}

extern "C" int hipattn_write_kv(const hipattn_write_kv_params_t* p, void* stream) {
  HIPATTN_REQUIRE(p != nullptr, HIPATTN_ERR_INVALID, "write_kv: params are null");
  HIPATTN_REQUIRE(p->k && p->v && p->status, HIPATTN_ERR_INVALID, "write_kv: k, v and status are required");
  HIPATTN_REQUIRE(p->N > 0 && p->B > 0 && p->HKV > 0 && p->D > 0 && p->n_rows > 0, HIPATTN_ERR_INVALID, "write_kv: bad shape N=%lld B=%d HKV=%d D=%d rows=%d",
                  (long long)p->N, p->B, p->HKV, p->D, p->n_rows);
  HIPATTN_REQUIRE(p->offsets || p->N % p->B == 0, HIPATTN_ERR_INVALID, "write_kv: %lld tokens are not a multiple of %d sequences", (long long)p->N, p->B);
  HIPATTN_REQUIRE(p->rows || p->n_rows >= p->B, HIPATTN_ERR_INVALID, "write_kv: %d entries, but a table of %d rows", p->B, p->n_rows);
  HIPATTN_REQUIRE(p->k_pool.cache && p->v_pool.cache, HIPATTN_ERR_INVALID, "write_kv: k and v must go to page pools");
  HIPATTN_REQUIRE(p->k_pool.n_pages == p->v_pool.n_pages && p->k_pool.page_size == p->v_pool.page_size && p->k_pool.fp8_e5m2 == p->v_pool.fp8_e5m2,
                  HIPATTN_ERR_INVALID, "write_kv: k and v must go to pools of the same pages and type");
  const int eb = p->dtype == HIPATTN_F32 ? 4 : 2;
  const int64_t ra = 16 / eb;
  int rc = validate_tokens(p->k_pool, eb, p->D, "k");
  if (rc) return rc;
  rc = validate_tokens(p->v_pool, eb, p->D, "v");
  if (rc) return rc;
  HIPATTN_REQUIRE((uintptr_t)p->k % 16 == 0 && (uintptr_t)p->v % 16 == 0 && p->k_stride_t % ra == 0 && p->k_stride_h % ra == 0 && p->v_stride_t % ra == 0 &&
                      p->v_stride_h % ra == 0,
                  HIPATTN_ERR_INVALID, "write_kv: rows of k and v must start on 16-byte boundaries");
  HIPATTN_REQUIRE((int64_t)p->HKV * p->D < (1 << 24) && p->k_pool.n_pages <= 0x7fffffffLL, HIPATTN_ERR_UNSUPPORTED, "write_kv: tokens of %lld values, %lld pages",
                  (long long)p->HKV * p->D, (long long)p->k_pool.n_pages);
  // tokens of a CTA: one each until the GPU is full four times over, then as many as have a few pieces for every thread
  int64_t span = p->N / (kSMs * 4);
  span = span < 1 ? 1 : (span > kMaxSpan ? kMaxSpan : span);
  const int64_t blocks = (p->N + span - 1) / span, pieces = 2 * (int64_t)p->HKV * (p->D / ra);
  int lanes = 32;      // threads to a token: a power of two that its pieces fill
  while (lanes < kWriteThreads && lanes < pieces) lanes *= 2;
  HIPATTN_REQUIRE(blocks < 0x7fffffffLL, HIPATTN_ERR_INVALID, "write_kv: grid of %lld blocks", (long long)blocks);
  const bool f8 = p->k_pool.fp8_e5m2 != 0;
  void (*kern)(const hipattn_write_kv_params_t, int, int) = nullptr;
  if (p->dtype == HIPATTN_F32) kern = write_kv_kernel<HIPATTN_F32, false>;
  if (p->dtype == HIPATTN_F16) kern = f8 ? write_kv_kernel<HIPATTN_F16, true> : write_kv_kernel<HIPATTN_F16, false>;
  if (p->dtype == HIPATTN_BF16) kern = f8 ? write_kv_kernel<HIPATTN_BF16, true> : write_kv_kernel<HIPATTN_BF16, false>;
  HIPATTN_REQUIRE(kern != nullptr, HIPATTN_ERR_INVALID, "write_kv: unknown dtype %d", p->dtype);
  InTurn launch(blocks, kWriteThreads, 0, (cudaStream_t)stream);
  HIPATTN_CUDA_OK(cudaLaunchKernelEx(&launch.cfg, kern, *p, (int)span, lanes));
  return check_launch("write_kv_kernel");
}
