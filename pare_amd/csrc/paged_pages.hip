// Pages of the paged cache (paged_kv.hip describes it) that several requests own:
// requests that begin as forks of others, pages given back by their last owner, live pages
// moved to the cache's front, the copies of pages that go with both, and which requests of a
// batch have the same first pages.
//
// shares [pages] counts a page's owners beyond the first: 0 for a page of one request, for a
// fresh one and for a free one, so that what takes pages from the ring leaves it alone. Only
// whole pages are shared; the page in which a fork ends is copied, so that what a request
// writes (always behind its last token) never lies in a page with another owner.
//
// Every result is the same whatever the order of the atomics: counts are integers, and what
// is listed is listed in the order of requests or of pages.
#include "paged.h"
#include "pmi_common.h"
#include "pmi_launch.h"

namespace pmi {
namespace {

// Inclusive sum over the workgroup's threads; `waves` [blockDim / 64] in LDS, `all` their sum.
PMI_DEV int wg_sum_upto(int v, int* waves, int& all) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, n = blockDim.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (l >= o) v += u;
  }
  __syncthreads();  // waves of the previous call are read
  if (l == 63) waves[w] = v;
  __syncthreads();
  all = 0;
  for (int i = 0; i < n; ++i) {
    v += i < w ? waves[i] : 0;
    all += waves[i];
  }
  return v;
}

PMI_DEV int held_pages(int len, int ps, int width) {
  return (int)min(((int64_t)max(len, 0) + ps - 1) / ps, (int64_t)width);
}

// ---- forks ------------------------------------------------------------------------

// Request r's whole pages as its parent's, and one owner more for each of them.
PMI_DEV void share_page(const PagedFork& f, int r, int parent, int j) {
  const int page = f.tables[parent * f.stride + j];
  f.tables[r * f.stride + j] = page;
  if ((unsigned)page < (unsigned)f.ring) atomicAdd(&f.shares[page], 1);
}

// One workgroup: who is granted, the fresh pages, lengths and page copies and, with few
// entries, the shared pages as well. Everything is read before anything is written, so a
// parent is what it was before the call (an empty one gives an empty fork), and no parent's row
// is written: a fork's own row was empty. Bound by its chain of loads and the scan.
constexpr int kForkThreads = 1024;
__global__ __launch_bounds__(kForkThreads) void fork_tables_kernel(PagedFork f, int fill) {
  __shared__ int waves[kForkThreads / 64];
  __shared__ int begin_s[kTablesMaxRequests];  // its length; -1: not asked, -2: refused
  __shared__ int upto_s[kTablesMaxRequests];   // fresh pages of the requests up to and with it
  __shared__ int refused_s, taken_s;
  const int tid = threadIdx.x, R = (int)f.R, ps = (int)f.ps, ring = (int)f.ring;
  const int count = min(max(f.pool[1], 0), ring), refused0 = f.pool[2];
  const int head = f.pool[0] >= 0 && f.pool[0] < ring ? f.pool[0] : 0;
  if (tid == 0) refused_s = 0, taken_s = 0;
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += kForkThreads) {
    const int r = r0 + tid;
    int n = -1, need = 0;
    if (r < R) {
      const int p = f.parents[r];
      if ((unsigned)p < (unsigned)R && p != r) {
        n = (int)min((int64_t)max(f.kv_lens[p], 0), f.width * ps);
        if (f.lengths) n = min(max(f.lengths[r], 0), n);
        if (f.kv_lens[r] > 0) n = -2;
        need = n > 0 && n % ps ? 1 : 0;
      }
    }
    int all;
    const int upto = base + wg_sum_upto(need, waves, all);
    base += all;
    if (need && upto > count) n = -2;
    if (r < R) {
      begin_s[r] = n;
      upto_s[r] = upto;
      if (n == -2) atomicAdd(&refused_s, 1);
      if (need && n >= 0) atomicMax(&taken_s, upto);
    }
  }
  __syncthreads();
  if (tid == 0) {
    f.pool[0] = ring > 0 ? (int)(((int64_t)head + taken_s) % ring) : 0;
    f.pool[1] = count - taken_s;
    f.pool[2] = refused0 + refused_s;
    f.pool[3] = 0;
  }
  for (int r = tid; r < R; r += kForkThreads) {
    const int n = begin_s[r], full = n / ps, parent = f.parents[r];
    int src = -1, dst = -1;
    if (n > 0 && n % ps) {
      src = f.tables[parent * f.stride + full];
      dst = f.free_pages[((int64_t)head + upto_s[r] - 1) % ring];
      f.tables[r * f.stride + full] = dst;
    }
    f.src[r] = src, f.dst[r] = dst;
    f.from[r] = n >= ps ? parent : -1;
    if (n >= 0) f.kv_lens[r] = n;
  }
  if (!fill) return;
  for (int r = tid >> 6; r < R; r += kForkThreads / 64) {
    const int full = begin_s[r] / ps;
    for (int j = tid & 63; j < full; j += 64) share_page(f, r, f.parents[r], j);
  }
}

// The shared pages of many entries: a workgroup takes 1024 of a row.
constexpr int kRowEntries = 1024;
__global__ __launch_bounds__(256) void share_pages_kernel(PagedFork f) {
  const int r = blockIdx.y, parent = f.from[r];
  if (parent < 0) return;
  const int full = f.kv_lens[r] / (int)f.ps, j0 = blockIdx.x * kRowEntries;
  for (int j = j0 + threadIdx.x; j < min(full, j0 + kRowEntries); j += 256) share_page(f, r, parent, j);
}

// ---- caches of few pages, in one workgroup ----------------------------------------------

// Releases and compactions of few table entries and pages are bound by their launches and the chain of
// loads. One workgroup of 1024 threads then does all, with a bit or a count of each page in LDS, 5 us each.
// A release and a compaction with its copies, in a graph, took in this form / in the launches further down
// (us): 12 requests of up to 19 pages 21.8 / 30.5, 64 of up to 222 (14208 entries) 49 / 34.
constexpr int kSmallPages = 16384, kSmallEntries = 4096, kSmallThreads = 1024;

// f(r, j, page) for the entries of all requests that `use(r)` tells to take, eight of a thread in flight.
template <typename Use, typename F>
PMI_DEV void each_entry(const int32_t* tables, int64_t stride, const int32_t* kv_lens, int R, int width, int ps, int ring,
                        Use use, F f) {
  constexpr int kFly = 8;
  const int n = R * width;
  for (int u0 = threadIdx.x; u0 < n; u0 += kSmallThreads * kFly) {
    int page[kFly], len[kFly];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int u = min(u0 + kSmallThreads * k, n - 1), r = u / width;
      page[k] = tables[r * stride + u - r * width];
      len[k] = use(r) ? kv_lens[r] : 0;
    }
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int u = u0 + kSmallThreads * k;
      if (u >= n) break;
      const int r = u / width, j = u - r * width;
      if (j < held_pages(len[k], ps, width) && (unsigned)page[k] < (unsigned)ring) f(r, j, page[k]);
    }
  }
}

// Bits of pages, and how many are set before each word of them.
struct PageBits {
  uint32_t bit[kSmallPages / 32];
  int before[kSmallPages / 32];
  int waves[kSmallThreads / 64];
  PMI_DEV bool has(int p) const { return bit[p >> 5] >> (p & 31) & 1; }
  PMI_DEV int rank(int p) const { return before[p >> 5] + __popc(bit[p >> 5] & ((1u << (p & 31)) - 1)); }
  // The bits are set (by all threads, before): the sums, and how many there are.
  PMI_DEV int count() {
    static_assert(kSmallPages / 32 <= kSmallThreads, "a word a thread");
    const int tid = threadIdx.x;
    __syncthreads();
    const int mine = tid < kSmallPages / 32 ? __popc(bit[tid]) : 0;
    int all;
    const int upto = wg_sum_upto(mine, waves, all);
    if (tid < kSmallPages / 32) before[tid] = upto - mine;
    __syncthreads();
    return all;
  }
};

__global__ __launch_bounds__(kSmallThreads) void release_small_kernel(PagedRelease f) {
  __shared__ PageBits left;
  __shared__ uint32_t gone[kSmallPages];  // owners that a page loses
  const int tid = threadIdx.x, R = (int)f.R, ring = (int)f.ring;
  const int count = min(max(f.pool[1], 0), ring), head = f.pool[0] >= 0 && f.pool[0] < ring ? f.pool[0] : 0;
  for (int p = tid; p < ring; p += kSmallThreads) gone[p] = 0;
  if (tid < kSmallPages / 32) left.bit[tid] = 0;
  __syncthreads();
  each_entry(f.tables, f.stride, f.kv_lens, R, (int)f.width, (int)f.ps, ring, [&](int r) { return f.done[r] != 0; },
             [&](int, int, int page) { atomicAdd(&gone[page], 1u); });
  __syncthreads();
  for (int p = tid; p < ring; p += kSmallThreads) {
    if (!gone[p]) continue;
    const int owners = f.shares[p] - (int)gone[p];
    f.shares[p] = max(owners, 0);
    if (owners < 0) atomicOr(&left.bit[p >> 5], 1u << (p & 31));
  }
  const int n = left.count();
  for (int p = tid; p < ring; p += kSmallThreads) {
    if (!left.has(p)) continue;
    // (more than the ring has room for cannot be the pool's)
    const int at = left.rank(p);
    if (at < ring - count) f.free_pages[(head + count + at) % ring] = p;
  }
  if (tid == 0) f.pool[1] = min(count + n, ring);
  for (int r = tid; r < R; r += kSmallThreads)
    if (f.done[r]) f.kv_lens[r] = 0;
}

__global__ __launch_bounds__(kSmallThreads) void compact_small_kernel(PagedCompact f) {
  __shared__ PageBits live;
  __shared__ uint16_t hole[kSmallPages / 2];
  const int tid = threadIdx.x, R = (int)f.R, ring = (int)f.ring, width = (int)f.width, ps = (int)f.ps;
  const auto all_rows = [](int) { return true; };
  if (tid < kSmallPages / 32) live.bit[tid] = 0;
  __syncthreads();
  each_entry(f.tables, f.stride, f.kv_lens, R, width, ps, ring, all_rows,
             [&](int, int, int page) { atomicOr(&live.bit[page >> 5], 1u << (page & 31)); });
  const int n = live.count();
  const int below = n < kSmallPages ? live.rank(n) : n, movers = n - below;
  for (int p = tid; p < ring; p += kSmallThreads) {
    f.free_pages[p] = p + n < ring ? n + p : n + p - ring;
    if (!live.has(p) && p < n) hole[p - live.rank(p)] = (uint16_t)p;
  }
  for (int i = movers + tid; i < ring / 2; i += kSmallThreads) f.src[i] = -1, f.dst[i] = -1;
  __syncthreads();
  for (int p = tid; p < ring; p += kSmallThreads) {
    const bool there = live.has(p);
    if (p < n) continue;  // stays, or is written for the page that moves there
    if (there) {
      const int i = live.rank(p) - below;
      f.src[i] = p, f.dst[i] = hole[i];
      if (f.shares) f.shares[hole[i]] = f.shares[p];
    }
    if (f.shares) f.shares[p] = 0;
  }
  each_entry(f.tables, f.stride, f.kv_lens, R, width, ps, ring, all_rows, [&](int r, int j, int page) {
    if (page >= n) f.tables[r * f.stride + j] = hole[live.rank(page) - below];
  });
  if (tid == 0) {
    f.moves[0] = movers;
    f.pool[0] = 0;
    f.pool[1] = ring - n;
    f.pool[3] = 0;
  }
}

// ---- pages given back by their last owner --------------------------------------------

constexpr int kChunk = 4096;  // pages of a workgroup of 1024 threads

// One owner less for each page of the finished requests: below zero where none is left.
__global__ __launch_bounds__(256) void leave_pages_kernel(PagedRelease f) {
  const int r = blockIdx.y;
  if (!f.done[r]) return;
  const int held = held_pages(f.kv_lens[r], (int)f.ps, (int)f.width), j0 = blockIdx.x * kRowEntries;
  for (int j = j0 + threadIdx.x; j < min(held, j0 + kRowEntries); j += 256) {
    const int page = f.tables[r * f.stride + j];
    if ((unsigned)page < (unsigned)f.ring) atomicSub(&f.shares[page], 1);
  }
}

// How many pages of each chunk have no owner left; behind the counts the pool as it was.
__global__ __launch_bounds__(1024) void count_left_kernel(PagedRelease f) {
  __shared__ int waves[16];
  const int64_t p0 = (int64_t)blockIdx.x * kChunk + threadIdx.x * 4;
  int n = 0, all;
#pragma unroll
  for (int e = 0; e < 4; ++e) n += p0 + e < f.ring && f.shares[p0 + e] < 0;
  wg_sum_upto(n, waves, all);
  if (threadIdx.x == 0) f.counts[blockIdx.x] = all;
  if (blockIdx.x == 0 && threadIdx.x < 2) f.counts[gridDim.x + threadIdx.x] = f.pool[threadIdx.x];
}

// They go behind the free ones of the ring, in the order of their numbers. With one workgroup
// there are no counts: it takes chunk after chunk.
__global__ __launch_bounds__(1024) void collect_left_kernel(PagedRelease f, int chunks) {
  __shared__ int waves[16];
  const int tid = threadIdx.x, ring = (int)f.ring;
  const bool alone = gridDim.x == 1;
  const int head0 = alone ? f.pool[0] : f.counts[chunks], count0 = alone ? f.pool[1] : f.counts[chunks + 1];
  const int count = min(max(count0, 0), ring), head = head0 >= 0 && head0 < ring ? head0 : 0;
  int before = 0;
  if (!alone) {
    int n = 0;
    for (int i = tid; i < (int)blockIdx.x; i += 1024) n += f.counts[i];
    wg_sum_upto(n, waves, before);
  }
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int64_t p0 = (int64_t)c * kChunk + tid * 4;
    bool left[4];
    int n = 0, all;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      left[e] = p0 + e < ring && f.shares[p0 + e] < 0;
      n += left[e];
    }
    int at = before + wg_sum_upto(n, waves, all) - n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (left[e]) {
        // (more than the ring has room for cannot be the pool's)
        if (at < ring - count) f.free_pages[((int64_t)head + count + at) % ring] = (int)(p0 + e);
        f.shares[p0 + e] = 0;
        ++at;
      }
    before += all;
  }
  if (blockIdx.x == gridDim.x - 1) {
    __syncthreads();
    if (tid == 0) f.pool[1] = min(count + before, ring);
    for (int r = tid; r < (int)f.R; r += 1024)
      if (f.done[r]) f.kv_lens[r] = 0;
  }
}

// ---- live pages to the front ---------------------------------------------------------

__global__ __launch_bounds__(256) void clear_live_kernel(PagedCompact f) {
  for (int64_t p = blockIdx.x * 256 + threadIdx.x; p < f.ring; p += (int64_t)gridDim.x * 256) f.live[p] = 0;
}

__global__ __launch_bounds__(256) void mark_live_kernel(PagedCompact f) {
  const int r = blockIdx.y;
  const int held = held_pages(f.kv_lens[r], (int)f.ps, (int)f.width), j0 = blockIdx.x * kRowEntries;
  for (int j = j0 + threadIdx.x; j < min(held, j0 + kRowEntries); j += 256) {
    const int page = f.tables[r * f.stride + j];
    if ((unsigned)page < (unsigned)f.ring) f.live[page] = 1;
  }
}

__global__ __launch_bounds__(1024) void count_live_kernel(PagedCompact f) {
  __shared__ int waves[16];
  const int64_t p0 = (int64_t)blockIdx.x * kChunk + threadIdx.x * 4;
  int n = 0, all;
#pragma unroll
  for (int e = 0; e < 4; ++e) n += p0 + e < f.ring && f.live[p0 + e];
  wg_sum_upto(n, waves, all);
  if (threadIdx.x == 0) f.counts[blockIdx.x] = all;
}

// With L live pages: those from page L on, in order, take the free ones before it, in order.
// to[p] is a live page's new place, or -1 - i for the i-th that moves.
__global__ __launch_bounds__(1024) void place_live_kernel(PagedCompact f, int chunks) {
  __shared__ int waves[16];
  const int tid = threadIdx.x;
  int n = 0, m = 0, total, before;
  for (int i = tid; i < chunks; i += 1024) {
    n += f.counts[i];
    m += i < (int)blockIdx.x ? f.counts[i] : 0;
  }
  wg_sum_upto(n, waves, total);
  wg_sum_upto(m, waves, before);
  // the live ones before page L
  const int border = total / kChunk;
  int below = 0, below_all;
  for (int i = tid; i < border; i += 1024) below += f.counts[i];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t p = (int64_t)border * kChunk + tid * 4 + e;
    below += p < total && f.live[p];
  }
  wg_sum_upto(below, waves, below_all);
  const int movers = total - below_all;
  const int64_t p0 = (int64_t)blockIdx.x * kChunk + tid * 4;
  bool live[4];
  int mine = 0, all;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    live[e] = p0 + e < f.ring && f.live[p0 + e];
    mine += live[e];
  }
  int rank = before + wg_sum_upto(mine, waves, all) - mine;  // live pages before this one
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t p = p0 + e;
    if (p >= f.ring) break;
    if (live[e]) {
      if (p < total) {
        f.to[p] = (int)p;
      } else {
        f.to[p] = -1 - (rank - below_all);
        f.src[rank - below_all] = (int)p;
      }
    } else {
      if (p < total) f.dst[p - rank] = (int)p;
      if (f.shares) f.shares[p] = 0;
    }
    rank += live[e];
    f.free_pages[p] = (int)((total + p) % f.ring);
  }
  for (int64_t i = movers + (int64_t)blockIdx.x * 1024 + tid; i < f.ring / 2; i += (int64_t)gridDim.x * 1024)
    f.src[i] = -1, f.dst[i] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    f.moves[0] = movers;
    f.pool[0] = 0;
    f.pool[1] = (int)f.ring - total;
    f.pool[3] = 0;
  }
}

// The tables' entries (the first R workgroup rows) and the owners of the pages that move.
__global__ __launch_bounds__(256) void move_live_kernel(PagedCompact f) {
  const int r = blockIdx.y, j0 = blockIdx.x * kRowEntries;
  if (r < (int)f.R) {
    const int held = held_pages(f.kv_lens[r], (int)f.ps, (int)f.width);
    for (int j = j0 + threadIdx.x; j < min(held, j0 + kRowEntries); j += 256) {
      int32_t* entry = f.tables + r * f.stride + j;
      const int page = *entry;
      if ((unsigned)page >= (unsigned)f.ring) continue;
      const int to = f.to[page];
      if (to != page) *entry = f.dst[-1 - to];
    }
  } else if (f.shares) {
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < f.moves[0]; i += (int64_t)gridDim.x * 256) {
      const int src = f.src[i], dst = f.dst[i];
      f.shares[dst] = f.shares[src];
      f.shares[src] = 0;
    }
  }
}

// ---- copies of pages -------------------------------------------------------------------

// Bound by the bytes. A unit is 16 KB of one page's keys or values of one layer (its first
// also takes the scales); the workgroups of a layer take its units in turn.
constexpr int kCopyBytes = 16384;
__global__ __launch_bounds__(256) void copy_pages_kernel(PagedCopy f) {
  const int tid = threadIdx.x, layer = blockIdx.y >> 1, of_v = blockIdx.y & 1;
  const int64_t n = f.count ? min(f.n, (int64_t)max(f.count[0], 0)) : f.n;
  uint8_t* codes = (uint8_t*)(of_v ? f.v[layer] : f.k[layer]);
  float* scales = of_v ? f.v_scale[layer] : f.k_scale[layer];
  const int per_page = (int)((f.page_bytes + kCopyBytes - 1) / kCopyBytes);
  for (int64_t u = blockIdx.x; u < n * per_page; u += gridDim.x) {
    const int64_t i = u / per_page;
    const int piece = (int)(u - i * per_page);
    const int src = f.src[i], dst = f.dst[i];
    if ((unsigned)src >= (unsigned)f.pages || (unsigned)dst >= (unsigned)f.pages) continue;
    const u32x4* a = reinterpret_cast<const u32x4*>(codes + src * f.page_bytes + (int64_t)piece * kCopyBytes);
    u32x4* b = reinterpret_cast<u32x4*>(codes + dst * f.page_bytes + (int64_t)piece * kCopyBytes);
    const int units = (int)(min(f.page_bytes - (int64_t)piece * kCopyBytes, (int64_t)kCopyBytes) / 16);
    u32x4 x[kCopyBytes / 4096];
#pragma unroll
    for (int k = 0; k < kCopyBytes / 4096; ++k)
      if (tid + 256 * k < units) x[k] = a[tid + 256 * k];
#pragma unroll
    for (int k = 0; k < kCopyBytes / 4096; ++k)
      if (tid + 256 * k < units) b[tid + 256 * k] = x[k];
    if (piece == 0)
      for (int h = tid; h < (int)f.KV; h += 256) scales[dst * f.KV + h] = scales[src * f.KV + h];
  }
}

// ---- requests with the same first pages ---------------------------------------------------

// A wave takes a request: how many of its first pages, whole and before its new tokens, are those
// of the last request before it that has new tokens (-1 if it has none itself). The last workgroup to
// arrive makes runs of them: a request with fewer than `least` pages in common begins one, and all of a
// run share what its members have in common.
constexpr int kRunThreads = 256;
struct RequestPages {
  int n, whole;  // new tokens; whole pages before them
};
PMI_DEV RequestPages request_pages(const PagedRuns& f, int r) {
  const int len = max(f.kv_lens[r], 0);
  int n = 1;
  if (f.q_starts) n = max(f.q_starts[r + 1] - f.q_starts[r], 0);
  if (len == 0) n = 0;
  return {n, min(max(len - n, 0) / (int)f.ps, (int)f.width)};
}
__global__ __launch_bounds__(kRunThreads) void shared_runs_kernel(PagedRuns f) {
  __shared__ int waves[kRunThreads / 64];
  __shared__ int common_s[kTablesMaxRequests], run_s[kTablesMaxRequests], least_s[kTablesMaxRequests];
  __shared__ int first_s[kTablesMaxRequests];
  __shared__ int s_last;
  const int tid = threadIdx.x, l = tid & 63, R = (int)f.R;
  const int r = blockIdx.x * (kRunThreads / 64) + (tid >> 6);
  if (r < R) {
    const RequestPages mine = request_pages(f, r);
    int common = mine.n > 0 ? 0 : -1;
    if (mine.n > 0) {
      int other = -1, whole = 0;
      for (int end = r; end > 0 && other < 0; end -= 64) {  // 64 requests before this one at a time
        const int at = end - 1 - l;
        RequestPages x = {0, 0};
        if (at >= 0) x = request_pages(f, at);
        const uint64_t live = __ballot(x.n > 0);
        if (live) {
          const int first = __builtin_ctzll(live);
          other = end - 1 - first;
          whole = __shfl(x.whole, first);
        }
      }
      if (other >= 0) {
        const int most = min(whole, mine.whole);
        const int32_t *a = f.tables + r * f.stride, *b = f.tables + other * f.stride;
        common = most;
        for (int j = 0; j < most; j += 256) {  // four entries a lane, a lane's next to each other in time
          uint64_t differ[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = j + 64 * e + l;
            const bool in = at < most;
            const int x = in ? a[at] : 0, y = in ? b[at] : 0;
            differ[e] = __ballot(in && (x != y || x < 0));
          }
          int found = -1;
#pragma unroll
          for (int e = 3; e >= 0; --e)
            if (differ[e]) found = j + 64 * e + __builtin_ctzll(differ[e]);
          if (found >= 0) {
            common = found;
            break;
          }
        }
      }
    }
    if (l == 0) __hip_atomic_store(&f.common[r], common, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const int old = __hip_atomic_fetch_add(f.counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  const int least = (int)f.least_pages;
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += kRunThreads) {
    const int x = r0 + tid;
    int c = -1;
    if (x < R) c = __hip_atomic_load(&f.common[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool begins = c >= 0 && c < least;
    int all;
    const int run = base + wg_sum_upto(begins, waves, all) - 1;
    base += all;
    if (x < R) {
      common_s[x] = c, run_s[x] = run;
      least_s[x] = INT32_MAX;
      if (begins) f.starts[run] = first_s[run] = x;
    }
  }
  __syncthreads();
  for (int x = tid; x < R; x += kRunThreads)
    if (common_s[x] >= least) atomicMin(&least_s[run_s[x]], common_s[x]);
  __syncthreads();
  for (int x = tid; x < R; x += kRunThreads) {
    const int pages = common_s[x] < 0 ? INT32_MAX : least_s[run_s[x]];
    f.lens[x] = pages == INT32_MAX ? 0 : pages * (int)f.ps;
  }
  for (int x = base + tid; x <= R; x += kRunThreads) f.starts[x] = R;
  // what a run is as one request (base of them; the next one's first request ends it)
  for (int x = tid; x < R; x += kRunThreads) {
    int4 run = {0, 0, 0, 0};
    const int pages = x < base ? least_s[x] : INT32_MAX;
    if (pages != INT32_MAX) {
      const int first = first_s[x], last = x + 1 < base ? first_s[x + 1] : R;
      run = int4{first, f.q_starts ? f.q_starts[first] : first, 0, pages * (int)f.ps};
      run.z = (f.q_starts ? f.q_starts[last] : last) - run.y;
    }
    reinterpret_cast<int4*>(f.runs)[x] = run;
  }
  if (tid == 0) __hip_atomic_store(f.counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

unsigned row_pieces(int64_t width) { return (unsigned)((width + kRowEntries - 1) / kRowEntries); }

bool one_workgroup(int64_t R, int64_t width, int64_t ring) { return ring <= kSmallPages && R * width <= kSmallEntries; }

}  // namespace

hipError_t launch_fork_tables(const PagedFork& f, hipStream_t stream) {
  const bool fill = f.R * f.width <= 16384;
  hipLaunchKernelGGL(fork_tables_kernel, dim3(1), dim3(kForkThreads), 0, stream, f, fill ? 1 : 0);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || fill) return e;
  hipLaunchKernelGGL(share_pages_kernel, dim3(row_pieces(f.width), (unsigned)f.R), dim3(256), 0, stream, f);
  return hipGetLastError();
}

int64_t page_chunks(int64_t ring) { return (ring + kChunk - 1) / kChunk; }

hipError_t launch_release_shared(const PagedRelease& f, hipStream_t stream) {
  if (one_workgroup(f.R, f.width, f.ring)) {
    hipLaunchKernelGGL(release_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, f);
    return hipGetLastError();
  }
  if (f.width > 0)
    hipLaunchKernelGGL(leave_pages_kernel, dim3(row_pieces(f.width), (unsigned)f.R), dim3(256), 0, stream, f);
  const int chunks = (int)page_chunks(f.ring);
  const bool alone = chunks <= 4;  // (no count of them first)
  if (!alone) hipLaunchKernelGGL(count_left_kernel, dim3((unsigned)chunks), dim3(1024), 0, stream, f);
  hipLaunchKernelGGL(collect_left_kernel, dim3(alone ? 1u : (unsigned)chunks), dim3(1024), 0, stream, f, chunks);
  return hipGetLastError();
}

hipError_t launch_compact_tables(const PagedCompact& f, hipStream_t stream) {
  if (one_workgroup(f.R, f.width, f.ring)) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, f);
    return hipGetLastError();
  }
  const unsigned chunks = (unsigned)page_chunks(f.ring), pieces = row_pieces(f.width);
  hipLaunchKernelGGL(clear_live_kernel, dim3(chunks), dim3(256), 0, stream, f);
  if (f.R > 0 && pieces > 0)
    hipLaunchKernelGGL(mark_live_kernel, dim3(pieces, (unsigned)f.R), dim3(256), 0, stream, f);
  hipLaunchKernelGGL(count_live_kernel, dim3(chunks), dim3(1024), 0, stream, f);
  hipLaunchKernelGGL(place_live_kernel, dim3(chunks), dim3(1024), 0, stream, f, (int)chunks);
  hipLaunchKernelGGL(move_live_kernel, dim3(pieces > 0 ? pieces : 1, (unsigned)f.R + 1), dim3(256), 0, stream, f);
  return hipGetLastError();
}

hipError_t launch_copy_pages(const PagedCopy& f, hipStream_t stream) {
  const int64_t units = f.n * ((f.page_bytes + kCopyBytes - 1) / kCopyBytes);
  int64_t wgs = (8 * device_cu_count() + 2 * f.layers - 1) / (2 * f.layers);
  if (wgs > units) wgs = units;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)wgs, (unsigned)(2 * f.layers)), dim3(256), 0, stream, f);
  return hipGetLastError();
}

hipError_t launch_shared_runs(const PagedRuns& f, hipStream_t stream) {
  hipLaunchKernelGGL(shared_runs_kernel, dim3((unsigned)((f.R + 3) / 4)), dim3(kRunThreads), 0, stream, f);
  return hipGetLastError();
}

}  // namespace pmi
