// The paged 8-bit cache: what its kernels and the C ABI layer share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pmi {

// The LDS of a workgroup holds up to four ints a request (shared_runs_kernel: 64 KB and its waves' sums).
constexpr int kTablesMaxRequests = 4096;

struct PagedTables {
  int32_t* tables;  // [R, width], row stride `stride`
  int64_t stride;
  const int32_t* kv_lens;
  const int32_t* new_lens;
  const int32_t* free_pages;  // a ring of free pages: [ring]
  const int32_t* pool;        // its head and count, requests refused, 0
  int32_t* q_starts;          // [R + 1]
  int32_t* kv_lens_out;       // [R], may be kv_lens
  int32_t* first;             // [R]
  int32_t* fresh;             // [R + 1]
  int32_t* positions;         // [total]
  int32_t* slots;             // [total]
  int32_t* pool_out;          // [4], may be pool
  int64_t R, width, ring, ps, total;
  int64_t max_len;  // no request grows past so many tokens
};
hipError_t launch_extend_tables(const PagedTables& t, hipStream_t stream);
hipError_t launch_release_tables(const int32_t* tables, int64_t stride, int32_t* kv_lens, const uint8_t* done,
                                 int32_t* free_pages, int32_t* pool, int64_t R, int64_t width, int64_t ring,
                                 int64_t ps, hipStream_t stream);

// Requests r that begin as forks of request parents[r] (none: not 0 .. R - 1, or r itself).
struct PagedFork {
  int32_t* tables;
  int64_t stride;
  int32_t* kv_lens;
  const int32_t* parents;
  const int32_t* lengths;  // tokens to begin with, or null: all of the parent's
  const int32_t* free_pages;
  int32_t* pool;
  int32_t* shares;  // [ring] a page's owners beyond the first
  int32_t* src;     // [R] the page to be copied for r and where to, or -1
  int32_t* dst;
  int32_t* from;  // [R] scratch
  int64_t R, width, ring, ps;
};
hipError_t launch_fork_tables(const PagedFork& f, hipStream_t stream);

struct PagedRelease {
  const int32_t* tables;
  int64_t stride;
  int32_t* kv_lens;
  const uint8_t* done;
  int32_t* free_pages;
  int32_t* pool;
  int32_t* shares;
  int32_t* counts;  // scratch [page_chunks(ring) + 2]
  int64_t R, width, ring, ps;
};
int64_t page_chunks(int64_t ring);
hipError_t launch_release_shared(const PagedRelease& f, hipStream_t stream);

struct PagedCompact {
  int32_t* tables;
  int64_t stride;
  const int32_t* kv_lens;
  int32_t* free_pages;
  int32_t* pool;
  int32_t* shares;  // or null
  int32_t* src;     // [ring / 2]
  int32_t* dst;
  int32_t* moves;   // [1] how many of them
  int32_t* live;    // scratch: [ring], [ring], [page_chunks(ring)]
  int32_t* to;
  int32_t* counts;
  int64_t R, width, ring, ps;
};
hipError_t launch_compact_tables(const PagedCompact& f, hipStream_t stream);

constexpr int kCopyLayers = 64;  // of a launch
struct PagedCopy {
  void* k[kCopyLayers];
  void* v[kCopyLayers];
  float* k_scale[kCopyLayers];
  float* v_scale[kCopyLayers];
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count;  // entries of them, or null: n
  int64_t n, layers, pages, KV, page_bytes;
};
hipError_t launch_copy_pages(const PagedCopy& f, hipStream_t stream);

// Runs of requests whose first pages are the same.
struct PagedRuns {
  const int32_t* tables;
  int64_t stride;
  const int32_t* kv_lens;
  const int32_t* q_starts;  // null: one query a request
  int32_t* starts;          // [R + 1]
  int32_t* lens;            // [R]
  int32_t* runs;            // [R, 4] of each: first request, first query, queries, positions shared; 0 behind the last
  int32_t* counter;         // 0, and 0 again afterwards
  int32_t* common;          // scratch [R]
  int64_t R, width, ps, least_pages;
};
hipError_t launch_shared_runs(const PagedRuns& f, hipStream_t stream);

struct PagedCache {
  void* k;  // [pages, KV, ps, D] codes
  void* v;  // [pages, KV, ps / 16, D, 16] codes
  float* k_scale;  // [pages, KV]
  float* v_scale;
  int64_t pages, KV, ps, D;
  bool fp8;  // e4m3, else int8
};

// qkv [T, ld] (H + 2 KV heads of D), 16-byte aligned rows; cos, sin [L, D / 2].
hipError_t launch_append_kv(const PagedCache& c, const void* qkv, int64_t ld, bool bf16, const float* cos_t,
                            const float* sin_t, int64_t L, const int32_t* positions, const int32_t* slots, void* q_out,
                            int64_t T, int64_t H, hipStream_t stream);
hipError_t launch_read_pages(const PagedCache& c, const int32_t* pages, int out_dtype, void* k, void* v, int64_t n,
                             hipStream_t stream);

constexpr int64_t kPagedMaxKeys = 1ll << 30;  // of a request: width * page_size

struct PagedAttention {
  const void* q;  // [T, H, D], element strides below
  int64_t q_token, q_head;
  void* out;  // [T, H, D] contiguous
  const int32_t* tables;
  int64_t stride;
  const int32_t* kv_lens;
  const int32_t* q_starts;  // null: one query a request
  int64_t T, R, width, H;
  int64_t max_q, max_kv;
  int64_t window;  // 0: none
  float scale;
  bool bf16;
  const int32_t* runs;      // [R, 4] runs of requests that share their first pages (PagedRuns), or null
  const int32_t* run_lens;  // [R]
};
// Whether the count of tiles that the requests of few query rows may have fits 32 bits.
bool paged_attention_tiles_fit(const PagedAttention& p, const PagedCache& c);
// Whether its workgroups fit a launch.
bool paged_attention_launch_fits(const PagedAttention& p, const PagedCache& c);
// Bytes of the workspace, its counters included, for calls of these limits.
size_t paged_attention_ws_bytes(const PagedAttention& p, const PagedCache& c);
hipError_t launch_paged_attention(const PagedAttention& p, const PagedCache& c, void* workspace, size_t ws_bytes,
                                  hipStream_t stream);

// Whether a call with runs reads what a run shares once for all of it.
bool paged_attention_shares(const PagedAttention& p, const PagedCache& c);
// The same of such a call, two launches.
bool paged_shared_launch_fits(const PagedAttention& p, const PagedCache& c);
size_t paged_shared_ws_bytes(const PagedAttention& p, const PagedCache& c);
hipError_t launch_paged_shared(const PagedAttention& p, const PagedCache& c, void* workspace, hipStream_t stream);

}  // namespace pmi
