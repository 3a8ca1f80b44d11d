// The paged cache of 8-bit keys and values: block tables and slot maps from
// request lengths, the write of new tokens with RoPE, and the read of whole pages.
//
// Cache. A page holds page_size tokens of every KV head (16, 32, 64, 128 or 256):
//   k_cache [pages, KV, page_size, D]          token-major codes
//   v_cache [pages, KV, page_size / 16, D, 16] token 16 b + j of a page at [b, :, j]
//   k_scale, v_scale fp32 [pages, KV]          value = code * scale
// Codes are int8 (top 127) or e4m3 (top 448). The blocks of 16 tokens of v_cache
// are what an MFMA operand of the product with the probabilities takes: 16
// consecutive tokens of one dimension are 16 bytes.
//
// None of these has a counterpart in the reference, whose decode is HuggingFace's
// cache (pare/eval/throughput.py:84-126 times HF generate).
#include <cfloat>

#include "paged.h"
#include "pmi_common.h"
#include "pmi_launch.h"

namespace pmi {
namespace {

// ---- block tables and slot maps -------------------------------------------------

// Inclusive sum over the workgroup's 1024 threads of two counts at once.
struct Pair {
  int64_t a, b;
};
PMI_DEV Pair wg_scan(Pair v, Pair* wave_sums) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t a = __shfl_up(v.a, o), b = __shfl_up(v.b, o);
    if (l >= o) v.a += a, v.b += b;
  }
  __syncthreads();  // wave_sums of the previous call are read
  if (l == 63) wave_sums[w] = v;
  __syncthreads();
  for (int i = 0; i < w; ++i) v.a += wave_sums[i].a, v.b += wave_sums[i].b;
  return v;
}

// First index i < n with v[i] > x (v ascending), or n - 1.
template <typename P>
PMI_DEV int first_above(const P* v, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

struct TablesArgs {
  int32_t* tables;
  int64_t stride;
  const int32_t* kv_lens;
  const int32_t* new_lens;
  const int32_t* free_pages;
  const int32_t* pool;
  int32_t* q_starts;
  int32_t* kv_lens_out;
  int32_t* first;
  int32_t* fresh;
  int32_t* positions;
  int32_t* slots;
  int32_t* pool_out;
  int R, width, ring, ps, total;
  int64_t max_len;
};

// Fresh page i of all (of request r, whose first is fresh page `base`) into its row.
PMI_DEV void fill_page(const TablesArgs& a, int i, int r, int base, int first, int head) {
  const int held = (first + a.ps - 1) / a.ps;
  a.tables[r * a.stride + held + i - base] = a.free_pages[((int64_t)head + i) % a.ring];
}

// Slot and position of token t from its request's first position (-1: refused). Fresh pages
// are taken from the ring itself, so that nothing waits for their entries.
PMI_DEV void token_slot(const TablesArgs& a, int t, int r, int start, int first, int base, int head, bool live) {
  int pos = 0, slot = -1;
  if (live && first >= 0) {
    pos = first + t - start;
    const int held = (first + a.ps - 1) / a.ps, j = pos / a.ps;
    const int page = j < held ? a.tables[r * a.stride + j] : a.free_pages[((int64_t)head + base + j - held) % a.ring];
    slot = page < 0 || page >= a.ring ? -1 : page * a.ps + pos % a.ps;
  }
  a.positions[t] = pos;
  a.slots[t] = slot;
}

// One workgroup: the per-request sums and, for few tokens, the fresh pages and slots as
// well. Bound by the chain of loads, two scans and the look-ups (128 requests of one token: 5 us,
// 6.6 in a graph with its launch), not by its bytes; the sums are 64-bit.
// need_r = ceil((len + new) / ps) - ceil(len / ps); a request is granted where its table row is wide
// enough, it stays within max_len and the sums up to it, of needs and of new tokens, are within the pool and
// the total, so the granted ones that need pages are the first of them in order.
// Everything is read before anything is written: kv_lens_out may be kv_lens,
// pool_out may be pool.
__global__ __launch_bounds__(1024) void extend_tables_kernel(TablesArgs a, int fill) {
  __shared__ Pair wave_sums[16];
  __shared__ int ends[kTablesMaxRequests];   // new tokens up to and with request r
  __shared__ int pages[kTablesMaxRequests];  // needed pages up to and with request r
  __shared__ int old_len[kTablesMaxRequests];
  __shared__ int taken_s, refused_s;
  const int tid = threadIdx.x;
  // a head or count that no pool has cannot lead outside the ring
  const int count = min(max(a.pool[1], 0), a.ring), refused0 = a.pool[2];
  const int head = a.pool[0] >= 0 && a.pool[0] < a.ring ? a.pool[0] : 0;
  if (tid == 0) taken_s = 0, refused_s = 0;
  Pair base = {0, 0};
  for (int r0 = 0; r0 < a.R; r0 += 1024) {
    const int r = r0 + tid;
    int len = 0, fresh = 0;
    int64_t need = 0;
    bool fits = true;
    if (r < a.R) {
      len = max(a.kv_lens[r], 0);
      fresh = max(a.new_lens[r], 0);
      const int64_t want = ((int64_t)len + fresh + a.ps - 1) / a.ps, held = ((int64_t)len + a.ps - 1) / a.ps;
      fits = want <= a.width && (int64_t)len + fresh <= a.max_len;
      need = fits ? want - held : 0;
    }
    Pair s = wg_scan(Pair{(int64_t)fresh, need}, wave_sums);
    s.a += base.a, s.b += base.b;
    if (r < a.R) {
      const bool granted = fits && (need == 0 || s.b <= count) && (fresh == 0 || s.a <= a.total);
      ends[r] = (int)min(s.a, (int64_t)a.total);
      pages[r] = (int)min(s.b, (int64_t)INT32_MAX);
      old_len[r] = granted ? len : -1;
      if (granted && need > 0) atomicMax(&taken_s, (int)s.b);
      if (!granted) atomicAdd(&refused_s, 1);
      a.q_starts[r + 1] = ends[r];
      a.first[r] = old_len[r];
      a.fresh[r + 1] = pages[r];
      a.kv_lens_out[r] = granted ? len + fresh : len;
    }
    // the sums of the whole chunk
    __syncthreads();
    for (int i = 0; i < 16; ++i) base.a += wave_sums[i].a, base.b += wave_sums[i].b;
  }
  __syncthreads();
  const int taken = taken_s;
  if (tid == 0) {
    a.q_starts[0] = 0;
    a.pool_out[0] = a.ring > 0 ? (int)(((int64_t)head + taken) % a.ring) : 0;
    a.pool_out[1] = count - taken;
    a.pool_out[2] = refused0 + refused_s;
    a.pool_out[3] = 0;
  }
  if (tid == 0) a.fresh[0] = 0;
  // past what was granted the sums count refused requests: nothing looks there
  for (int r = tid; r < a.R; r += 1024)
    if (pages[r] > taken) a.fresh[r + 1] = taken;
  if (!fill) return;
  for (int i = tid; i < taken; i += 1024) {
    const int r = first_above(pages, a.R, i);
    fill_page(a, i, r, r ? pages[r - 1] : 0, old_len[r], head);
  }
  for (int t = tid; t < a.total; t += 1024) {
    const int r = first_above(ends, a.R, t);
    token_slot(a, t, r, r ? ends[r - 1] : 0, old_len[r], r ? pages[r - 1] : 0, head, t < (a.R ? ends[a.R - 1] : 0));
  }
}

// The fresh pages and slots of many tokens.
__global__ __launch_bounds__(256) void fill_tables_kernel(TablesArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.total) return;
  if (a.R == 0) return token_slot(a, t, 0, 0, -1, 0, 0, false);
  const int taken = a.fresh[a.R];
  const int head = a.ring > 0 ? (int)(((int64_t)a.pool_out[0] + a.ring - taken) % a.ring) : 0;
  for (int64_t i = t; i < taken; i += a.total) {
    const int r = first_above(a.fresh + 1, a.R, (int)i);
    fill_page(a, (int)i, r, a.fresh[r], a.first[r], head);
  }
  const int r = first_above(a.q_starts + 1, a.R, t);
  token_slot(a, t, r, a.q_starts[r], a.first[r], a.fresh[r], head, t < a.q_starts[a.R]);
}

// Pages of the finished requests behind the free ones of the ring, in request order.
__global__ __launch_bounds__(1024) void release_tables_kernel(const int32_t* __restrict__ tables, int64_t stride,
                                                              int32_t* __restrict__ kv_lens,
                                                              const uint8_t* __restrict__ done,
                                                              int32_t* __restrict__ free_pages,
                                                              int32_t* __restrict__ pool, int R, int width, int ring,
                                                              int ps) {
  __shared__ Pair wave_sums[16];
  __shared__ int ends[kTablesMaxRequests];
  const int tid = threadIdx.x;
  const int count = min(max(pool[1], 0), ring), head = pool[0] >= 0 && pool[0] < ring ? pool[0] : 0;
  Pair base = {0, 0};
  for (int r0 = 0; r0 < R; r0 += 1024) {
    const int r = r0 + tid;
    int64_t held = 0;
    if (r < R && done[r]) held = min(((int64_t)max(kv_lens[r], 0) + ps - 1) / ps, (int64_t)width);
    Pair s = wg_scan(Pair{held, 0}, wave_sums);
    if (r < R) {
      ends[r] = (int)min(base.a + s.a, (int64_t)INT32_MAX);
      if (done[r]) kv_lens[r] = 0;
    }
    __syncthreads();
    for (int i = 0; i < 16; ++i) base.a += wave_sums[i].a;
  }
  __syncthreads();
  // more pages than the ring has room for cannot be the pool's: they are left out
  const int n = min(ends[R - 1], ring - count);
  for (int i = tid; i < n; i += 1024) {
    const int r = first_above(ends, R, i);
    free_pages[((int64_t)head + count + i) % ring] = tables[r * stride + i - (r ? ends[r - 1] : 0)];
  }
  if (tid == 0) pool[1] = count + n;
}

// ---- the write of new tokens ----------------------------------------------------

struct AppendArgs {
  const void* qkv;
  const float* cos_t;
  const float* sin_t;
  const int32_t* positions;
  const int32_t* slots;
  void* q_out;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  int64_t ld;  // elements per row of qkv
  int64_t n_slots;
  int T, H, KV, ps, L;
  int chunk;   // tokens per workgroup of the cache's part, at most 64
  int cache_wgs;  // its workgroups per head
};

template <typename T>
PMI_DEV void load8(const T* p, float* v) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  const T8 x = *reinterpret_cast<const T8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
}
template <typename T>
PMI_DEV void store8(T* p, const float* v) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  T8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (T)v[e];
  *reinterpret_cast<T8*>(p) = x;
}

// The angles of pairs d .. d + 7 at a position.
template <int D>
PMI_DEV void load_angles(const AppendArgs& a, int d, int pos, float* c, float* s) {
  const f32x4* cp = reinterpret_cast<const f32x4*>(a.cos_t + (int64_t)pos * (D / 2) + d);
  const f32x4* sp = reinterpret_cast<const f32x4*>(a.sin_t + (int64_t)pos * (D / 2) + d);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const f32x4 x = cp[q], y = sp[q];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[4 * q + e] = x[e], s[4 * q + e] = y[e];
  }
}
PMI_DEV void rotate8(float* lo, float* hi, const float* c, const float* s) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x1 = lo[e], x2 = hi[e];
    lo[e] = x1 * c[e] - x2 * s[e];
    hi[e] = x2 * c[e] + x1 * s[e];
  }
}

// Pairs d .. d + 7 of one head's row, rotated: lo and hi are its two halves' parts.
template <typename T, int D>
PMI_DEV void rotated8(const AppendArgs& a, const T* row, int d, int pos, float* lo, float* hi) {
  float c[8], s[8];
  load8(row + d, lo);
  load8(row + d + D / 2, hi);
  load_angles<D>(a, d, pos, c, s);
  rotate8(lo, hi, c, s);
}

// Four values as codes: x * inv rounded to the nearest code, within +-top.
template <bool FP8>
PMI_DEV uint32_t code4(const float* x, float inv) {
  if constexpr (FP8) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fminf(fmaxf(x[e] * inv, -448.f), 448.f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int q = (int)fminf(fmaxf(rintf(x[e] * inv), -127.f), 127.f);
      w |= (uint32_t)(q & 255) << (8 * e);
    }
    return w;
  }
}
template <bool FP8>
PMI_DEV void decode4(uint32_t w, float* v) {
  if constexpr (FP8) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(w >> (8 * e));
  }
}

// |x| as bits: ordered as the values are, with infinities and NaN above them, so
// that a maximum keeps them and the page's scale shows them (as NaN).
PMI_DEV uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// What of a run stays on the chip between its maximum and its codes: 512 units of 16
// values, keys in registers (2 units a thread), values in LDS as they came.
constexpr int kHeldUnits = 2;
constexpr int kHeldBytes = 256 * kHeldUnits * 16 * 2;

// One run of new tokens, consecutive slots of one page, of one KV head: the larger
// of the page's scale and what they need; the codes of the tokens before them again
// where it grew; their own codes. All 256 threads. Runs of up to 64 tokens (D 128; 128
// of D 64) are read once, longer ones again for their codes.
template <typename T, int D, bool FP8>
PMI_DEV void append_run(const AppendArgs& a, int t0, int n, int slot, int kh, uint32_t* red, T* held) {
  constexpr float kTop = FP8 ? 448.f : 127.f;
  constexpr int kHeldRows = 256 * kHeldUnits * 16 / D;
  const int tid = threadIdx.x;
  const int page = slot / a.ps, first = slot - page * a.ps, units = n * (D / 16);
  const int64_t cell = (int64_t)page * a.KV + kh;
  const T* base = (const T*)a.qkv + (int64_t)(a.H + kh) * D;
  uint8_t* kc = a.k_cache + cell * a.ps * D;
  uint8_t* vc = a.v_cache + cell * a.ps * D;
  uint32_t mk = 0, mv = 0;
  float lo[kHeldUnits][8], hi[kHeldUnits][8];
  const auto turned = [&](int u, float* l, float* h) {
    const int i = u / (D / 16), pos = min(max(a.positions[t0 + i], 0), a.L - 1);
    rotated8<T, D>(a, base + (int64_t)(t0 + i) * a.ld, 8 * (u % (D / 16)), pos, l, h);
  };
  const auto largest = [&](uint32_t m, const float* l, const float* h) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, max(abs_bits(l[e]), abs_bits(h[e])));
    return m;
  };
  const auto values = [&](int u) { return base + (int64_t)(t0 + u / (D / 8)) * a.ld + (int64_t)a.KV * D + 8 * (u % (D / 8)); };
  typedef T T8 __attribute__((ext_vector_type(8)));
  const auto largest_value = [&](const T8& x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mv = max(mv, abs_bits((float)x[e]));
  };
  __syncthreads();  // red and held of the previous run are read
  {
    T8 x[2 * kHeldUnits];
#pragma unroll
    for (int j = 0; j < 2 * kHeldUnits; ++j)
      if (tid + 256 * j < 2 * units) x[j] = *reinterpret_cast<const T8*>(values(tid + 256 * j));
#pragma unroll
    for (int j = 0; j < kHeldUnits; ++j)
      if (tid + 256 * j < units) turned(tid + 256 * j, lo[j], hi[j]);
#pragma unroll
    for (int j = 0; j < 2 * kHeldUnits; ++j)
      if (tid + 256 * j < 2 * units) {
        reinterpret_cast<T8*>(held)[tid + 256 * j] = x[j];
        largest_value(x[j]);
      }
#pragma unroll
    for (int j = 0; j < kHeldUnits; ++j)
      if (tid + 256 * j < units) mk = largest(mk, lo[j], hi[j]);
  }
  for (int u = tid + 512 * kHeldUnits; u < 2 * units; u += 256)
    largest_value(*reinterpret_cast<const T8*>(values(u)));
  for (int u = tid + 256 * kHeldUnits; u < units; u += 256) {
    float l[8], h[8];
    turned(u, l, h);
    mk = largest(mk, l, h);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o));
  }
  if ((tid & 63) == 0) red[2 * (tid >> 6)] = mk, red[2 * (tid >> 6) + 1] = mv;
  const float before_k = first ? a.k_scale[cell] : 0.f, before_v = first ? a.v_scale[cell] : 0.f;
  __syncthreads();  // and everybody has the page's scales before they are replaced
#pragma unroll
  for (int w = 0; w < 4; ++w) mk = max(mk, red[2 * w]), mv = max(mv, red[2 * w + 1]);
  const float want_k = __builtin_bit_cast(float, mk) * (1.f / kTop), want_v = __builtin_bit_cast(float, mv) * (1.f / kTop);
  const bool grow_k = abs_bits(want_k) > abs_bits(before_k), grow_v = abs_bits(want_v) > abs_bits(before_v);
  // An infinity becomes NaN too: its page's codes times an infinite scale would be NaN, an infinity
  // of either sign or (a code of 0 written later) NaN again.
  const auto or_nan = [](float s) { return s < INFINITY ? s : __builtin_nanf(""); };
  const float sk = or_nan(grow_k ? want_k : before_k), sv = or_nan(grow_v ? want_v : before_v);
  // (finite, also for subnormal scales)
  const float inv_k = sk > 0.f ? fminf(1.f / sk, FLT_MAX) : 0.f, inv_v = sv > 0.f ? fminf(1.f / sv, FLT_MAX) : 0.f;
  if (tid == 0) a.k_scale[cell] = sk, a.v_scale[cell] = sv;

  if (first && grow_k) {
    const float f = before_k / sk;
    for (int u = tid; u < first * (D / 16); u += 256) {
      u32x4 w = *reinterpret_cast<u32x4*>(kc + 16 * u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[4];
        decode4<FP8>(w[e], v);
        w[e] = code4<FP8>(v, f);
      }
      *reinterpret_cast<u32x4*>(kc + 16 * u) = w;
    }
  }
  const auto store_key = [&](int u, const float* l, const float* h) {
    uint8_t* dst = kc + (first + u / (D / 16)) * D + 8 * (u % (D / 16));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<u32x2*>(dst) = u32x2{code4<FP8>(l, inv_k), code4<FP8>(l + 4, inv_k)};
    *reinterpret_cast<u32x2*>(dst + D / 2) = u32x2{code4<FP8>(h, inv_k), code4<FP8>(h + 4, inv_k)};
  };
#pragma unroll
  for (int j = 0; j < kHeldUnits; ++j)
    if (tid + 256 * j < units) store_key(tid + 256 * j, lo[j], hi[j]);
  for (int u = tid + 256 * kHeldUnits; u < units; u += 256) {
    float l[8], h[8];
    turned(u, l, h);
    store_key(u, l, h);
  }
  // v: one thread takes the 16 tokens of a block at one dimension
  const float fv = grow_v && first ? before_v / sv : 1.f;
  const int b0 = (grow_v ? 0 : first) / 16, b1 = (first + n + 15) / 16;
  for (int u = tid; u < (b1 - b0) * D; u += 256) {
    const int b = b0 + u / D, d = u % D;  // b is the same in a whole wave
    u32x4* at = reinterpret_cast<u32x4*>(vc + ((int64_t)b * D + d) * 16);
    u32x4 w = {0, 0, 0, 0};
    if (16 * b < first || 16 * b + 16 > first + n) w = *at;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j0 = 16 * b + 4 * q;  // token of the page
      float fresh[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = j0 + e - first;
        fresh[e] = 0.f;
        if (i >= 0 && i < n)
          fresh[e] = (float)(i < kHeldRows ? held[i * D + d] : base[(int64_t)(t0 + i) * a.ld + (int64_t)a.KV * D + d]);
      }
      const uint32_t cnew = code4<FP8>(fresh, inv_v);
      if (j0 >= first && j0 + 4 <= first + n) {
        w[q] = cnew;
      } else if (j0 < first + n) {
        float old[4];
        decode4<FP8>(w[q], old);
        const uint32_t cold = grow_v ? code4<FP8>(old, fv) : w[q];
        uint32_t o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + e;
          o |= (j < first ? cold : j < first + n ? cnew : w[q]) & (255u << (8 * e));
        }
        w[q] = o;
      }
    }
    *at = w;
  }
}

// Bound by the bytes of qkv and of the rotated q for many tokens (prompts of 6000 tokens, 28 / 4
// heads of 128, bf16, pages of 32 of e4m3: 20 us for 105 MB), by the chain slots, values, maximum, codes for few (64 tokens, 32 / 8 heads,
// pages of 64: 8 us). A run is read once: its keys wait for the maximum in registers, its
// values in LDS, from where a thread takes the 16 tokens of one dimension (6000 tokens: 33 us with a
// second read, a loop over the slots and the angles loaded for every head).
// Grid: (cache_wgs + query workgroups, KV). The first take `chunk` tokens of one KV
// head each and write the runs that begin among them; the others rotate the queries, a
// thread the same dimensions of the KV head's whole group, with one load of their angles.
template <typename T, int D, bool FP8>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  __shared__ uint32_t red[8];
  __shared__ int run_end;
  __shared__ __attribute__((aligned(16))) T held[kHeldBytes / sizeof(T)];
  const int tid = threadIdx.x, kh = blockIdx.y;
  if ((int)blockIdx.x >= a.cache_wgs) {
    const int g = a.H / a.KV;
    const int64_t u = (int64_t)(blockIdx.x - a.cache_wgs) * 256 + tid, t = u / (D / 16);
    const int d = 8 * (int)(u % (D / 16));
    if (t >= a.T) return;
    const int pos = min(max(a.positions[t], 0), a.L - 1);
    float c[8], s[8];
    load_angles<D>(a, d, pos, c, s);
    const T* src = (const T*)a.qkv + t * a.ld + (int64_t)kh * g * D + d;
    T* dst = (T*)a.q_out + (t * a.H + kh * g) * D + d;
#pragma unroll 4
    for (int h = 0; h < g; ++h) {
      float lo[8], hi[8];
      load8(src + h * D, lo);
      load8(src + h * D + D / 2, hi);
      rotate8(lo, hi, c, s);
      store8(dst + h * D, lo);
      store8(dst + h * D + D / 2, hi);
    }
    return;
  }
  // every wave looks at the whole chunk: lane l at its token l, and where runs begin
  const int lane = tid & 63, c0 = blockIdx.x * a.chunk, at = c0 + lane;
  int mine = -1, before = -1;
  if (lane < a.chunk && at < a.T) {
    mine = a.slots[at];
    if (at > 0) before = a.slots[at - 1];
  }
  const bool begins = mine >= 0 && mine < a.n_slots && !(mine % a.ps != 0 && before == mine - 1);
  for (uint64_t todo = __ballot(begins); todo; todo &= todo - 1) {
    const int l = __builtin_ctzll(todo), t = c0 + l;
    const int slot = __builtin_amdgcn_readlane(mine, l);
    const int room = min(a.ps - slot % a.ps, a.T - t);
    __syncthreads();
    if (tid == 0) run_end = room;
    __syncthreads();
    if (tid < room && a.slots[t + tid] != slot + tid) atomicMin(&run_end, tid);
    __syncthreads();
    append_run<T, D, FP8>(a, t, run_end, slot, kh, red, held);
  }
}

// ---- whole pages as values --------------------------------------------------------

// One workgroup per page and head; a thread takes 16 codes of a key, or four dimensions of a
// block of V, whose tokens are then four values a store (6.7 us with one dimension a thread, 6.0 so:
// 188 pages of 32 tokens, 4 heads of 128, bf16, 19 MB with the codes). Bound by the launch and the
// chain page, scale, codes, values, then by the bytes of the values.
template <typename T, bool FP8>
__global__ __launch_bounds__(256) void read_pages_kernel(const int32_t* __restrict__ pages,
                                                         const uint8_t* __restrict__ k_cache,
                                                         const uint8_t* __restrict__ v_cache,
                                                         const float* __restrict__ k_scale,
                                                         const float* __restrict__ v_scale, T* __restrict__ k_out,
                                                         T* __restrict__ v_out, int64_t n_pages, int KV, int ps, int D) {
  const int i = blockIdx.x / KV, kh = blockIdx.x - i * KV;
  const int page = pages[i];
  const bool ok = page >= 0 && page < n_pages;
  const int64_t cell = ok ? (int64_t)page * KV + kh : 0;
  const int64_t out = (int64_t)blockIdx.x * ps * D;
  const float sk = ok ? k_scale[cell] : 0.f, sv = ok ? v_scale[cell] : 0.f;
  const int units = ps * D / 16;  // 16 codes
  const u32x4* k_codes = reinterpret_cast<const u32x4*>(k_cache + cell * ps * D);
  const u32x4* v_codes = reinterpret_cast<const u32x4*>(v_cache + cell * ps * D);
  const u32x4 none = {0, 0, 0, 0};
  for (int u = threadIdx.x; u < units + units / 4; u += 256) {
    if (u < units) {
      const u32x4 w = ok ? k_codes[u] : none;
      float v[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) decode4<FP8>(w[q], v + 4 * q);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = ok ? v[e] * sk : 0.f;
      store8(k_out + out + 16 * u, v);
      store8(k_out + out + 16 * u + 8, v + 8);
      continue;
    }
    const int b = 4 * (u - units) / D, d = 4 * (u - units) - b * D;
    u32x4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = ok ? v_codes[b * D + d + j] : none;
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // four tokens of four dimensions
      float v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) decode4<FP8>(w[j][q], v[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (T)(ok ? v[j][e] * sv : 0.f);
        *reinterpret_cast<T4*>(v_out + out + (int64_t)(16 * b + 4 * q + e) * D + d) = y;
      }
    }
  }
}

}  // namespace

hipError_t launch_extend_tables(const PagedTables& t, hipStream_t stream) {
  TablesArgs a = {t.tables,    t.stride,      t.kv_lens, t.new_lens, t.free_pages, t.pool,
                  t.q_starts,  t.kv_lens_out, t.first,   t.fresh,    t.positions,  t.slots,
                  t.pool_out,
                  (int)t.R,    (int)t.width,  (int)t.ring, (int)t.ps, (int)t.total, t.max_len};
  // One workgroup looks up 1024 tokens at a time; past a few rounds a grid is quicker (700
  // requests of 16-token pages, 270000 tokens: 23 + 5 us with the pages in the one workgroup).
  const bool fill = t.total <= 4096;
  hipLaunchKernelGGL(extend_tables_kernel, dim3(1), dim3(1024), 0, stream, a, fill ? 1 : 0);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || fill) return e;
  hipLaunchKernelGGL(fill_tables_kernel, dim3((unsigned)((t.total + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_release_tables(const int32_t* tables, int64_t stride, int32_t* kv_lens, const uint8_t* done,
                                 int32_t* free_pages, int32_t* pool, int64_t R, int64_t width, int64_t ring,
                                 int64_t ps, hipStream_t stream) {
  hipLaunchKernelGGL(release_tables_kernel, dim3(1), dim3(1024), 0, stream, tables, stride, kv_lens, done, free_pages,
                     pool, (int)R, (int)width, (int)ring, (int)ps);
  return hipGetLastError();
}

namespace {
template <typename T, int D, bool FP8>
hipError_t append(const AppendArgs& a, int64_t query_wgs, hipStream_t stream) {
  hipLaunchKernelGGL((append_kernel<T, D, FP8>), dim3((unsigned)(a.cache_wgs + query_wgs), (unsigned)a.KV), dim3(256),
                     0, stream, a);
  return hipGetLastError();
}
template <typename T>
hipError_t append_t(const AppendArgs& a, int D, bool fp8, int64_t wgs, hipStream_t stream) {
  if (D == 64) return fp8 ? append<T, 64, true>(a, wgs, stream) : append<T, 64, false>(a, wgs, stream);
  return fp8 ? append<T, 128, true>(a, wgs, stream) : append<T, 128, false>(a, wgs, stream);
}
}  // namespace

hipError_t launch_append_kv(const PagedCache& c, const void* qkv, int64_t ld, bool bf16, const float* cos_t,
                            const float* sin_t, int64_t L, const int32_t* positions, const int32_t* slots, void* q_out,
                            int64_t T, int64_t H, hipStream_t stream) {
  AppendArgs a = {qkv, cos_t, sin_t, positions, slots, q_out, (uint8_t*)c.k, (uint8_t*)c.v, c.k_scale, c.v_scale,
                  ld, c.pages * c.ps, (int)T, (int)H, (int)c.KV, (int)c.ps, (int)L, 0, 0};
  // Few tokens are mostly one run each (a decode step): a workgroup for each of them.
  // Many are mostly runs of whole pages, and a run falls to where it begins: chunks of 8
  // spread those over the XCDs (7 prompts of 6000 tokens in pages of 32, 28 / 4 heads, with
  // the read of their pages: 25.2 us; chunks of 4 27.2, of 16 28.4, of 32 26.8, of 2 40.9).
  a.chunk = T <= 1024 ? 1 : 8;
  a.cache_wgs = (int)((T + a.chunk - 1) / a.chunk);
  const int64_t wgs = (T * (c.D / 16) + 255) / 256;
  return bf16 ? append_t<__bf16>(a, (int)c.D, c.fp8, wgs, stream) : append_t<f16>(a, (int)c.D, c.fp8, wgs, stream);
}

namespace {
template <typename T>
hipError_t read_t(const PagedCache& c, const int32_t* pages, void* k, void* v, int64_t n, hipStream_t stream) {
  const dim3 grid((unsigned)(n * c.KV));
  if (c.fp8)
    hipLaunchKernelGGL((read_pages_kernel<T, true>), grid, dim3(256), 0, stream, pages, (const uint8_t*)c.k,
                       (const uint8_t*)c.v, c.k_scale, c.v_scale, (T*)k, (T*)v, c.pages, (int)c.KV, (int)c.ps,
                       (int)c.D);
  else
    hipLaunchKernelGGL((read_pages_kernel<T, false>), grid, dim3(256), 0, stream, pages, (const uint8_t*)c.k,
                       (const uint8_t*)c.v, c.k_scale, c.v_scale, (T*)k, (T*)v, c.pages, (int)c.KV, (int)c.ps,
                       (int)c.D);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_read_pages(const PagedCache& c, const int32_t* pages, int out_dtype, void* k, void* v, int64_t n,
                             hipStream_t stream) {
  if (out_dtype == 0) return read_t<f16>(c, pages, k, v, n, stream);
  if (out_dtype == 1) return read_t<__bf16>(c, pages, k, v, n, stream);
  return read_t<float>(c, pages, k, v, n, stream);
}

}  // namespace pmi
