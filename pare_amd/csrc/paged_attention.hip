// Attention over the paged 8-bit cache (paged_kv.hip describes it).
//
// A query i of a request with n queries and a length of L keys sees positions
// p <= L - n + i (and p > L - n + i - window):
//   o = sum_p e_p (vs_p v_p) / sum_p e_p,   e_p = exp(scale q . (ks_p k_p) - max)
// with the codes k_p, v_p and their pages' scales. A query that sees nothing gives 0.
#include <type_traits>

#include "paged.h"
#include "pmi_common.h"
#include "pmi_launch.h"

namespace pmi {
namespace {

struct AttnArgs {
  const void* q;
  void* out;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  const int32_t* tables;
  const int32_t* kv_lens;
  const int32_t* q_starts;
  int64_t stride, q_token, q_head, n_pages;
  int T, R, width, H, KV, ps, ps_log, window;
  float scale;
  // split over the keys: `per` positions a workgroup, at most S of them
  int per, S, row_tiles, max_q, max_kv;
  int* counters;
  float* part;
};

// ---- operands from codes ----------------------------------------------------------
// Eight codes (two words) as fp16, exact: e4m3 by the conversion, int8 c as 1152 + c
// (c + 128 under a 0x64 exponent byte) - 1152.
template <bool FP8>
PMI_DEV f16x8 codes8(uint32_t a, uint32_t b) {
  if constexpr (FP8) {
    const f16x2 r0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.f, false);
    const f16x2 r1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.f, true);
    const f16x2 r2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.f, false);
    const f16x2 r3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.f, true);
    return __builtin_bit_cast(f16x8, u32x4{as_u32(r0), as_u32(r1), as_u32(r2), as_u32(r3)});
  } else {
    const uint32_t K = 0x64646464u;
    const f16x2 off = {(f16)-1152.f, (f16)-1152.f};
    a ^= 0x80808080u, b ^= 0x80808080u;
    const f16x2 r0 = as_f16x2(__builtin_amdgcn_perm(K, a, 0x04010400u)) + off;
    const f16x2 r1 = as_f16x2(__builtin_amdgcn_perm(K, a, 0x04030402u)) + off;
    const f16x2 r2 = as_f16x2(__builtin_amdgcn_perm(K, b, 0x04010400u)) + off;
    const f16x2 r3 = as_f16x2(__builtin_amdgcn_perm(K, b, 0x04030402u)) + off;
    return __builtin_bit_cast(f16x8, u32x4{as_u32(r0), as_u32(r1), as_u32(r2), as_u32(r3)});
  }
}

// Masks of the bytes first .. last - 1 of 16.
PMI_DEV u32x4 byte_mask(int first, int last) {
  u32x4 m;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int f = min(max(first - 4 * e, 0), 4), t = min(max(last - 4 * e, 0), 4);
    const uint32_t below = f == 4 ? 0xffffffffu : (1u << (8 * f)) - 1, upto = t == 4 ? 0xffffffffu : (1u << (8 * t)) - 1;
    m[e] = upto & ~below;
  }
  return m;
}

// A row of q as fp16 that the products take exactly: bf16 rows are scaled by a power of two
// to a largest value in [1, 2) (what falls under 2^-24 of it is lost to fp16's range, and
// is 2^-16 of bf16's own rounding of the largest). mul takes the power back.
template <typename T, int D>
struct QueryRow {
  f16x8 v[D / 32];
  float mul;
};

// Lane (c = l % 16, h = l / 16) of the tile's column c: step 2 j + s holds dimensions 64 j +
// 16 h + 8 s .. + 7, the order in which a lane's 16-byte piece of a key gives them.
template <typename T, int D>
PMI_DEV void load_query(QueryRow<T, D>& q, const T* row, bool live, int h) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  T8 raw[D / 32];
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      T8 z = {};
      if (live) z = *reinterpret_cast<const T8*>(row + 64 * j + 16 * h + 8 * s);
      raw[2 * j + s] = z;
    }
  q.mul = 1.f;
  if constexpr (sizeof(T) == 2 && !__is_same(T, f16)) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf((float)raw[i][e]));
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    // 2^-exponent as bits; rows of zeros (or subnormals), infinities keep 1
    const uint32_t e = __builtin_bit_cast(uint32_t, m) >> 23;
    const bool ok = e >= 1 && e <= 253;
    const float down = ok ? __builtin_bit_cast(float, (254u - e) << 23) : 1.f;
    q.mul = ok ? __builtin_bit_cast(float, e << 23) : 1.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) q.v[i][x] = (f16)((float)raw[i][x] * down);
  } else {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q.v[i] = __builtin_bit_cast(f16x8, raw[i]);
  }
}

PMI_DEV float max_over_h(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
PMI_DEV float sum_over_h(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// (m, l, o) joined with another part of the same row; a part that saw no key is left out.
PMI_DEV void join(float& m, float& l, f32x4& o, float pm, float pl, f32x4 po, bool use) {
  use = use && !(pm == -INFINITY && pl == 0.f);
  const float nm = fmaxf(m, pm);
  const float fo = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nm), fn = __builtin_amdgcn_exp2f(pm - nm);
  l = use ? fmaf(l, fo, pl * fn) : l;
#pragma unroll
  for (int x = 0; x < 4; ++x) o[x] = use ? fmaf(o[x], fo, po[x] * fn) : o[x];
  m = use ? nm : m;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPBias = 16384.f;  // probabilities are held in fp16 times this

// ---- few query rows ------------------------------------------------------------------
// Up to 16 query rows (tokens x heads of one KV head) per workgroup against a range of
// keys: bound by the bytes of the codes. Four waves take the range's 64-token tiles in
// turn. All operands come straight from memory to registers:
//   S^T = K q^T: 16x16x32 fp16 products, rows = tokens. Row m of product t is token
//     16 (m / 4) + 4 t + m % 4 of the tile, so that a lane's results of the four products
//     are 16 consecutive tokens, 16 h .. 16 h + 15 (h = lane / 16), all of one page;
//   O^T = V^T P^T: a lane's operand of P is then what it holds, and that of V its 16-byte
//     piece of the page's block (one dimension, 16 tokens).
// Scales: a lane's 16 tokens share theirs, so ks multiplies the scores and vs the
// probabilities, in fp32, before these become fp16: times vs / (largest vs of the range)
// and 2^14, so that they use fp16's range from the top.
constexpr int64_t kFewWgs = 1024;

template <typename T, int D, bool FP8>
__global__ __launch_bounds__(256, 2) void attention_few_kernel(AttnArgs a) {
  constexpr int DT = D / 16;  // 16-dimension tiles of the output
  __shared__ float s_acc[4][16][D];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_last;
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = l & 15, h = l >> 4;
  const int sp = blockIdx.x, kh = blockIdx.y % a.KV, rt = blockIdx.y / a.KV;
  const int r = blockIdx.z;
  const int G = a.H / a.KV;
  // What does not hang on another load is loaded first: lengths, and the pages of a range that
  // begins at a multiple of `per`.
  const int32_t* table = a.tables + (int64_t)r * a.stride;
  auto look_up = [&](int p) { return table[min((p + 16 * h) >> a.ps_log, a.width - 1)]; };
  int early0 = -1, early1 = -1;
  if (!a.window && a.width > 0) {
    early0 = look_up(sp * a.per + 64 * wave);
    early1 = look_up(sp * a.per + 64 * wave + 256);
  }
  const int len0 = a.kv_lens[r];
  int start = r, n = 1;
  if (a.q_starts) {
    start = a.q_starts[r];
    n = a.q_starts[r + 1] - start;
  }
  const int len = min(min(max(len0, 0), a.max_kv), a.width * a.ps);
  // the limits of queries are set by what the request has, also past max_q
  const int shift = len - n;
  n = min(n, a.max_q);
  const int rows = n * G - rt * 16;  // of this tile and the ones behind it
  if (rows <= 0 || start < 0 || (int64_t)start + n > a.T) return;
  const int row = rt * 16 + c;
  const bool live = c < rows;
  const int i = row / G;
  // positions that this column's query sees: [lo, hi)
  const int hi = live ? max(0, min(len, shift + i + 1)) : 0;
  const int lo = a.window ? max(0, shift + i + 1 - a.window) : 0;
  const int i_first = rt * 16 / G, i_last = (rt * 16 + min(rows, 16) - 1) / G;
  const int all_hi = a.n_pages ? max(0, min(len, shift + i_last + 1)) : 0;
  const int first_seen = a.window ? max(0, shift + i_first + 1 - a.window) : 0, all_lo = first_seen & ~15;
  const int range = max(0, all_hi - all_lo);
  const int splits = max(1, (range + a.per - 1) / a.per);
  if (sp >= splits) return;
  const int p0 = all_lo + sp * a.per, p1 = min(all_hi, p0 + a.per);
  // tiles inside of [safe_lo, safe_hi) need no mask
  const int safe_hi = max(0, min(len, shift + i_first + 1));
  const int safe_lo = a.window ? max(0, shift + i_last + 1 - a.window) : 0;

  QueryRow<T, D> q;
  load_query<T, D>(q, (const T*)a.q + (int64_t)(start + (live ? i : 0)) * a.q_token +
                          (int64_t)(kh * G + (live ? row - i * G : 0)) * a.q_head, live, h);
  const float qmul = q.mul * a.scale * kLog2e;

  f32x4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, sum = 0.f, vref = 0.f;
  const int64_t cell_bytes = (int64_t)a.ps * D;

  // Look-ups run ahead: a tile's entry of the table (of the lane's 16 tokens, block h) is loaded
  // two tiles before it, its scales and keys one, its values half a tile. Every load of the main
  // loop is issued on every pass, at a place inside the cache (page 0 for entries outside it, which
  // are masked): behind a branch the compiler can no longer tell how many are younger than the
  // one it waits for, and waits for all of them.
  u32x4 kw[D / 16], vw[DT];
  auto valid = [&](int entry, int p) { return p + 16 * h < p1 && (unsigned)entry < a.n_pages ? entry : -1; };
  auto load_k = [&](int page, int p) {
    const int b = (l >> 2) & 3;  // the block of the lane's row
    const int64_t cell = (int64_t)max(__shfl(page, 16 * b), 0) * a.KV + kh;
    const uint8_t* at = a.k + cell * cell_bytes + (((p + 16 * b) & (a.ps - 1)) + (l & 3)) * D + 16 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
        kw[t * (D / 64) + j] = *reinterpret_cast<const u32x4*>(at + 4 * t * D + 64 * j);
  };
  auto load_v = [&](int page, int p) {
    const int64_t cell = (int64_t)max(page, 0) * a.KV + kh;
    const uint8_t* at = a.v + cell * cell_bytes + ((((p + 16 * h) & (a.ps - 1)) >> 4) * D + c) * 16;
#pragma unroll
    for (int d = 0; d < DT; ++d) vw[d] = *reinterpret_cast<const u32x4*>(at + 256 * d);
  };
  int p = p0 + 64 * wave;
  int page = -1, entry = -1;
  float bks = 0.f, bvs = 0.f;  // scales of the lane's block
  auto load_scales = [&](int pg) {
    const int64_t cell = (int64_t)max(pg, 0) * a.KV + kh;
    bks = a.k_scale[cell];
    bvs = a.v_scale[cell];
  };
  auto tile = [&](auto last) {
    constexpr bool kLast = decltype(last)::value;
    const bool gone = page < 0;
    const float ks = gone ? 0.f : bks * qmul, tvs = gone ? 0.f : bvs;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const u32x4 w = kw[t * (D / 64) + j];
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FP8>(w[0], w[1]), q.v[2 * j], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FP8>(w[2], w[3]), q.v[2 * j + 1], s[t], 0, 0, 0);
      }
    }
    int next_page = -1;
    if constexpr (!kLast) {
      next_page = valid(entry, p + 256);
      load_scales(next_page);
      entry = look_up(p + 512);
      load_k(next_page, p + 256);
    }
    // the largest value scale so far is the unit of acc
    const float top = fmaxf(vref, max_over_h(tvs < INFINITY ? tvs : 0.f));
    if (__any(top > vref)) {
      const float f = vref > 0.f ? vref / top : 1.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
      vref = top;
    }
    const float vs = vref > 0.f ? tvs * (kPBias / vref) : 0.f;
    const bool masked = p < safe_lo || p + 64 > safe_hi || p + 64 > p1 || __any(gone);
    const int at = p + 16 * h;
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = s[e >> 2][e & 3] * ks;
    if (masked) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = !gone && at + e >= lo && at + e < min(hi, p1) ? x[e] : -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, x[e]);
    mx = max_over_h(mx);
    const float nm = fmaxf(m, mx);
    if (__any(nm > m)) {
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nm);
      sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
      m = nm;
    }
    const float base = m == -INFINITY ? 0.f : m;
    f16x8 pw[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float ex = __builtin_amdgcn_exp2f(x[e] - base);
      sum += ex;
      float w = ex * vs;
      if (masked) w = x[e] == -INFINITY ? 0.f : w;
      pw[e >> 3][e & 7] = (f16)w;
    }
    if (FP8 && masked) {
      // codes of tokens that no row sees may be NaN
      const u32x4 keep = byte_mask(first_seen - at, gone ? 0 : p1 - at);
#pragma unroll
      for (int d = 0; d < DT; ++d) vw[d] &= keep;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FP8>(vw[d][0], vw[d][1]), pw[0], acc[d], 0, 0, 0);
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FP8>(vw[d][2], vw[d][3]), pw[1], acc[d], 0, 0, 0);
    }
    if constexpr (!kLast) {
      load_v(next_page, p + 256);
      page = next_page;
    }
  };
  if (p < p1) {
    page = valid(a.window ? look_up(p) : early0, p);
    entry = a.window ? look_up(p + 256) : early1;
    load_scales(page);
    load_k(page, p);
    load_v(page, p);
    for (; p + 256 < p1; p += 256) tile(std::false_type{});
    tile(std::true_type{});
  }

  // the four waves' results, joined in their order
  sum = sum_over_h(sum);
  const float unit = vref * (1.f / kPBias);
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&s_acc[wave][c][16 * d + 4 * h]) = acc[d] * unit;
  if (h == 0) s_m[wave][c] = m, s_l[wave][c] = sum;
  __syncthreads();
  constexpr int kPer = D / 16;  // dimensions per thread: 16 threads a row
  const int orow = tid >> 4, od = (tid & 15) * kPer;
  float om = -INFINITY, ol = 0.f, o[kPer];
#pragma unroll
  for (int w = 0; w < 4; ++w) om = fmaxf(om, s_m[w][orow]);
#pragma unroll
  for (int x = 0; x < kPer; ++x) o[x] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = s_m[w][orow] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][orow] - om);
    ol = fmaf(s_l[w][orow], f, ol);
    // (a wave without a key it sees holds zeros, or NaN of a page that shows them)
#pragma unroll
    for (int x = 0; x < kPer; ++x) o[x] = f == 0.f ? o[x] : fmaf(s_acc[w][orow][od + x], f, o[x]);
  }
  const int grow = rt * 16 + orow;
  const bool mine = orow < rows;
  T* dst = (T*)a.out + ((int64_t)(start + grow / G) * a.H + kh * G + grow % G) * D + od;
  auto store = [&](float inv) {
    typedef T Tv __attribute__((ext_vector_type(kPer)));
    Tv y;
#pragma unroll
    for (int x = 0; x < kPer; ++x) y[x] = (T)(o[x] * inv);
    if (mine) *reinterpret_cast<Tv*>(dst) = y;
  };
  if (splits == 1) {
    store(ol > 0.f ? 1.f / ol : (ol != ol ? ol : 0.f));
    return;
  }

  // Partial rows to the workspace; the last workgroup of the item to arrive joins them in
  // split order. Stores and loads are coherent across the XCDs' L2 caches (sc1).
  constexpr int kSc1 = 16, kRec = D + 4;  // floats of a row: values, max, sum
  const int item = (r * a.row_tiles + rt) * a.KV + kh;
  const int tile_rows = min(16, a.max_q * G);
  float* base = a.part + (int64_t)item * a.S * tile_rows * kRec;
  const __amdgpu_buffer_rsrc_t rp = rsrc(base, (int64_t)a.S * tile_rows * kRec * 4);
  const int rec = (sp * tile_rows + orow) * kRec * 4;
  if (mine) {
#pragma unroll
    for (int x = 0; x < kPer; x += 4)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{o[x], o[x + 1], o[x + 2], o[x + 3]}), rp,
                                             rec + 4 * (od + x), 0, kSc1);
    if ((tid & 15) == 0) {
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, om), rp, rec + 4 * D, 0, kSc1);
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, ol), rp, rec + 4 * D + 4, 0, kSc1);
    }
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const int old = __hip_atomic_fetch_add(&a.counters[item], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == splits - 1;
  }
  __syncthreads();
  if (!s_last) return;
  // All threads: D / 4 of them a row, rows x G groups of splits, joined through LDS.
  constexpr int kRowThreads = D / 4, kRowSlots = 256 / kRowThreads;
  const int slot = tid / kRowThreads, dim = 4 * (tid % kRowThreads);
  const int n_rows = min(rows, 16);
  const int groups = n_rows >= kRowSlots ? 1 : kRowSlots / n_rows;  // groups of splits a row
  for (int r0 = 0; r0 < n_rows; r0 += kRowSlots) {
    const int left = min(n_rows - r0, kRowSlots);
    const int jr = slot % left, grp = slot / left;
    const bool on = grp < groups;
    float jm = -INFINITY, jl = 0.f;
    f32x4 jo = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = on ? grp : splits; s0 < splits; s0 += 8 * groups) {
      float ms[8], ls[8];
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int off = (min(s0 + k * groups, splits - 1) * tile_rows + r0 + jr) * kRec * 4;
        ms[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, off + 4 * D, 0, kSc1));
        ls[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, off + 4 * D + 4, 0, kSc1));
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, off + 4 * dim, 0, kSc1));
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads stay together, ahead of their uses
#pragma unroll
      for (int k = 0; k < 8; ++k) join(jm, jl, jo, ms[k], ls[k], v[k], s0 + k * groups < splits);
    }
    __syncthreads();
    float* mine_f = &s_acc[0][0][0] + slot * (D + 2);
    *reinterpret_cast<float2*>(mine_f) = float2{jm, jl};
#pragma unroll
    for (int x = 0; x < 4; ++x) mine_f[2 + dim + x] = jo[x];
    __syncthreads();
    if (slot < left) {
      jm = -INFINITY, jl = 0.f, jo = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int g = 0; g < groups; ++g) {
        const float* f = &s_acc[0][0][0] + (slot + g * left) * (D + 2);
        join(jm, jl, jo, f[0], f[1], f32x4{f[2 + dim], f[3 + dim], f[4 + dim], f[5 + dim]}, true);
      }
      const float inv = jl > 0.f ? 1.f / jl : (jl != jl ? jl : 0.f);
      const int row1 = rt * 16 + r0 + slot;
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = (T)(jo[x] * inv);
      *reinterpret_cast<T4*>((T*)a.out + ((int64_t)(start + row1 / G) * a.H + kh * G + row1 % G) * D + dim) = y;
    }
  }
  if (tid == 0) __hip_atomic_store(&a.counters[item], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T, int D>
hipError_t few(const AttnArgs& a, bool fp8, hipStream_t stream) {
  const dim3 grid((unsigned)a.S, (unsigned)(a.KV * a.row_tiles), (unsigned)a.R);
  if (fp8)
    hipLaunchKernelGGL((attention_few_kernel<T, D, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attention_few_kernel<T, D, false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

struct FewPlan {
  int row_tiles, per, S;
  size_t part;
};
FewPlan few_plan(const PagedAttention& p, const PagedCache& c) {
  FewPlan f;
  const int64_t G = p.H / c.KV;
  f.row_tiles = (int)((p.max_q * G + 15) / 16);
  const int64_t range = p.window ? (p.max_kv < p.window + p.max_q + 15 ? p.max_kv : p.window + p.max_q + 15) : p.max_kv;
  const int64_t items = p.R * c.KV * f.row_tiles;
  // Up to kFewWgs workgroups where the range allows it, 256 tokens (a tile a wave) each or more.
  int64_t S = items > (int64_t)kWsCounterBytes / 4 ? 1 : kFewWgs / items;
  if (S < 1) S = 1;
  f.per = (int)(((range + S - 1) / S + 255) / 256 * 256);
  if (f.per < 256) f.per = 256;
  f.S = (int)((range + f.per - 1) / f.per);
  if (f.S < 1) f.S = 1;
  const int64_t rows = p.max_q * G < 16 ? p.max_q * G : 16;
  f.part = f.S > 1 ? (size_t)(items * f.S * rows * (c.D + 4) * 4) : 0;
  return f;
}

}  // namespace

size_t paged_attention_ws_bytes(const PagedAttention& p, const PagedCache& c) {
  const FewPlan f = few_plan(p, c);
  return f.part ? kWsCounterBytes + f.part : 0;
}

hipError_t launch_paged_attention(const PagedAttention& p, const PagedCache& c, void* workspace, size_t ws_bytes,
                                  hipStream_t stream) {
  AttnArgs a = {p.q, p.out, (const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, p.tables, p.kv_lens,
                p.q_starts, p.stride, p.q_token, p.q_head, c.pages, (int)p.T, (int)p.R, (int)p.width, (int)p.H,
                (int)c.KV, (int)c.ps, __builtin_ctz((unsigned)c.ps), (int)p.window, p.scale};
  const FewPlan f = few_plan(p, c);
  a.per = f.per, a.S = f.S, a.row_tiles = f.row_tiles, a.max_q = (int)p.max_q, a.max_kv = (int)p.max_kv;
  a.counters = (int*)workspace;
  a.part = (float*)((char*)workspace + kWsCounterBytes);
  if (p.bf16) return c.D == 64 ? few<__bf16, 64>(a, c.fp8, stream) : few<__bf16, 128>(a, c.fp8, stream);
  return c.D == 64 ? few<f16, 64>(a, c.fp8, stream) : few<f16, 128>(a, c.fp8, stream);
}

}  // namespace pmi
