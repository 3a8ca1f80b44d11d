// Attention over the paged 8-bit cache (paged_kv.hip describes it).
//
// A query i of a request with n queries and a length of L keys sees positions
// p <= L - n + i (and p > L - n + i - window):
//   o = sum_p e_p (vs_p v_p) / sum_p e_p,   e_p = exp(scale q . (ks_p k_p) - max)
// with the codes k_p, v_p and their pages' scales. A query that sees nothing gives 0.
#include <cfloat>
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
  int max_q, max_kv;
  int splits, per;  // many rows: ranges of keys, and tokens in one
  int few_rows;   // requests of up to so many query rows (tokens x heads of a KV head) are `few`
  int few_wgs;    // workgroups of the few-row part
  int* counters;  // one of each of them, and behind them one of each item of many rows
  float *few_part, *many_part;
  // runs of requests with the same first pages (kParts)
  const int4* runs;         // [R] first request, first query, queries, keys; no queries: none
  const int32_t* run_lens;  // [R] positions that a request shares
  int run_rows;       // runs of up to so many query rows are `few`
  int many_wgs;       // workgroups that the ranges of a run's keys are made for
  // Parts of rows, D + 4 floats each (values, max, sum): of several ranges of runs of many rows, in
  // tiles of kRows; of runs in one range or of few rows [2, T, H] (the second for the second half of a
  // tile's keys); of the keys behind what is shared [T, H].
  float *parts_many, *parts_one, *parts_own;
  int2* where;        // [T, H] a row's first shared part (its offset from parts_many in records), and 4 n + a
                      // of n parts that lie kRows (a = 0), kRows / 2 (1) or T H records (2) apart
  int part_records;   // that parts_many and parts_one hold
};

// What a launch computes: whole rows; or, where requests share their first pages, parts of
// rows. A run is then a request whose queries are those of all its members and whose keys are the
// shared ones, which all of its queries see; each member has the keys behind them for itself. All
// parts are of one launch, and a second one joins them (join_parts_kernel). Numbers 2 r are
// the requests, 2 r + 1 the runs.
enum Mode { kWhole, kParts };

// What a request's queries see, from its row of kv_lens and q_starts.
struct Request {
  int row;            // of the tables
  bool run;
  int start, n;       // its queries (none: nothing to do)
  int len, shift;     // its keys, of those within the bounds; query i sees positions up to shift + i
  int first_seen;     // the first position that its first query sees
  int lo, hi;         // positions that any of its queries sees: [lo, hi), lo a multiple of 16
};
// The first position that a query sees whose last is `last` (negative ones see nothing, and a
// large window less them would leave the integers).
PMI_DEV int first_position(const AttnArgs& a, int last) { return a.window && last >= a.window ? last + 1 - a.window : 0; }
// Positions that are shared, in whole pages.
PMI_DEV int shared_len(const AttnArgs& a, int len) { return min(max(len, 0), a.width * a.ps) & ~(a.ps - 1); }
template <Mode MODE>
PMI_DEV Request request(const AttnArgs& a, int r) {
  Request q;
  q.run = MODE == kParts && (r & 1);
  if constexpr (MODE == kParts) r >>= 1;
  if (q.run) {
    const int4 run = a.runs[r];
    const bool there = run.x >= 0 && run.x < a.R && run.y >= 0 && run.z > 0 && (int64_t)run.y + run.z <= a.T;
    q.row = there ? run.x : 0;
    q.start = there ? run.y : 0;
    q.len = there ? min(shared_len(a, run.w), a.max_kv) : 0;
    q.n = q.len ? run.z : 0;
    q.shift = q.len;  // (all queries see all of them)
    q.first_seen = q.lo = 0;
    q.hi = a.n_pages ? q.len : 0;
    return q;
  }
  const int len0 = a.kv_lens[r];
  q.row = r;
  q.start = r, q.n = 1;
  if (a.q_starts) {
    q.start = a.q_starts[r];
    q.n = a.q_starts[r + 1] - q.start;
  }
  q.len = min(min(max(len0, 0), a.max_kv), a.width * a.ps);
  q.shift = max(len0, 0) - q.n;  // (with the keys past the bounds and the queries past max_q)
  q.n = min(q.n, a.max_q);
  if (q.n < 0 || q.start < 0 || (int64_t)q.start + q.n > a.T) q.n = 0;
  if constexpr (MODE == kParts) {
    const int len = shared_len(a, a.run_lens[r]);
    q.first_seen = q.shift + 1 > len ? min(len, q.len) : 0;  // (none of its own queries may lie among them)
  } else {
    q.first_seen = min(first_position(a, q.shift), q.len);
  }
  q.lo = q.first_seen & ~15;
  q.hi = a.n_pages ? max(q.lo, min(q.len, q.shift + q.n)) : q.lo;
  return q;
}

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

// 2^e <= m < 2^(e + 1) as `up`, and its inverse, both finite and normal: e from -126 (also
// of zero and subnormal m) to 113 (also of larger, infinite and NaN m).
struct PowerOfTwo {
  float up, down;
};
PMI_DEV PowerOfTwo power_below(float m) {
  const uint32_t e = min(max(__builtin_bit_cast(uint32_t, m) >> 23, 1u), 240u);
  return {__builtin_bit_cast(float, e << 23), __builtin_bit_cast(float, (254u - e) << 23)};
}

// A row of q as fp16 that the products take exactly: bf16 rows are scaled by a power of two
// to a largest value in [1, 2) (what falls under 2^-24 of it is lost to fp16's range, and
// is 2^-16 of bf16's own rounding of the largest), at most 2^15 of rows from 2^114 on, so that
// the power times the scale stays finite. mul takes the power back.
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
    const PowerOfTwo w = power_below(m);
    q.mul = w.up;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) q.v[i][x] = (f16)((float)raw[i][x] * w.down);
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

// The largest of each four neighbouring lanes.
PMI_DEV float max_of_4(float v) {
  const auto from = [](float x, auto ctrl) {
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = fmaxf(v, from(v, std::integral_constant<int, 0xb1>{}));         // quad_perm 1, 0, 3, 2
  return fmaxf(v, from(v, std::integral_constant<int, 0x4e>{}));      // quad_perm 2, 3, 0, 1
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
// Probabilities, times their page's value scale, are held in fp16: as 2^kPBias of the largest of
// them that the row has seen (2^weight), so that neither a page of large values without weight nor
// one that the row does not see pushes the others out of fp16's range. Neither that reference nor
// the one that the scores are taken off (2^max) is raised before it has grown 2^kSlack-fold: raising one
// rescales all sums, and some row of a tile has a new maximum more often than not. 2^8 2^6 < 65504, and
// what is lost under fp16's range is below 2^-25 / 2^8 of the largest product.
// weight is at least max + kLeastWeight, so that their quotient is finite: values under 2^-24 of
// 2^kLeastWeight are lost.
constexpr float kPBias = 8.f, kSlack = 6.f, kLeastWeight = -100.f;

// The two references of a row, and what they make of the values' scales. All -inf: nothing seen.
struct Row {
  float max = -INFINITY, weight = -INFINITY;
  float gain = 0.f;  // 2^(max - weight + kPBias)
};
// Raises them; what the row's sum and its accumulators have to be multiplied with.
struct Rescale {
  float sum, acc;
};
PMI_DEV Rescale raise(Row& r, float max, float weight) {
  weight = fmaxf(fmaxf(r.weight, weight), max + kLeastWeight);
  const Rescale f = {r.max == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r.max - max),
                     r.weight == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r.weight - weight)};
  r.max = max, r.weight = weight;
  r.gain = max == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(max - weight + kPBias);
  return f;
}
// What the accumulators count in.
PMI_DEV float unit_of(const Row& r) { return r.max == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r.weight - r.max - kPBias); }
// A finite scale's share of a probability (weights under 2^-126 have none, whatever their values).
PMI_DEV float share_of(float scale, const Row& r) { return fminf(scale * r.gain, FLT_MAX); }

// ---- few query rows ------------------------------------------------------------------
// Requests of few query rows (tokens x heads of one KV head): bound by the bytes of the
// codes. An item is 16 rows of one KV head of a request against the request's keys, in
// tiles of 64 tokens. The tiles of all items, in order, are dealt evenly to a fixed number
// of workgroups (two per CU, four with heads of 64): lengths differ from request to
// request, and with a part of each request per workgroup the longest decided
// (64 requests of 2048 to 8191 keys, 8 KV heads of 128: 142 us that way).
//
// Four waves take the tiles of a workgroup's part of an item in turn. All operands come
// straight from memory to registers:
//   S^T = K q^T: 16x16x32 fp16 products, rows = tokens. Row m of product t is token
//     16 (m / 4) + 4 t + m % 4 of the tile, so that a lane's results of the four products
//     are 16 consecutive tokens, 16 h .. 16 h + 15 (h = lane / 16), all of one page;
//   O^T = V^T P^T: a lane's operand of P is then what it holds, and that of V its 16-byte
//     piece of the page's block (one dimension, 16 tokens).
// Scales: a lane's 16 tokens share theirs, so ks multiplies the scores and vs the
// probabilities, in fp32, before these become fp16.
//
// An item that several workgroups share is joined by the last of them to arrive, in
// order. A workgroup shares at most two items: the one it begins in (record 2 w) and the one
// it ends in (record 2 w + 1), and only the latter can begin in it, so the
// workgroup in which an item begins lends it its counter.
constexpr int kMinShare = 4;  // tiles per workgroup, at least
// Few tiles: items are cut every so many tiles instead, a part a workgroup, so that none has parts
// of two. The smallest cut whose parts are at most half the workgroups is taken with heads of 128,
// or else at most all of them: one workgroup a CU, whose waves have some tiles each, beats two of
// half the tiles and twice the parts to join (8 requests of 4000 keys, 8 KV heads: 18.3 us, 19.6 with
// two a CU, 22.3 dealt evenly; 1 of 32000: 21.2, dealt evenly 26.7; 24 of 1000: 15.4 and 20.3; with
// heads of 64 a half as many took 14.5 us instead of 13.3).
constexpr int kCuts = 6;
constexpr int cut_of(int k) { return k < 4 ? 4 * (k + 1) : k == 4 ? 24 : 32; }

template <int D>
struct FewLds {
  float acc[4][16][D + 4];  // rows 16 bytes apart in the banks
  float m[4][16], l[4][16];
  int last;
};

template <typename T, int D, bool FP8, Mode MODE>
PMI_DEV void few_rows(const AttnArgs& a, FewLds<D>& lds, int wg) {
  constexpr int DT = D / 16;  // 16-dimension tiles of the output
  float(&s_acc)[4][16][D + 4] = lds.acc;
  float(&s_m)[4][16] = lds.m;
  float(&s_l)[4][16] = lds.l;
  int& s_last = lds.last;
  const int wgs = a.few_wgs;
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = l & 15, h = l >> 4;
  const int G = a.H / a.KV;

  // The tiles of all requests, and where this workgroup begins. Every wave works it out for
  // itself, a lane a run of requests: no barrier, and one round of loads up to 64 requests.
  // (The host sees to it that the sum is below 2^31.)
  auto tiles_of = [&](const Request& rq) { return max(1, (rq.hi - rq.lo + 63) >> 6); };
  auto items_of = [&](const Request& rq) {
    return rq.n * G > (rq.run ? a.run_rows : a.few_rows) ? 0 : (rq.n * G + 15) / 16 * a.KV;
  };
  constexpr int kOf = MODE == kWhole ? 1 : 2;  // numbers of a request
  const int requests = kOf * a.R;
  const int run = kOf * ((a.R + 63) >> 6), r_lane = run * l;
  int in_lane = 0, parts_lane[kCuts] = {};  // tiles, and parts of cut_of(k) tiles
  auto count = [&](const Request& rq) {
    const int nt = tiles_of(rq), items = items_of(rq);
    in_lane += nt * items;
#pragma unroll
    for (int k = 0; k < kCuts; ++k) parts_lane[k] += (nt + cut_of(k) - 1) / cut_of(k) * items;
  };
  for (int x = r_lane; x < min(requests, r_lane + run); x += kOf) {
    if constexpr (MODE == kWhole) {
      count(request<MODE>(a, x));
    } else {
      const Request own = request<MODE>(a, x), of_run = request<MODE>(a, x + 1);  // (their loads together)
      count(own);
      count(of_run);
    }
  }
  auto scan = [&](int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o);
      if (l >= o) v += u;
    }
    return v;
  };
  constexpr int kHalf = D == 128 ? 1 : 0;
  // (a call of few tiles takes the first cut, and no other chain of shuffles than its scan)
  int cut = cut_of(0), upto = scan(cut * parts_lane[0]);
  if (__builtin_amdgcn_readlane(upto, 63) > cut * (wgs >> kHalf)) {
    // the parts of all, two counts a word (a lane's 1023, or more, are too many)
    uint32_t parts_all[kCuts / 2];
#pragma unroll
    for (int j = 0; j < kCuts / 2; ++j) {
      parts_all[j] = (uint32_t)min(parts_lane[2 * j], 1023) | (uint32_t)min(parts_lane[2 * j + 1], 1023) << 16;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) parts_all[j] += __shfl_xor(parts_all[j], o);
      parts_all[j] = __builtin_amdgcn_readfirstlane(parts_all[j]);
    }
    cut = 0;
#pragma unroll
    for (int half = kHalf; half >= 0; --half)
#pragma unroll
      for (int k = 0; k < kCuts; ++k)
        if (!cut && (parts_all[k / 2] >> (16 * (k & 1)) & 0xffff) <= (uint32_t)min(wgs >> half, 1022))
          cut = cut_of(k), in_lane = cut_of(k) * parts_lane[k];
    upto = scan(in_lane);
  } else {
    in_lane = cut * parts_lane[0];
  }
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const int share = cut ? cut : max(kMinShare, (int)(((uint32_t)total + wgs - 1) / wgs));
  if ((int64_t)share * wg >= total) return;
  int g = share * wg;
  const int g_end = min((int64_t)g + share, (int64_t)total);
  const int lane0 = __builtin_ctzll(__ballot(upto > g));
  int r = run * lane0;
  int off = g - (__builtin_amdgcn_readlane(upto, lane0) - __builtin_amdgcn_readlane(in_lane, lane0));  // tiles of r before g
  while (g < g_end && r < requests) {
  const Request rq = request<MODE>(a, r);
  const int row_tiles = (rq.n * G + 15) / 16, nt = tiles_of(rq);
  const int span = cut ? (nt + cut - 1) / cut * cut : nt;  // what an item takes of the order
  const int all = span * items_of(rq);
  if (off >= all) {
    off -= all, ++r;
    continue;
  }
  const int item = off / span, tile0 = off - item * span;
  const int n_tiles = min(g_end - g, nt - tile0), n_span = min(g_end - g, span - tile0);
  const int kh = item / row_tiles, rt = item - kh * row_tiles;
  const int item_g = g - tile0;  // the item's first tile of all
  g += n_span, off += n_span;

  const int32_t* table = a.tables + (int64_t)rq.row * a.stride;
  auto look_up = [&](int p) { return table[min((p + 16 * h) >> a.ps_log, a.width - 1)]; };
  const int start = rq.start, len = rq.len, shift = rq.shift;
  const int rows = rq.n * G - rt * 16;  // of this tile of rows and the ones behind it
  const int row = rt * 16 + c;
  const bool live = c < rows;
  const int i = row / G;
  // positions that this column's query sees: [lo, hi)
  const int hi = live ? max(0, min(len, shift + i + 1)) : 0;
  const int lo = MODE == kWhole ? first_position(a, shift + i) : rq.first_seen;
  const int i_first = rt * 16 / G, i_last = (rt * 16 + min(rows, 16) - 1) / G;
  const int first_seen = rq.first_seen;
  const int p0 = rq.lo + 64 * tile0, p1 = min(rq.hi, p0 + 64 * n_tiles);
  // tiles inside of [safe_lo, safe_hi) need no mask
  const int safe_hi = max(0, min(len, shift + i_first + 1));
  const int safe_lo = MODE == kWhole ? first_position(a, shift + i_last) : first_seen;

  QueryRow<T, D> q;
  load_query<T, D>(q, (const T*)a.q + (int64_t)(start + (live ? i : 0)) * a.q_token +
                          (int64_t)(kh * G + (live ? row - i * G : 0)) * a.q_head, live, h);
  const float qmul = q.mul * a.scale * kLog2e;

  f32x4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  Row ref;
  float sum = 0.f;
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
    // (a page that holds an infinity or NaN: what sees it becomes NaN, not an infinity by its codes' signs)
    const bool bad = !(bks < INFINITY) || !(bvs < INFINITY);
    const float ks = gone ? 0.f : bad ? __builtin_nanf("") : bks * qmul, tvs = gone ? 0.f : bvs;
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
    const float most = max_over_h(mx + __builtin_amdgcn_logf(tvs < INFINITY ? tvs : 0.f));
    mx = max_over_h(mx);
    const float nm = fmaxf(ref.max, mx);
    if (__any(nm > ref.max + kSlack || most > ref.weight + kSlack)) {
      const Rescale f = raise(ref, nm, most);
      sum *= f.sum;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f.acc;
    }
    const float vs = share_of(tvs, ref), base = ref.max == -INFINITY ? 0.f : ref.max;
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
    page = valid(look_up(p), p);
    entry = look_up(p + 256);
    load_scales(page);
    load_k(page, p);
    load_v(page, p);
    for (; p + 256 < p1; p += 256) tile(std::false_type{});
    tile(std::true_type{});
  }

  // the four waves' results, joined in their order
  sum = sum_over_h(sum);
  const float unit = unit_of(ref);
#pragma unroll
  for (int d = 0; d < DT; ++d)
    if (live) *reinterpret_cast<f32x4*>(&s_acc[wave][c][16 * d + 4 * h]) = acc[d] * unit;
  if (h == 0) s_m[wave][c] = ref.max, s_l[wave][c] = sum;
  __syncthreads();
  constexpr int kPer = D / 16;  // dimensions per thread: 16 threads a row
  const int orow = tid >> 4, od = (tid & 15) * kPer;
  const bool mine = orow < rows;
  float om = -INFINITY, ol = 0.f, o[kPer];
#pragma unroll
  for (int x = 0; x < kPer; ++x) o[x] = 0.f;
  if (mine) {
    float mw[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mw[w] = s_m[w][orow], om = fmaxf(om, mw[w]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // a wave that saw no key holds zeros; the sum of one whose scores are all NaN is NaN
      const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - om);
      ol = fmaf(s_l[w][orow], f, ol);
#pragma unroll
      for (int x = 0; x < kPer; x += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(&s_acc[w][orow][od + x]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x + e] = fmaf(v[e], f, o[x + e]);
      }
    }
  }
  const int grow = rt * 16 + orow;
  const int64_t out_row = (int64_t)(start + grow / G) * a.H + kh * G + grow % G;
  T* dst = (T*)a.out + out_row * D + od;
  // a row that is a part: its values from dimension d on
  const bool is_part = MODE == kParts && (rq.run || first_seen > 0);
  auto keep_part = [&](int64_t at, int d, const auto& v, int n, float m, float l) {
    float* rec = (rq.run ? a.parts_one : a.parts_own) + at * (D + 4);
#pragma unroll
    for (int x = 0; x < n; x += 4) *reinterpret_cast<f32x4*>(rec + d + x) = f32x4{v[x], v[x + 1], v[x + 2], v[x + 3]};
    if (d == 0) {
      *reinterpret_cast<float2*>(rec + D) = float2{m, l};
      if (rq.run) a.where[at] = int2{(int)((a.parts_one - a.parts_many) / (D + 4) + at), 4};
    }
  };
  auto store = [&]() {
    if (is_part) {
      if (mine) keep_part(out_row, od, o, kPer, om, ol);
      return;
    }
    const float inv = ol > 0.f ? 1.f / ol : (ol != ol ? ol : 0.f);
    typedef T Tv __attribute__((ext_vector_type(kPer)));
    Tv y;
#pragma unroll
    for (int x = 0; x < kPer; ++x) y[x] = (T)(o[x] * inv);
    if (mine) *reinterpret_cast<Tv*>(dst) = y;
  };
  if (n_tiles == nt) {
    store();
    __syncthreads();  // s_acc is read
    continue;
  }

  // Partial rows to the workspace. Stores and loads are coherent across the XCDs' L2 caches
  // (sc1).
  constexpr int kSc1 = 16, kRec = D + 4;  // floats of a row: values, max, sum
  const int first_wg = item_g / share, parts = (item_g + nt - 1) / share - first_wg + 1;
  const __amdgpu_buffer_rsrc_t rp = rsrc(a.few_part + (int64_t)first_wg * 32 * kRec, (int64_t)parts * 32 * kRec * 4);
  // record of part s: the first one's second, the others' first
  auto record = [&](int s, int rr) { return ((s ? 2 * s : 1) * 16 + rr) * kRec * 4; };
  const int rec = record(wg - first_wg, orow);
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
    const int old = __hip_atomic_fetch_add(&a.counters[first_wg], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == parts - 1;
  }
  __syncthreads();
  if (!s_last) continue;
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
    auto batch = [&](auto fly, int s0) {
      constexpr int kFly = decltype(fly)::value;
      float ms[kFly], ls[kFly];
      f32x4 v[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        const int at = record(min(s0 + k * groups, parts - 1), r0 + jr);
        ms[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, at + 4 * D, 0, kSc1));
        ls[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, at + 4 * D + 4, 0, kSc1));
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, at + 4 * dim, 0, kSc1));
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads stay together, ahead of their uses
      float nm = jm;
#pragma unroll
      for (int k = 0; k < kFly; ++k) nm = fmaxf(nm, s0 + k * groups < parts ? ms[k] : -INFINITY);
      const float f = jm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(jm - nm);
      jl *= f, jo *= f;
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        // (a part that saw no key: weight 0; its sum may be NaN, see above)
        const bool use = s0 + k * groups < parts;
        const float w = use && ms[k] != -INFINITY ? __builtin_amdgcn_exp2f(ms[k] - nm) : 0.f;
        jl = fmaf(use ? ls[k] : 0.f, w, jl);
#pragma unroll
        for (int x = 0; x < 4; ++x) jo[x] = fmaf(use ? v[k][x] : 0.f, w, jo[x]);
      }
      jm = nm;
    };
    if (on) {
      if (parts <= 4 * groups)
        batch(std::integral_constant<int, 4>{}, grp);
      else
        for (int s0 = grp; s0 < parts; s0 += 16 * groups) batch(std::integral_constant<int, 16>{}, s0);
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
      const int row1 = rt * 16 + r0 + slot;
      const int64_t out1 = (int64_t)(start + row1 / G) * a.H + kh * G + row1 % G;
      if (is_part) {
        keep_part(out1, dim, jo, 4, jm, jl);
        continue;
      }
      const float inv = jl > 0.f ? 1.f / jl : (jl != jl ? jl : 0.f);
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = (T)(jo[x] * inv);
      *reinterpret_cast<T4*>((T*)a.out + out1 * D + dim) = y;
    }
  }
  if (tid == 0) __hip_atomic_store(&a.counters[first_wg], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();  // s_acc is read
  }
}

template <typename T, int D, bool FP8, Mode MODE>
__global__ __launch_bounds__(256, 2) void attention_few_kernel(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) FewLds<D> lds;
  few_rows<T, D, FP8, MODE>(a, lds, blockIdx.x);
}

template <typename T, int D, Mode MODE>
hipError_t few(const AttnArgs& a, bool fp8, hipStream_t stream) {
  if (fp8)
    hipLaunchKernelGGL((attention_few_kernel<T, D, true, MODE>), dim3(a.few_wgs), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attention_few_kernel<T, D, false, MODE>), dim3(a.few_wgs), dim3(256), 0, stream, a);
  return hipGetLastError();
}

// ---- many query rows -----------------------------------------------------------------
// Requests with more query rows: bound by the softmax's vector instructions, 11 a score,
// beside the matrix cores (prompts of 345 to 2048 tokens, 32 / 8 heads of 128, int8: 110 us, 580
// TFLOP/s; chunks of 198 to 500 tokens in a window of 4096, 16 / 2 heads of 64, e4m3: 50 us, 320
// TFLOP/s, the same rate of scores; counters: 32 % of a wave's cycles issue vector
// instructions, two waves a SIMD). Scores multiplied a tile ahead of the softmax cost more in
// copies than they hid (126 us for the prompts), three workgroups a CU too (59 us for the chunks). A
// workgroup takes 128 query rows (32 a wave, tokens x heads of one KV head, so that the heads
// share the keys) against tiles of 64 keys. The tile's codes become fp16 once, on their way
// from registers to LDS (two slots), and serve the four waves:
//   S^T = K q^T, 32x32x16 products, rows = tokens: row m of product u is token 32 u + 16 (m / 16) +
//     8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so that eight of a lane's results are eight
//     consecutive tokens, its operand of P;
//   O^T = V^T P^T from V^T in LDS, rows = dimensions.
// A block of 16 tokens, and with it a page's scales, is the same for all lanes. In LDS,
// 16-byte chunk x of row y lies at x ^ (y % 16) (K of heads of 128) or x ^ (y / 2 % 8) (K of heads
// of 64, and V^T): reads of 16 consecutive rows fall in different banks.
// Where the rows give fewer workgroups than the CUs hold, the keys are split as well
// (`splits` ranges of `per` tokens), and the last range to arrive joins them.
constexpr int kRows = 128;
// Keys of a run's range, at least (us, 64 requests of 8192 shared keys, 256 / 512 / 768 / 1024: 49 / 42 / 45 / 52; 16 of 8000
// 31 / 28 / 30 / 34): every range is 68 KB of parts.
constexpr int kLeastRange = 512;

// HALVES (kParts): 2 for runs of up to half as many rows: two waves take the first 32 keys of each
// tile, two the last, as parts of their own. Nothing waits for the ranges: their parts are joined by
// another launch (joined by the last range of an item, 16 x 128 rows of 16 ranges took 81 us, so 36).
template <typename T, int D, bool FP8, Mode MODE, int HALVES>
PMI_DEV void many_tile(const AttnArgs& a, uint8_t* lds, int& s_last, const Request& rq, int rt, int kh, int index,
                       int sp, int splits);

template <typename T, int D, bool FP8, Mode MODE>
PMI_DEV void many_rows(const AttnArgs& a, uint8_t* lds, int& s_last, int wg) {
  const int l = threadIdx.x & 63;
  const int G = a.H / a.KV;

  // which rows: the row tiles of all requests in order, each request's last ones (with the most
  // keys) first, the KV heads innermost (an XCD then keeps few heads' keys in its L2)
  const auto number = [](int r) { return MODE == kWhole ? r : 2 * r + 1; };
  auto tiles_of = [&](int r) {
    const Request rq = request<MODE>(a, number(r));
    return rq.n * G > (MODE == kWhole ? a.few_rows : a.run_rows) ? (rq.n * G + kRows - 1) / kRows : 0;
  };
  const int kh = wg % a.KV, rest = wg / a.KV;
  int splits = a.splits, sp = 0, index = 0;
  if constexpr (MODE == kWhole) sp = rest % splits, index = rest / splits;
  const int run = (a.R + 63) >> 6, r_lane = run * l;
  int in_lane = 0;
  for (int x = r_lane; x < min(a.R, r_lane + run); ++x) in_lane += tiles_of(x);
  int upto = in_lane;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(upto, o);
    if (l >= o) upto += u;
  }
  const int all_tiles = __builtin_amdgcn_readlane(upto, 63);
  if constexpr (MODE == kParts) {
    // (the host does not know how many runs there are, nor what they share. Runs that no batch has may be so many
    // that the product passes 32 bits: it is made only where the ranges' parts have room for it)
    splits = all_tiles > 0 && all_tiles <= a.many_wgs / a.KV ? a.many_wgs / (all_tiles * a.KV) : 1;
    sp = rest % splits, index = rest / splits;
  }
  if (index >= all_tiles) return;
  const int lane0 = __builtin_ctzll(__ballot(upto > index));
  int r = run * lane0;
  int at_tile = index - (__builtin_amdgcn_readlane(upto, lane0) - __builtin_amdgcn_readlane(in_lane, lane0));
  int count = tiles_of(r);
  while (at_tile >= count) {
    at_tile -= count;
    if (++r >= a.R) return;
    count = tiles_of(r);
  }
  const int rt = count - 1 - at_tile;
  const Request rq = request<MODE>(a, number(r));
  if (MODE == kParts && rq.n * G <= kRows / 2)
    many_tile<T, D, FP8, MODE, MODE == kParts ? 2 : 1>(a, lds, s_last, rq, rt, kh, index, sp, splits);
  else
    many_tile<T, D, FP8, MODE, 1>(a, lds, s_last, rq, rt, kh, index, sp, splits);
}

template <typename T, int D, bool FP8, Mode MODE, int HALVES>
PMI_DEV void many_tile(const AttnArgs& a, uint8_t* lds, int& s_last, const Request& rq, int rt, int kh, int index,
                       int sp, int splits) {
  constexpr int KP = D / 64;       // 16-byte pieces of K, and of V, per thread and tile
  constexpr int kSlot = 64 * D * 2;  // bytes of K (or V) of a tile as fp16
  constexpr int U = 2 / HALVES;    // of the tile's two halves, those of a wave
  constexpr int kTileRows = kRows / HALVES;
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = l & 31, h = l >> 5;
  const int G = a.H / a.KV;
  const int row_wave = HALVES == 1 ? wave : wave & 1, half = HALVES == 1 ? 0 : wave >> 1;
  const int start = rq.start, len = rq.len, shift = rq.shift;
  const int rows = min(kTileRows, rq.n * G - rt * kTileRows);
  const int row = rt * kTileRows + row_wave * 32 + c;
  const bool live = row_wave * 32 + c < rows;
  const int i = row / G;
  const int hi = live ? max(0, min(len, shift + i + 1)) : 0;
  const int lo = MODE == kWhole ? first_position(a, shift + i) : rq.first_seen;
  const int i_first = rt * kTileRows / G, i_last = (rt * kTileRows + rows - 1) / G;
  const int first_seen = MODE == kWhole ? min(first_position(a, shift + i_first), len) : rq.first_seen;
  const int all_lo = first_seen & ~15;
  const int all_hi = a.n_pages ? max(all_lo, min(len, shift + i_last + 1)) : all_lo;
  const int per = MODE == kParts ? max(kLeastRange, ((len + splits - 1) / splits + 63) & ~63) : a.per;
  const int parts = max(1, (all_hi - all_lo + per - 1) / per);
  if (sp >= parts) return;
  const int p0 = all_lo + sp * per, p1 = min(all_hi, p0 + per);
  const int safe_hi = max(0, min(len, shift + i_first + 1));
  const int safe_lo = MODE == kWhole ? first_position(a, shift + i_last) : first_seen;

  // the wave's query rows: step s holds dimensions 16 s + 8 h .. + 7
  f16x8 qv[D / 16];
  // (the sign of the scale goes into q: block maxima need a factor that is not negative)
  float qmul = fabsf(a.scale) * kLog2e;
  {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T* qr = (const T*)a.q + (int64_t)(start + (live ? i : i_first)) * a.q_token +
                  (int64_t)(kh * G + (live ? row - i * G : 0)) * a.q_head;
    T8 raw[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) raw[s] = *reinterpret_cast<const T8*>(qr + 16 * s + 8 * h);
    if constexpr (__is_same(T, f16)) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s) qv[s] = a.scale < 0.f ? -raw[s] : raw[s];
    } else {
      float m = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf((float)raw[s][e]));
      m = fmaxf(m, __shfl_xor(m, 32));
      PowerOfTwo w = power_below(m);
      qmul *= w.up;
      if (a.scale < 0.f) w.down = -w.down;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) qv[s][e] = (f16)((float)raw[s][e] * w.down);
    }
  }

  typedef float f32x16 __attribute__((ext_vector_type(16)));
  f32x16 acc[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
  Row ref;
  float sum = 0.f;
  const int32_t* table = a.tables + (int64_t)rq.row * a.stride;
  const int64_t cell_bytes = (int64_t)a.ps * D;

  // The four blocks of the tile at p, block b in the lanes with l % 4 = b, so that their pages and
  // scales are one instruction each (as scalars they were a sixth of the issued ones).
  struct Blocks {
    int page;  // -1: not there
    float ks, vs;
  };
  const int lane_token = 16 * (l & 3);
  auto look_up = [&](int p) { return table[min((p + lane_token) >> a.ps_log, a.width - 1)]; };
  auto blocks_of = [&](int p, int entry) {
    const bool there = p + lane_token < p1 && (unsigned)entry < a.n_pages;
    const int64_t cell = (int64_t)(there ? entry : 0) * a.KV + kh;
    return Blocks{there ? entry : -1, a.k_scale[cell], a.v_scale[cell]};
  };
  auto of_block = [](float v, int b) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), b));
  };
  // A wave's 64 pieces of 16 bytes (piece tid + 256 k of the tile, token-major for K, dimension-major
  // in a block for V) are all of one block, so that addresses are the same but for a constant.
  u32x4 kw[KP], vw[KP];
  auto block_of = [&](int k) { return (64 * wave + 256 * k) / D; };
  auto load_tile = [&](int p, const Blocks& x) {
#pragma unroll
    for (int k = 0; k < KP; ++k) {
      const int idx = tid + 256 * k, b = block_of(k);
      const int64_t cell = (int64_t)max(__builtin_amdgcn_readlane(x.page, b), 0) * a.KV + kh;
      const int tok = (p + 16 * b) & (a.ps - 1);
      const int64_t at = cell * cell_bytes + tok * D;  // of both: a block of v is 16 tokens of D bytes
      kw[k] = *reinterpret_cast<const u32x4*>(a.k + at + (uint32_t)(16 * (idx % D)));
      vw[k] = *reinterpret_cast<const u32x4*>(a.v + at + (uint32_t)(16 * (idx % D)));
    }
  };
  // 16 consecutive rows in different banks: one row fills the 64 banks (D = 128), or two do
  auto swizzle = [](int krow) { return D == 128 ? krow & 15 : (krow >> 1) & 7; };
  auto store_tile = [&](int p, const Blocks& x, int slot) {
    uint8_t* kb = lds + slot * 2 * kSlot;
    uint8_t* vb = kb + kSlot;
    // codes of tokens that no row sees may be NaN (e4m3)
    const bool edge = FP8 && (p < first_seen || p + 64 > p1 || __any(x.page < 0));
#pragma unroll
    for (int k = 0; k < KP; ++k) {
      const int idx = tid + 256 * k;
      const int krow = idx / (D / 16), kpiece = idx % (D / 16);
      const f16x8 k0 = codes8<FP8>(kw[k][0], kw[k][1]), k1 = codes8<FP8>(kw[k][2], kw[k][3]);
      *reinterpret_cast<f16x8*>(kb + krow * D * 2 + (((2 * kpiece) ^ swizzle(krow)) << 4)) = k0;
      *reinterpret_cast<f16x8*>(kb + krow * D * 2 + (((2 * kpiece + 1) ^ swizzle(krow)) << 4)) = k1;
      const int vblk = block_of(k), vd = idx % D;
      if (edge) vw[k] &= byte_mask(first_seen - p - 16 * vblk,
                                     __builtin_amdgcn_readlane(x.page, vblk) < 0 ? 0 : p1 - p - 16 * vblk);
      const f16x8 v0 = codes8<FP8>(vw[k][0], vw[k][1]), v1 = codes8<FP8>(vw[k][2], vw[k][3]);
      *reinterpret_cast<f16x8*>(vb + vd * 128 + (((2 * vblk) ^ ((vd >> 1) & 7)) << 4)) = v0;
      *reinterpret_cast<f16x8*>(vb + vd * 128 + (((2 * vblk + 1) ^ ((vd >> 1) & 7)) << 4)) = v1;
    }
  };

  if (p0 < p1) {
    Blocks cur = blocks_of(p0, look_up(p0));
    load_tile(p0, cur);
    Blocks next = blocks_of(p0 + 64, look_up(p0 + 64));
    store_tile(p0, cur, 0);
    load_tile(p0 + 64, next);
    int entry = look_up(p0 + 128);
    int slot = 0;
    for (int p = p0; p < p1; p += 64, slot ^= 1) {
      __syncthreads();  // the slot is written; the other one is read
      const uint8_t* kb = lds + slot * 2 * kSlot;
      const uint8_t* vb = kb + kSlot;
      __builtin_amdgcn_s_setprio(1);  // products ahead of the other wave's softmax
      f32x16 s[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int krow = 32 * (u + half) + 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
          const f16x8 k8 = *reinterpret_cast<const f16x8*>(kb + krow * D * 2 + (((2 * x + h) ^ swizzle(krow)) << 4));
          s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, qv[x], s[u], 0, 0, 0);
        }
      __builtin_amdgcn_s_setprio(0);
      const bool gone = cur.page < 0;
      float ks = gone ? 0.f : cur.ks, vs = gone ? 0.f : cur.vs;
      const bool bad = !(ks < INFINITY) || !(vs < INFINITY);
      // result 16 u + 4 j + e: token 32 u + 16 (j / 2) + 8 h + 4 (j % 2) + e, block 2 u + j / 2.
      // Hidden tokens get -inf, which stays one through the factors k1 (at least FLT_MIN).
      if (p < safe_lo || p + 64 > safe_hi || p + 64 > p1 || __any(gone)) {
        const int from = lo - p - 8 * h - 32 * half, to = min(hi, p1) - p - 8 * h - 32 * half;
#pragma unroll
        for (int y = 0; y < 16 * U; ++y) {
          const int at = 16 * (y >> 3) + (y & 7);
          const int end = __builtin_amdgcn_readlane(cur.page, 2 * half + (y >> 3)) >= 0 ? to : 0;
          s[y >> 4][y & 15] = at >= from && at < end ? s[y >> 4][y & 15] : -INFINITY;
        }
      }
      if (const uint64_t which = __ballot(bad)) {
        // a page that holds an infinity or NaN: what sees it becomes NaN
        if (bad) ks = 0.f, vs = 0.f;
#pragma unroll
        for (int b = 0; b < 2 * U; ++b)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float t = s[b >> 1][8 * (b & 1) + e];
            s[b >> 1][8 * (b & 1) + e] = t == -INFINITY || !(which >> (2 * half + b) & 1) ? t : __builtin_nanf("");
          }
      }
      const float vlog = __builtin_amdgcn_logf(vs);
      // (FLT_MIN after all factors, the query's power of two among them; the sums are below 2^33, so what
      // it raises is a score of 0 all the same)
      float k1[2 * U];
#pragma unroll
      for (int b = 0; b < 2 * U; ++b) k1[b] = fmaxf(of_block(ks, 2 * half + b) * qmul, FLT_MIN);
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2 * U; ++b) {
        float t = s[b >> 1][8 * (b & 1)];
#pragma unroll
        for (int e = 1; e < 8; ++e) t = fmaxf(t, s[b >> 1][8 * (b & 1) + e]);
        mx = fmaxf(mx, t * k1[b]);
      }
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float nm = fmaxf(ref.max, mx);
      // (the largest product of the tile is at most the one of its largest score and its largest scale)
      if (__any(nm > ref.max + kSlack || mx + max_of_4(vlog) > ref.weight + kSlack)) {
        float most = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) {
          float t = s[b >> 1][8 * (b & 1)];
#pragma unroll
          for (int e = 1; e < 8; ++e) t = fmaxf(t, s[b >> 1][8 * (b & 1) + e]);
          most = fmaxf(most, fmaf(t, k1[b], of_block(vlog, 2 * half + b)));
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        const Rescale f = raise(ref, nm, most);
        sum *= f.sum;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] *= f.acc;
      }
      // The next tile to its slot (past the range: page 0 of the cache, never used), among the
      // exponentials: at the top of the loop this took 114.9 us instead of 112.1.
      store_tile(p + 64, next, slot ^ 1);
      const Blocks after = blocks_of(p + 128, entry);
      load_tile(p + 128, after);
      entry = look_up(p + 192);
      const float base = ref.max == -INFINITY ? 0.f : ref.max;
#pragma unroll
      for (int b = 0; b < 2 * U; ++b) {
        const float v1 = share_of(of_block(vs, 2 * half + b), ref);
        f16x8 pw;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ex = __builtin_amdgcn_exp2f(fmaf(s[b >> 1][8 * (b & 1) + e], k1[b], -base));
          sum += ex;
          pw[e] = (f16)(ex * v1);
        }
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const int vrow = 32 * d + c;
          const f16x8 v8 = *reinterpret_cast<const f16x8*>(vb + vrow * 128 + (((2 * b + 4 * half + h) ^ ((vrow >> 1) & 7)) << 4));
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, pw, acc[d], 0, 0, 0);
        }
      }
      cur = next;
      next = after;
    }
  }

  // result 4 j + e of tile d: dimension 32 d + 8 j + 4 h + e
  sum += __shfl_xor(sum, 32);
  const float unit = unit_of(ref);
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int64_t out_row = (int64_t)(start + i) * a.H + kh * G + row - i * G;
  T* dst = (T*)a.out + out_row * D + 4 * h;
  if constexpr (MODE == kParts) {
    static_assert(HALVES <= 2, "the second half's records lie behind the first's");
    const int64_t in_one = (a.parts_one - a.parts_many) / (D + 4) + (int64_t)half * a.T * a.H + out_row;
    const int64_t at = splits == 1 ? in_one : ((int64_t)(index * a.KV + kh) * splits + sp) * kRows + wave * 32 + c;
    float* rec = a.parts_many + at * (D + 4);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = acc[d][4 * j + e] * unit;
        if (live) *reinterpret_cast<f32x4*>(rec + 32 * d + 8 * j + 4 * h) = y;
      }
    if (live && h == 0) *reinterpret_cast<float2*>(rec + D) = float2{ref.max, sum};
    if (live && h == 0 && sp == 0 && half == 0)
      a.where[out_row] = int2{(int)at, 4 * HALVES * parts + (splits == 1 ? 2 : HALVES - 1)};
    return;
  }
  if (parts == 1) {
    const float inv = sum > 0.f ? unit / sum : (sum != sum ? sum : 0.f);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        T4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(acc[d][4 * j + e] * inv);
        if (live) *reinterpret_cast<T4*>(dst + 32 * d + 8 * j) = y;
      }
    return;
  }

  // partial rows, as in the kernel above: values, max, sum
  constexpr int kSc1 = 16, kRec = D + 4;
  const int item = index * a.KV + kh;
  const __amdgpu_buffer_rsrc_t rp = rsrc(a.many_part + (int64_t)item * splits * kRows * kRec, (int64_t)parts * kRows * kRec * 4);
  const int rrow = wave * 32 + c;
  if (live) {
    const int rec = (sp * kRows + rrow) * kRec * 4;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = acc[d][4 * j + e] * unit;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rp, rec + 4 * (32 * d + 8 * j + 4 * h), 0, kSc1);
      }
    if (h == 0) {
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, ref.max), rp, rec + 4 * D, 0, kSc1);
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, sum), rp, rec + 4 * D + 4, 0, kSc1);
    }
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    const int old = __hip_atomic_fetch_add(&a.counters[a.few_wgs + item], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == parts - 1;
  }
  __syncthreads();
  if (!s_last) return;
  constexpr int kRowThreads = D / 4;
  for (int y = tid / kRowThreads; y < rows; y += 256 / kRowThreads) {
    const int dim = 4 * (tid % kRowThreads);
    float jm = -INFINITY, jl = 0.f;
    f32x4 jo = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 4) {
      float ms[4], ls[4];
      f32x4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = (min(s0 + k, parts - 1) * kRows + y) * kRec * 4;
        ms[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, at + 4 * D, 0, kSc1));
        ls[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rp, at + 4 * D + 4, 0, kSc1));
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, at + 4 * dim, 0, kSc1));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) join(jm, jl, jo, ms[k], ls[k], v[k], s0 + k < parts);
    }
    const int grow = rt * kRows + y;
    const int64_t out1 = (int64_t)(start + grow / G) * a.H + kh * G + grow % G;
    const float inv = jl > 0.f ? 1.f / jl : (jl != jl ? jl : 0.f);
    T4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)(jo[e] * inv);
    *reinterpret_cast<T4*>((T*)a.out + out1 * D + dim) = o;
  }
  if (tid == 0) __hip_atomic_store(&a.counters[a.few_wgs + item], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The requests of few rows first, then those of many, in one launch, so that the end of the one
// fills with the other (32 / 8 heads of 128: 8 single tokens of 2000 keys and a prompt of 2048 72 us, in
// two launches 81; 32 of 3000 and a chunk of 512 behind 1000 79 and 84; two prompts of 300, where the
// first find nothing to do, 17.6 and 18.6).
template <typename T, int D, bool FP8, Mode MODE>
__global__ __launch_bounds__(256, 2) void attention_rows_kernel(AttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [2 slots][K, V]
  __shared__ int s_last;
  static_assert(sizeof(FewLds<D>) <= 2 * 2 * 64 * D * 2, "fits the slots");
  // (of parts the runs' are the longest: they begin first)
  if constexpr (MODE == kParts) {
    const int many = (int)gridDim.x - a.few_wgs;
    if ((int)blockIdx.x < many)
      many_rows<T, D, FP8, MODE>(a, lds, s_last, blockIdx.x);
    else
      few_rows<T, D, FP8, MODE>(a, *reinterpret_cast<FewLds<D>*>(lds), blockIdx.x - many);
    return;
  }
  if ((int)blockIdx.x < a.few_wgs)
    few_rows<T, D, FP8, MODE>(a, *reinterpret_cast<FewLds<D>*>(lds), blockIdx.x);
  else
    many_rows<T, D, FP8, MODE>(a, lds, s_last, blockIdx.x - a.few_wgs);
}

template <typename T, int D, Mode MODE>
hipError_t many(const AttnArgs& a, bool fp8, int64_t wgs, hipStream_t stream) {
  constexpr int kLds = 2 * 2 * 64 * D * 2;
  if (fp8)
    hipLaunchKernelGGL((attention_rows_kernel<T, D, true, MODE>), dim3((unsigned)wgs), dim3(256), kLds, stream, a);
  else
    hipLaunchKernelGGL((attention_rows_kernel<T, D, false, MODE>), dim3((unsigned)wgs), dim3(256), kLds, stream, a);
  return hipGetLastError();
}

// The parts of the rows that share keys. D / 4 threads a row and four groups of them, which take every
// fourth shared part, the first its own as well; the groups are joined in LDS, in order. Bound by its
// chain of loads (lengths, where, parts). Workgroup (r, KV head, z) takes every gridDim.z-th of the head's
// rows of request r, some at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_parts_kernel(AttnArgs a) {
  constexpr int kRowThreads = D / 4, kGroups = 4, kFly = 8, kSlots = 256 / kRowThreads / kGroups;
  __shared__ __attribute__((aligned(16))) float s_o[kSlots][kGroups][D];
  __shared__ float2 s_ml[kSlots][kGroups];
  const int r = blockIdx.x, kh = blockIdx.y, G = a.H / a.KV;
  const Request rq = request<kParts>(a, 2 * r);
  if (rq.n <= 0 || rq.first_seen <= 0) return;
  const int dim = 4 * (threadIdx.x % kRowThreads), group = threadIdx.x / kRowThreads % kGroups;
  const int slot = threadIdx.x / kRowThreads / kGroups;
  for (int row0 = blockIdx.z * kSlots; row0 < rq.n * G; row0 += gridDim.z * kSlots) {
    const int row = min(row0 + slot, rq.n * G - 1);
    const int64_t out_row = (int64_t)(rq.start + row / G) * a.H + kh * G + row % G;
    const float* own = a.parts_own + out_row * (D + 4);
    const bool first = group == 0;
    float m = first ? own[D] : -INFINITY, l = first ? own[D + 1] : 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (first) o = *reinterpret_cast<const f32x4*>(own + dim);
    const int2 at = a.where[out_row];
    int apart = at.y & 2 ? a.T * a.H : at.y & 1 ? kRows / 2 : kRows;
    // (as a power of two the compiler would shift by it, 64 bits by an amount of a lane's own, which has given
    // wrong lanes on this hardware)
    asm("" : "+v"(apart));
    // (nobody wrote it if the runs are not this batch's)
    const bool there = at.x >= 0 && at.y >= 4 && (int64_t)at.x + (int64_t)apart * ((at.y >> 2) - 1) < a.part_records;
    const int n = there ? at.y >> 2 : 0;
    const float* rec = a.parts_many + (int64_t)at.x * (D + 4);
    for (int s0 = group; s0 < n; s0 += kFly * kGroups) {
      float2 ml[kFly];
      f32x4 v[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        const float* p = rec + (int64_t)min(s0 + kGroups * k, n - 1) * apart * (D + 4);
        ml[k] = *reinterpret_cast<const float2*>(p + D);
        v[k] = *reinterpret_cast<const f32x4*>(p + dim);
      }
#pragma unroll
      for (int k = 0; k < kFly; ++k) join(m, l, o, ml[k].x, ml[k].y, v[k], s0 + kGroups * k < n);
    }
    __syncthreads();  // the previous rows are read
    *reinterpret_cast<f32x4*>(&s_o[slot][group][dim]) = o;
    if (dim == 0) s_ml[slot][group] = float2{m, l};
    __syncthreads();
    if (!first || row0 + slot >= rq.n * G) continue;
#pragma unroll
    for (int g = 1; g < kGroups; ++g)
      join(m, l, o, s_ml[slot][g].x, s_ml[slot][g].y, *reinterpret_cast<const f32x4*>(&s_o[slot][g][dim]), true);
    const float inv = l > 0.f ? 1.f / l : (l != l ? l : 0.f);
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] * inv);
    *reinterpret_cast<T4*>((T*)a.out + out_row * D + dim) = y;
  }
}

// Workgroups of the few-row part: what the CUs hold at once of its own kernel (with heads of 64 half
// as many of the joint one, the others follow).
int few_wgs(int64_t D) { return device_cu_count() * (D == 64 ? 4 : 2); }
// Query rows of a KV head up to which a request is one of few. From 17 on its codes are read and
// converted by two to four items, where the other form has one row tile; but that one shares its keys among
// fewer workgroups. us, few / many rows, KV heads x D, requests x keys each (int8, fp16):
//   rows                     16          32          48          64
//   8 x 128,  1 x  4000   13 /  24    14 /  28    17 /  31    17 /  34
//   8 x 128,  8 x  4000   20 /  36    28 /  41    41 /  49    48 /  53
//   8 x 128, 64 x  4000   96 / 170   181 / 177   263 / 191   346 / 181
//   8 x 128, 16 x 32000  190 / 396   304 / 403   524 / 435   621 / 434
//   8 x  64, 16 x 32000  116 / 291   158 / 293   247 / 322   307 / 324
// 64 is best while the requests do not fill the CUs; 32 would be where many of 33 to 64 rows do.
constexpr int kFewRows = 64;

struct ManyPlan {
  int64_t items;  // at most: row tiles of all requests x KV heads
  int splits, per;
  size_t part;
};
ManyPlan many_plan(const PagedAttention& p, const PagedCache& c) {
  ManyPlan f = {};
  const int64_t G = p.H / c.KV;
  if (p.max_q * G <= kFewRows) return f;
  // row tiles: every request's last one may be partly filled, and has more than kFewRows rows
  const int64_t most = p.T * G / (kFewRows + 1) < p.R ? p.T * G / (kFewRows + 1) : p.R;
  f.items = (p.T * G / kRows + most) * c.KV;
  // what a row tile sees: up to the window behind each of its queries, from a multiple of 16 on
  const int64_t seen = p.window + (kRows + G - 2) / G + 15, range = p.window && seen < p.max_kv ? seen : p.max_kv;
  // two workgroups a CU; a range of at least eight tiles, as its join costs about two
  int64_t S = f.items > 0 ? 2 * device_cu_count() / f.items : 1;
  if (S > range / 512) S = range / 512;
  if (S < 1 || f.items > (int64_t)kWsCounterBytes / 4 - few_wgs(c.D)) S = 1;
  f.per = (int)(((range + S - 1) / S + 63) / 64 * 64);
  if (f.per < 64) f.per = 64;
  f.splits = (int)((range + f.per - 1) / f.per);
  if (f.splits < 1) f.splits = 1;
  f.part = f.splits > 1 ? (size_t)(f.items * f.splits * kRows * (c.D + 4) * 4) : 0;
  return f;
}

}  // namespace

size_t few_part_bytes(int64_t D) { return (size_t)few_wgs(D) * 32 * (D + 4) * 4; }

bool paged_attention_tiles_fit(const PagedAttention& p, const PagedCache& c) {
  // of every request the rows of one of few rows, in tiles of 16; keys in tiles of 64, one more for a
  // range that begins inside a tile, and up to four for its last cut
  const int64_t rows = p.max_q * (p.H / c.KV), row_tiles = ((rows < kFewRows ? rows : kFewRows) + 15) / 16;
  const int64_t keys = p.width * c.ps < p.max_kv ? p.width * c.ps : p.max_kv;
  return (double)p.R * (double)c.KV * (double)row_tiles * (double)(keys / 64 + 5) < 2147483648.0;
}

bool paged_attention_launch_fits(const PagedAttention& p, const PagedCache& c) {
  const ManyPlan f = many_plan(p, c);
  return few_wgs(c.D) + f.items * f.splits < (1ll << 24);  // of 256 threads: 2^32
}

size_t paged_attention_ws_bytes(const PagedAttention& p, const PagedCache& c) {
  return kWsCounterBytes + few_part_bytes(c.D) + many_plan(p, c).part;
}

namespace {

// The arguments that all parts of a call have in common.
AttnArgs attention_args(const PagedAttention& p, const PagedCache& c, void* workspace) {
  AttnArgs a = {p.q, p.out, (const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, p.tables, p.kv_lens,
                p.q_starts, p.stride, p.q_token, p.q_head, c.pages, (int)p.T, (int)p.R, (int)p.width, (int)p.H,
                (int)c.KV, (int)c.ps, __builtin_ctz((unsigned)c.ps), (int)p.window, p.scale};
  a.max_q = (int)p.max_q, a.max_kv = (int)p.max_kv;
  a.few_rows = kFewRows;
  a.counters = (int*)workspace;
  a.few_part = (float*)((char*)workspace + kWsCounterBytes);
  a.many_part = (float*)((char*)a.few_part + few_part_bytes(c.D));
  a.few_wgs = few_wgs(c.D);
  a.runs = (const int4*)p.runs, a.run_lens = p.run_lens;
  return a;
}

// Requests of few rows alone (n = 0), or n workgroups of both.
template <Mode MODE>
hipError_t launch_mode(const AttnArgs& a, const PagedAttention& p, const PagedCache& c, int64_t n, hipStream_t stream) {
  if (n == 0) {
    if (p.bf16) return c.D == 64 ? few<__bf16, 64, MODE>(a, c.fp8, stream) : few<__bf16, 128, MODE>(a, c.fp8, stream);
    return c.D == 64 ? few<f16, 64, MODE>(a, c.fp8, stream) : few<f16, 128, MODE>(a, c.fp8, stream);
  }
  if (p.bf16)
    return c.D == 64 ? many<__bf16, 64, MODE>(a, c.fp8, n, stream) : many<__bf16, 128, MODE>(a, c.fp8, n, stream);
  return c.D == 64 ? many<f16, 64, MODE>(a, c.fp8, n, stream) : many<f16, 128, MODE>(a, c.fp8, n, stream);
}

// Query rows up to which a run is one of few: those read its codes once for every 16 rows (us with 16 / 32, 64
// requests of 8 families, 4000 / 16000 keys each: 39 / 69, 65 / 155; 8 of one, 8000: 22.0 / 25.1).
constexpr int kRunRows = 16;

// Row tiles of all runs of many rows x KV heads, at most.
int64_t run_items(const PagedAttention& p, const PagedCache& c) {
  const int64_t G = p.H / c.KV, rows = p.T * G;
  if (rows <= kRunRows) return 0;
  const int64_t runs = rows / (kRunRows + 1) < p.R ? rows / (kRunRows + 1) : p.R;
  return (rows / kRows + runs) * c.KV;
}
// Workgroups of runs of many rows: those that the CUs hold, as ranges of keys, or one for each row tile.
int64_t run_wgs(const PagedAttention& p, const PagedCache& c) {
  const int64_t items = run_items(p, c), held = 2 * device_cu_count();
  return items == 0 ? 0 : items > held ? items : held;
}
// Records of their ranges: those are several only where all ranges together are as many as the CUs hold.
int64_t run_records(const PagedAttention& p, const PagedCache& c) {
  return run_items(p, c) ? (int64_t)2 * device_cu_count() * kRows : 0;
}
size_t part_bytes(int64_t rows, int64_t D) { return (size_t)(rows * (D + 4) * 4); }

}  // namespace

// Parts pay where what is read per request without them is much. us, in parts / whole (32 / 8 heads of 128
// unless said, int8, one token each; `families` of equal share, 300 more keys each; without the 6 of
// finding the runs):
//   16 requests, 1 family, 1000 / 2000 / 4000 keys   20.8 / 14.2   21.1 / 18.4   23.0 / 25.6
//   64 requests, 1 family, 1000 / 2000 / 8000         32.5 / 21.8   34.4 / 39.1   40.1 / 101
//   64 requests, 8 families, 1000 / 2000 / 16000      29.8 / 21.4   31.4 / 40.9   65 / 218
//   64 of 4 KV heads of 64, 1 family, 4000 / 8000     26.4 / 22.8   29.0 / 42.7
//   8 requests, 1 family, 4000 / 8000                 20.6 / 18.4   22.0 / 25.6
// Many rows a request make better use of keys by themselves: 7 tokens each of 32 (28 rows), 4000 keys, 45.6 /
// 52.1; 16 of 64 (64 rows), 2000 keys, 121 / 80.
constexpr int kShareRows = 32;
constexpr int64_t kShareKeys = 2048, kShareBytes = 1ll << 27;
bool paged_attention_shares(const PagedAttention& p, const PagedCache& c) {
  return p.R > 1 && p.T < (1ll << 30) && p.window == 0 && p.max_q * (p.H / c.KV) <= kShareRows &&
         p.max_kv >= kShareKeys && p.R * c.KV * 2 * c.D >= (kShareBytes + p.max_kv - 1) / p.max_kv;
}

bool paged_shared_launch_fits(const PagedAttention& p, const PagedCache& c) {
  // (parts are counted in 32 bits, and requests and runs together)
  return few_wgs(c.D) + run_wgs(p, c) < (1ll << 23) && p.R < (1ll << 29) && p.R * c.KV < (1ll << 21) &&
         run_records(p, c) + 3 * p.T * p.H < (1ll << 31);
}

size_t paged_shared_ws_bytes(const PagedAttention& p, const PagedCache& c) {
  return kWsCounterBytes + few_part_bytes(c.D) + part_bytes(run_records(p, c) + 3 * p.T * p.H, c.D) +
         (size_t)(p.T * p.H * 8);
}

hipError_t launch_paged_shared(const PagedAttention& p, const PagedCache& c, void* workspace, hipStream_t stream) {
  AttnArgs a = attention_args(p, c, workspace);
  const int64_t wgs = run_wgs(p, c), rows = p.T * p.H, records = run_records(p, c);
  a.parts_many = a.many_part;
  a.parts_one = a.parts_many + records * (c.D + 4);
  a.parts_own = a.parts_one + 2 * rows * (c.D + 4);
  a.where = (int2*)(a.parts_own + rows * (c.D + 4));
  a.part_records = (int)(records + 2 * rows);
  a.run_rows = kRunRows;
  a.many_wgs = 2 * device_cu_count();
  if (hipError_t e = launch_mode<kParts>(a, p, c, wgs ? a.few_wgs + wgs : 0, stream); e != hipSuccess) return e;
  // (of a row's four groups of D / 4 threads each; up to 8 workgroups share a request's rows)
  const int64_t slots = 64 / (c.D / 4), pieces = (p.max_q * (p.H / c.KV) + slots - 1) / slots;
  const dim3 grid((unsigned)p.R, (unsigned)c.KV, (unsigned)(pieces < 8 ? pieces : 8)), block(256);
  if (p.bf16) {
    if (c.D == 64)
      hipLaunchKernelGGL((join_parts_kernel<__bf16, 64>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((join_parts_kernel<__bf16, 128>), grid, block, 0, stream, a);
  } else {
    if (c.D == 64)
      hipLaunchKernelGGL((join_parts_kernel<f16, 64>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((join_parts_kernel<f16, 128>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttention& p, const PagedCache& c, void* workspace, size_t ws_bytes,
                                  hipStream_t stream) {
  AttnArgs a = attention_args(p, c, workspace);
  const ManyPlan f = many_plan(p, c);
  if (f.items == 0) return launch_mode<kWhole>(a, p, c, 0, stream);
  // Any batch of several requests may have some of few rows; a lone one stays with many.
  if (p.R == 1) a.few_rows = 0, a.few_wgs = 0;
  a.splits = f.splits, a.per = f.per;
  return launch_mode<kWhole>(a, p, c, a.few_wgs + f.items * f.splits, stream);
}

}  // namespace pmi
