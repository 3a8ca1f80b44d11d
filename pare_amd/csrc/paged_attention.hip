// Attention over the paged 8-bit cache (paged_kv.hip describes it).
//
// A query i of a request with n queries and a length of L keys sees positions
// p <= L - n + i (and p > L - n + i - window):
//   o = sum_p e_p (vs_p v_p) / sum_p e_p,   e_p = exp(scale q . (ks_p k_p) - max)
// with the codes k_p, v_p and their pages' scales. A query that sees nothing gives 0.
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
  int T, R, width, H, KV, ps, window;
  float scale;
};

template <bool FP8>
PMI_DEV float code_value(uint8_t c) {
  if constexpr (FP8)
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  else
    return (float)(int8_t)c;
}

// One wave per (token, head): 64 positions at a time, a lane a position for the
// scores and D / 64 dimensions a lane for the values.
template <typename T, int D, bool FP8>
__global__ __launch_bounds__(64) void attention_rows_kernel(AttnArgs a) {
  const int t = blockIdx.x, h = blockIdx.y, l = threadIdx.x;
  int r = t, i = 0, n = 1;
  if (a.q_starts) {
    int lo = 0, hi = a.R;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.q_starts[mid + 1] > t)
        hi = mid;
      else
        lo = mid + 1;
    }
    r = lo;
    if (r >= a.R) return;
    i = t - a.q_starts[r];
    n = a.q_starts[r + 1] - a.q_starts[r];
  }
  const int64_t cap = (int64_t)a.width * a.ps;
  const int len = (int)min((int64_t)max(a.kv_lens[r], 0), cap);
  const int last = len - n + i;  // the last position that this query sees
  const int p0 = a.window > 0 ? max(0, last - a.window + 1) : 0;
  const int kh = h / (a.H / a.KV);
  const T* qr = (const T*)a.q + t * a.q_token + h * a.q_head;
  float m = -INFINITY, sum = 0.f, acc[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) acc[e] = 0.f;
  for (int b = p0; b <= last; b += 64) {
    const int p = b + l;
    bool live = p <= last;
    const int page = live ? a.tables[r * a.stride + p / a.ps] : -1;
    live = page >= 0 && page < a.n_pages;
    const int64_t cell = live ? (int64_t)page * a.KV + kh : 0;
    const int off = p % a.ps;
    float s = -INFINITY, vs = 0.f;
    if (live) {
      const uint8_t* kr = a.k + (cell * a.ps + off) * D;
      float d = 0.f;
      for (int e = 0; e < D; ++e) d = fmaf((float)qr[e], code_value<FP8>(kr[e]), d);
      s = d * a.k_scale[cell] * a.scale;
      vs = a.v_scale[cell];
    }
    float mx = s;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float nm = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : __expf(m - nm);
    const float e = live ? __expf(s - nm) : 0.f;
    sum = fmaf(sum, f, wave_sum(e));
    m = nm;
    const float w = live ? e * vs : 0.f;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) acc[x] *= f;
    for (int j = 0; j < 64; ++j) {
      const float wj = __shfl(w, j);
      if (!__shfl((int)live, j)) continue;
      const int64_t cj = ((int64_t)__shfl((int)(cell >> 32), j) << 32) | (uint32_t)__shfl((int)cell, j);
      const int oj = __shfl(off, j);
      const uint8_t* vb = a.v + cj * a.ps * D + (int64_t)(oj / 16) * D * 16 + oj % 16;
#pragma unroll
      for (int x = 0; x < D / 64; ++x) acc[x] = fmaf(wj, code_value<FP8>(vb[(l + 64 * x) * 16]), acc[x]);
    }
  }
  T* o = (T*)a.out + ((int64_t)t * a.H + h) * D;
#pragma unroll
  for (int x = 0; x < D / 64; ++x) o[l + 64 * x] = (T)(sum > 0.f || sum != sum ? acc[x] / sum : 0.f);
}

template <typename T, int D>
hipError_t rows(const AttnArgs& a, bool fp8, hipStream_t stream) {
  const dim3 grid((unsigned)a.T, (unsigned)a.H);
  if (fp8)
    hipLaunchKernelGGL((attention_rows_kernel<T, D, true>), grid, dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL((attention_rows_kernel<T, D, false>), grid, dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_ws_bytes(const PagedAttention& p, const PagedCache& c) { return 0; }

hipError_t launch_paged_attention(const PagedAttention& p, const PagedCache& c, void* workspace, size_t ws_bytes,
                                  hipStream_t stream) {
  AttnArgs a = {p.q, p.out, (const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, p.tables, p.kv_lens,
                p.q_starts, p.stride, p.q_token, p.q_head, c.pages, (int)p.T, (int)p.R, (int)p.width, (int)p.H,
                (int)c.KV, (int)c.ps, (int)p.window, p.scale};
  if (p.bf16) return c.D == 64 ? rows<__bf16, 64>(a, c.fp8, stream) : rows<__bf16, 128>(a, c.fp8, stream);
  return c.D == 64 ? rows<f16, 64>(a, c.fp8, stream) : rows<f16, 128>(a, c.fp8, stream);
}

}  // namespace pmi
