// 8-bit integer matrix product with a scale per token and per channel, and the
// quantisation of rows that feeds it.
//
//   code = round(x * 127 / amax),  scale = amax / 127     (per row of K values)
//   y[m, n] = sx[m] sw[n] sum_k cx[m, k] cw[n, k] (+ bias[n])
//
// The sum is exact in int32 (K <= 131072: 127^2 K < 2^31); the scales are applied
// in fp32 and y is rounded once. The reference only simulates this (its
// quantize_inputs path rounds the activations and multiplies in floating point,
// pare/layers/linear.py:120-138).
#include "pmi_common.h"
#include "pmi_launch.h"
#include "w8a8.h"

namespace pmi {
namespace {

// Codes of a row, zeros from K to ld. One workgroup per row.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t x_ld,
                                                            int8_t* __restrict__ codes, float* __restrict__ scales,
                                                            int K, int ld) {
  __shared__ uint32_t red[4];
  const int tid = threadIdx.x;
  const T* row = x + (int64_t)blockIdx.x * x_ld;
  uint32_t m = 0;
  for (int k = tid; k < K; k += 256) m = max(m, __builtin_bit_cast(uint32_t, (float)row[k]) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  const float amax = __builtin_bit_cast(float, m);
  const float inv = amax > 0.f ? 127.f / amax : 0.f;
  if (tid == 0) scales[blockIdx.x] = amax * (1.f / 127.f);
  int8_t* out = codes + (int64_t)blockIdx.x * ld;
  for (int k = tid; k < ld; k += 256)
    out[k] = k < K ? (int8_t)(int)fminf(fmaxf(rintf((float)row[k] * inv), -127.f), 127.f) : (int8_t)0;
}

template <typename T>
__global__ __launch_bounds__(256) void w8a8_kernel(const int8_t* __restrict__ x, const float* __restrict__ sx,
                                                   const int8_t* __restrict__ w, const float* __restrict__ sw,
                                                   const T* __restrict__ bias, T* __restrict__ y, int M, int N,
                                                   int ld) {
  const int n = blockIdx.x * 16 + (threadIdx.x >> 4), m = blockIdx.y * 16 + (threadIdx.x & 15);
  if (n >= N || m >= M) return;
  const u32x4* xr = reinterpret_cast<const u32x4*>(x + (int64_t)m * ld);
  const u32x4* wr = reinterpret_cast<const u32x4*>(w + (int64_t)n * ld);
  int s = 0;
  for (int k = 0; k < ld / 16; ++k) {
    const u32x4 a = xr[k], b = wr[k];
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_sdot4((int)a[e], (int)b[e], s, false);
  }
  float v = (float)s * sx[m] * sw[n];
  if (bias) v += (float)bias[n];
  y[(int64_t)m * N + n] = (T)v;
}

template <typename T>
hipError_t product(const W8A8& p, hipStream_t stream) {
  hipLaunchKernelGGL(w8a8_kernel<T>, dim3((unsigned)((p.N + 15) / 16), (unsigned)((p.M + 15) / 16)), dim3(256), 0,
                     stream, p.x, p.sx, p.w, p.sw, (const T*)p.bias, (T*)p.y, (int)p.M, (int)p.N, (int)p.ld);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_rows(const void* x, int x_dtype, int64_t x_ld, int8_t* codes, float* scales, int64_t M,
                                int64_t K, int64_t ld, hipStream_t stream) {
  const dim3 grid((unsigned)M), block(256);
  if (x_dtype == 0)
    hipLaunchKernelGGL(quantize_rows_kernel<f16>, grid, block, 0, stream, (const f16*)x, x_ld, codes, scales, (int)K,
                       (int)ld);
  else if (x_dtype == 1)
    hipLaunchKernelGGL(quantize_rows_kernel<__bf16>, grid, block, 0, stream, (const __bf16*)x, x_ld, codes, scales,
                       (int)K, (int)ld);
  else
    hipLaunchKernelGGL(quantize_rows_kernel<float>, grid, block, 0, stream, (const float*)x, x_ld, codes, scales,
                       (int)K, (int)ld);
  return hipGetLastError();
}

hipError_t launch_w8a8(const W8A8& p, hipStream_t stream) {
  if (p.dtype == 0) return product<f16>(p, stream);
  if (p.dtype == 1) return product<__bf16>(p, stream);
  return product<float>(p, stream);
}

}  // namespace pmi
