// 8-bit integer products: what their kernels and the C ABI layer share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pmi {

constexpr int64_t kW8A8MaxK = 131072;  // 127^2 K stays below 2^31

// Codes int8 [M, ld] (zeros from K on) and fp32 scales [M] of x [M, K], row stride x_ld.
// x_dtype: PMI_F16, PMI_BF16 or PMI_F32.
hipError_t launch_quantize_rows(const void* x, int x_dtype, int64_t x_ld, int8_t* codes, float* scales, int64_t M,
                                int64_t K, int64_t ld, hipStream_t stream);

struct W8A8 {
  const int8_t* x;  // [M, ld] codes
  const float* sx;  // [M]
  const int8_t* w;  // [N, ld] codes
  const float* sw;  // [N]
  const void* bias; // [N] of y's type, or null
  void* y;          // [M, N]
  int64_t M, N, ld; // ld % 16 == 0
  int dtype;        // of y: PMI_F16, PMI_BF16 or PMI_F32
};
hipError_t launch_w8a8(const W8A8& p, hipStream_t stream);
// The same of x [M, K] of y's type, row stride x_ld, which becomes codes first: p.x and
// p.sx are where they may be kept.
hipError_t launch_w8a8_rows(const W8A8& p, const void* x, int64_t x_ld, int64_t K, hipStream_t stream);

}  // namespace pmi
