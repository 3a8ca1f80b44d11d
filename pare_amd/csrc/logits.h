// Logits before a token is chosen: what their kernels and the C ABI layer share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pmi {

struct Logits {
  const void* x;  // [R, V], rows `stride` elements apart
  int64_t stride;
  const int32_t* history;  // [R, L] tokens, or null
  int64_t history_stride, L;  // L < 2^30: the kernel's 32-bit index goes up to a stride of its threads past it
  const int32_t* history_lens;  // [R], or null: L
  const int32_t* prompt_lens;   // [R], or null: 0
  const float* repetition;      // [R] each, or null
  const float* presence;
  const float* frequency;
  const int32_t* bias_ids;  // [R, n_bias], or null
  const float* bias;
  int64_t n_bias;
  const uint32_t* allowed;  // [masks, words], or null
  int64_t masks, words;
  const int32_t* allowed_rows;  // [R], or null: row r
  int64_t R, V;
  int dtype;  // PMI_F16, PMI_BF16 or PMI_F32
};
bool logits_launch_fits(const Logits& f);  // its threads in 32 bits
hipError_t launch_process_logits(const Logits& f, void* out, int64_t out_stride, hipStream_t stream);

constexpr int64_t kGreedyMaxRows = 16384;  // a counter each
size_t greedy_ws_bytes(int64_t R, int64_t V, int dtype);
hipError_t launch_greedy_tokens(const Logits& f, int64_t* tokens, int64_t token_stride, void* workspace,
                                hipStream_t stream);

}  // namespace pmi
