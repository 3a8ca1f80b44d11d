// Penalties for repeated tokens, biases and masks on logits, before a token is chosen.
//
// Row r, token t, in fp32, rounded once:
//   x = x > 0 ? x / rho : x * rho          where t is in the row's history
//   x = x - beta c - alpha                 where t is c > 0 times in it behind the prompt
//   x = x + the row's biases of t, in their order
//   x = -inf                               where the row's mask has no bit for t
// The reference has no counterpart: its decode is HuggingFace's generate
// (pare/eval/throughput.py:84-126).
#include "logits.h"
#include "pmi_common.h"
#include "pmi_launch.h"

namespace pmi {
namespace {

template <typename T>
struct Frame {  // what 16 bytes hold
  static constexpr int kSize = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
};

// A value above another one, or the same earlier in the row; NaN is the largest, as argmax has it.
PMI_DEV bool better(float v, int i, float b, int bi) {
  if (bi < 0) return i >= 0;
  if (i < 0) return false;
  if (v != v) return b == b || i < bi;
  if (b != b) return false;
  return v > b || (v == b && i < bi);
}

PMI_DEV void better_of_wave(float& v, int& i) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(v, o);
    const int oi = __shfl_xor(i, o);
    if (better(ov, oi, v, i)) v = ov, i = oi;
  }
}

constexpr int kThreads = 256;
constexpr int kSlice = 4096;  // tokens of a workgroup
constexpr int kNoBias = 0x7fffffff;

// A workgroup takes kSlice tokens of a row, in frames of 16 bytes that are aligned in memory (a row
// of odd size begins inside one). What the slice's tokens count in the history is made in LDS from all
// of the row's history, so that no list of a row's distinct tokens is needed; bit 31 is for
// the prompt's. Of a token's biases LDS holds the first entry; whether any token has two is known
// as well, and only then the others are looked for.
// WRITE: the logits to `out`; else the largest of them, the slices' joined by the last to arrive.
template <typename T, bool WRITE>
__global__ __launch_bounds__(kThreads) void logits_kernel(Logits f, T* out, int64_t out_stride,
                                                          int64_t* __restrict__ tokens, int64_t token_stride,
                                                          int* __restrict__ counters, float* __restrict__ part,
                                                          int slices) {
  constexpr int E = Frame<T>::kSize, kFrames = kSlice / E / kThreads;  // frames of a thread
  typedef typename Frame<T>::Vec Vec;
  __shared__ __attribute__((aligned(16))) uint32_t counts[kSlice];
  __shared__ __attribute__((aligned(16))) int biases[kSlice];
  __shared__ int twice, s_last;
  __shared__ float best_s[kThreads / 64];
  __shared__ int at_s[kThreads / 64];
  const int tid = threadIdx.x;
  const int r = blockIdx.x / slices, slice = blockIdx.x - r * slices;
  const int V = (int)f.V;
  const T* row = (const T*)f.x + r * f.stride;
  const int shift = (int)((uintptr_t)row % 16 / sizeof(T));  // values of the first frame that are not the row's
  const int s0 = slice * kSlice - shift;                     // the slice's first token
  const bool penalties = f.history != nullptr, biased = f.n_bias > 0;

  Vec x[kFrames];
  uint32_t bits[kFrames];
  const uint32_t* mask = nullptr;
  if (f.allowed) {
    const int m = f.allowed_rows ? f.allowed_rows[r] : r;
    if ((unsigned)m < (unsigned)f.masks) mask = f.allowed + m * f.words;
  }
#pragma unroll
  for (int k = 0; k < kFrames; ++k) {
    const int t = s0 + E * (tid + kThreads * k);
    if (t >= 0 && t + E <= V) {
      x[k] = *reinterpret_cast<const Vec*>(row + t);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[k][e] = t + e >= 0 && t + e < V ? row[t + e] : (T)0.f;
    }
    bits[k] = 0xffffffffu;
    if (mask && t + E > 0 && t < V) {  // bit e: token t + e (any for those that the row does not have)
      const int at = max(t, 0), word = at >> 5;
      const uint64_t two = mask[word] | (uint64_t)mask[min(word + 1, (V - 1) >> 5)] << 32;
      bits[k] = (uint32_t)(two >> (at & 31)) << (at - t);
    }
  }

  const int32_t* ids = biased ? f.bias_ids + r * f.n_bias : nullptr;
  const float* values = biased ? f.bias + r * f.n_bias : nullptr;
  const int n_bias = (int)f.n_bias;
  float rho = 1.f, alpha = 0.f, beta = 0.f;
  if (penalties || biased) {
    for (int i = tid; i < kSlice / 4; i += kThreads) {
      reinterpret_cast<u32x4*>(counts)[i] = u32x4{0, 0, 0, 0};
      reinterpret_cast<u32x4*>(biases)[i] = u32x4{kNoBias, kNoBias, kNoBias, kNoBias};
    }
    if (tid == 0) twice = 0;
    __syncthreads();
    const auto of_slice = [&](int t) { return t >= 0 && t < V && t >= s0 && t < s0 + kSlice; };
    if (penalties) {
      if (f.repetition) rho = f.repetition[r];
      if (f.presence) alpha = f.presence[r];
      if (f.frequency) beta = f.frequency[r];
      const int32_t* past = f.history + r * f.history_stride;
      const int n = (int)(f.history_lens ? min((int64_t)max(f.history_lens[r], 0), f.L) : f.L);
      const int prompt = f.prompt_lens ? f.prompt_lens[r] : 0;
      for (int i = tid; i < n; i += kThreads) {
        const int t = past[i];
        if (!of_slice(t)) continue;
        if (i < prompt)
          atomicOr(&counts[t - s0], 0x80000000u);
        else
          atomicAdd(&counts[t - s0], 1u);
      }
    }
    if (biased) {
      for (int i = tid; i < n_bias; i += kThreads)
        if (of_slice(ids[i])) atomicMin(&biases[ids[i] - s0], i);
      __syncthreads();
      for (int i = tid; i < n_bias; i += kThreads)
        if (of_slice(ids[i]) && biases[ids[i] - s0] != i) twice = 1;
    }
    __syncthreads();
  }

  T* to = WRITE ? out + r * out_stride : nullptr;
  const bool wide = WRITE && (int)((uintptr_t)to % 16 / sizeof(T)) == shift;
  float best = 0.f;
  int best_at = -1;
#pragma unroll
  for (int k = 0; k < kFrames; ++k) {
    const int in = E * (tid + kThreads * k), t = s0 + in;
    if (t >= V || t + E <= 0) continue;
    if (penalties || biased) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        const u32x4 c = *reinterpret_cast<const u32x4*>(counts + in + 4 * q);
        const u32x4 b = *reinterpret_cast<const u32x4*>(biases + in + 4 * q);
        if (!(c[0] | c[1] | c[2] | c[3]) && (b[0] & b[1] & b[2] & b[3]) == (uint32_t)kNoBias) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = (float)x[k][4 * q + e];
          if (c[e]) {
            v = v > 0.f ? v / rho : v * rho;
            const uint32_t n = c[e] & 0x7fffffffu;
            if (n) v = v - beta * (float)n - alpha;
          }
          if (b[e] != (uint32_t)kNoBias) {
            float sum = values[b[e]];
            if (twice)
              for (int i = (int)b[e] + 1; i < n_bias; ++i)
                if (ids[i] == t + 4 * q + e) sum += values[i];
            v += sum;
          }
          x[k][4 * q + e] = (T)v;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!(bits[k] >> e & 1)) x[k][e] = (T)-INFINITY;
      if (!WRITE && t + e >= 0 && t + e < V && better((float)x[k][e], t + e, best, best_at))
        best = (float)x[k][e], best_at = t + e;
    }
    if constexpr (WRITE) {
      if (wide && t >= 0 && t + E <= V) {
        *reinterpret_cast<Vec*>(to + t) = x[k];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (t + e >= 0 && t + e < V) to[t + e] = x[k][e];
      }
    }
  }
  if constexpr (!WRITE) {
    better_of_wave(best, best_at);
    if ((tid & 63) == 0) best_s[tid >> 6] = best, at_s[tid >> 6] = best_at;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kThreads / 64; ++w)
        if (better(best_s[w], at_s[w], best, best_at)) best = best_s[w], best_at = at_s[w];
      if (slices == 1) {
        tokens[r * token_stride] = max(best_at, 0);
        s_last = 0;
      } else {
        // coherent across the XCDs' L2 caches
        float* at = part + 2 * ((int64_t)r * slices + slice);
        __hip_atomic_store(at, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(reinterpret_cast<int*>(at + 1), best_at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        s_last = __hip_atomic_fetch_add(&counters[r], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
      }
    }
    __syncthreads();
    if (!s_last || tid >= 64) return;
    best = 0.f, best_at = -1;
    for (int i = tid; i < slices; i += 64) {
      float* at = part + 2 * ((int64_t)r * slices + i);
      const float v = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int vi = __hip_atomic_load(reinterpret_cast<int*>(at + 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (better(v, vi, best, best_at)) best = v, best_at = vi;
    }
    better_of_wave(best, best_at);
    if (tid == 0) {
      tokens[r * token_stride] = max(best_at, 0);
      __hip_atomic_store(&counters[r], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// Slices of a row; one that begins inside a frame may need one more.
int64_t slices_of(int64_t V, int64_t size) { return (V + 16 / size - 1 + kSlice - 1) / kSlice; }
int64_t size_of(int dtype) { return dtype == 2 ? 4 : 2; }

template <bool WRITE>
hipError_t launch(const Logits& f, void* out, int64_t out_stride, int64_t* tokens, int64_t token_stride, void* ws,
                  hipStream_t stream) {
  const int64_t size = size_of(f.dtype);
  const bool aligned = (uintptr_t)f.x % 16 == 0 && f.stride * size % 16 == 0;
  const int slices = (int)(aligned ? (f.V + kSlice - 1) / kSlice : slices_of(f.V, size));
  const dim3 grid((unsigned)(f.R * slices)), block(kThreads);
  int* counters = (int*)ws;
  float* part = WRITE ? nullptr : (float*)((char*)ws + kWsCounterBytes);
  if (f.dtype == 0)
    hipLaunchKernelGGL((logits_kernel<f16, WRITE>), grid, block, 0, stream, f, (f16*)out, out_stride, tokens,
                       token_stride, counters, part, slices);
  else if (f.dtype == 1)
    hipLaunchKernelGGL((logits_kernel<__bf16, WRITE>), grid, block, 0, stream, f, (__bf16*)out, out_stride, tokens,
                       token_stride, counters, part, slices);
  else
    hipLaunchKernelGGL((logits_kernel<float, WRITE>), grid, block, 0, stream, f, (float*)out, out_stride, tokens,
                       token_stride, counters, part, slices);
  return hipGetLastError();
}

}  // namespace

int64_t logits_workgroups(int64_t R, int64_t V, int dtype) { return R * slices_of(V, size_of(dtype)); }

hipError_t launch_process_logits(const Logits& f, void* out, int64_t out_stride, hipStream_t stream) {
  return launch<true>(f, out, out_stride, nullptr, 0, nullptr, stream);
}

size_t greedy_ws_bytes(int64_t R, int64_t V, int dtype) {
  return kWsCounterBytes + (size_t)logits_workgroups(R, V, dtype) * 8;
}

hipError_t launch_greedy_tokens(const Logits& f, int64_t* tokens, int64_t token_stride, void* workspace,
                                hipStream_t stream) {
  return launch<false>(f, nullptr, 0, tokens, token_stride, workspace, stream);
}

}  // namespace pmi
