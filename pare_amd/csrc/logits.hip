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

// Values as integers in their order, NaN above all of them and both zeros the same; a value and its token
// as one, where the lower token is the larger of two equal values.
PMI_DEV uint32_t ordered(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
  return v != v ? ~0u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
PMI_DEV uint64_t keyed(uint32_t value, int token) { return (uint64_t)value << 32 | (uint32_t)~token; }
PMI_DEV int token_of(uint64_t key) { return ~(int)(uint32_t)key; }
PMI_DEV uint64_t largest_of_wave(uint64_t key) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor(key, o);
    key = other > key ? other : key;
  }
  return key;
}

// Tokens of a workgroup, its threads, and how LDS holds what its tokens count and their biases' entries:
// in 16 bits while the history is shorter than 2^15 tokens (bit 15 is for the prompt's) and there are
// fewer entries than 2^16 - 1 (whose numbers leave two), else in 32.
template <int SLICE, int THREADS, typename C>
struct Form {
  static constexpr int kSlice = SLICE, kThreads = THREADS;
  typedef C Count;
  static constexpr uint32_t kPrompt = 1u << (8 * sizeof(C) - 1), kNoBias = (C)~(C)0, kSeveral = kNoBias - 1;
};

// A workgroup takes a slice of a row, in frames of 16 bytes that are aligned in memory (a row
// of odd size begins inside one). What the slice's tokens count in the history is made in LDS from all
// of the row's history, so that no list of a row's distinct tokens is needed. Of a token's biases LDS holds the
// entry, or that there are several: such a token goes through all entries, in their order (64 x 128257 bf16 with 300
// / 5000 biases, of which two are of one token: 36 / 513 us, without 8.5 / 15.4; with all biased tokens of the slice
// going through them 297 / 17200).
// WRITE: the logits to `out`; else the largest of them, the slices' joined by the last to arrive.
template <typename T, bool WRITE, typename F>
__global__ __launch_bounds__(F::kThreads) void logits_kernel(Logits f, T* out, int64_t out_stride,
                                                             int64_t* __restrict__ tokens, int64_t token_stride,
                                                             int* __restrict__ counters,
                                                             uint64_t* __restrict__ part, int slices) {
  constexpr int E = Frame<T>::kSize, kSlice = F::kSlice, kThreads = F::kThreads;
  constexpr int kFrames = kSlice / E / kThreads;  // frames of a thread
  typedef typename Frame<T>::Vec Vec;
  typedef typename F::Count C;
  typedef C CVec __attribute__((ext_vector_type(E)));
  __shared__ __attribute__((aligned(16))) C counts[kSlice];
  __shared__ __attribute__((aligned(16))) C biases[kSlice];
  __shared__ int twice, s_last;
  __shared__ uint64_t best_s[kThreads / 64];
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
      bits[k] = __builtin_amdgcn_alignbit(mask[min(word + 1, (V - 1) >> 5)], mask[word], at & 31) << (at - t);
    }
  }

  const int32_t* ids = biased ? f.bias_ids + r * f.n_bias : nullptr;
  const float* values = biased ? f.bias + r * f.n_bias : nullptr;
  const int n_bias = (int)f.n_bias;
  float rho = 1.f, alpha = 0.f, beta = 0.f;
  if (penalties || biased) {
    constexpr int kWords = kSlice * (int)sizeof(C) / 16;
    for (int i = tid; i < kWords; i += kThreads) {
      reinterpret_cast<u32x4*>(counts)[i] = u32x4{0, 0, 0, 0};
      reinterpret_cast<u32x4*>(biases)[i] = u32x4{~0u, ~0u, ~0u, ~0u};
    }
    if (tid == 0) twice = 0;
    const auto of_slice = [&](int t) {
      return (uint32_t)t < (uint32_t)V && (uint32_t)t - (uint32_t)s0 < (uint32_t)kSlice;
    };
    const int32_t* past = f.history + r * f.history_stride;
    const int n = !penalties ? 0 : (int)(f.history_lens ? min((int64_t)max(f.history_lens[r], 0), f.L) : f.L);
    const int prompt = penalties && f.prompt_lens ? f.prompt_lens[r] : 0;
    if (penalties) {
      if (f.repetition) rho = f.repetition[r];
      if (f.presence) alpha = f.presence[r];
      if (f.frequency) beta = f.frequency[r];
    }
    __syncthreads();
    constexpr int kFly = 8;  // tokens in flight a thread
    for (int i0 = tid; i0 < n; i0 += kThreads * kFly) {
      int t[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) t[k] = i0 + kThreads * k < n ? past[i0 + kThreads * k] : -1;
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        if (!of_slice(t[k])) continue;
        constexpr uint32_t kPer = 4 / sizeof(C);  // counts of a word
        const uint32_t at = t[k] - s0, up = 8 * sizeof(C) * (at % kPer);
        uint32_t* word = reinterpret_cast<uint32_t*>(counts) + at / kPer;
        if (i0 + kThreads * k < prompt)
          atomicOr(word, F::kPrompt << up);
        else
          atomicAdd(word, 1u << up);
      }
    }
    if (biased) {
      for (int i = tid; i < n_bias; i += kThreads)
        if (of_slice(ids[i])) biases[ids[i] - s0] = (C)i;  // (whichever comes last)
      __syncthreads();
      for (int i = tid; i < n_bias; i += kThreads)
        if (of_slice(ids[i]) && biases[ids[i] - s0] != (C)i) biases[ids[i] - s0] = (C)F::kSeveral, twice = 1;
    }
    __syncthreads();
  }

  T* to = WRITE ? out + r * out_stride : nullptr;
  const bool wide = WRITE && (int)((uintptr_t)to % 16 / sizeof(T)) == shift;
  uint32_t best = 0;  // below every value's
  int best_at = 0;
#pragma unroll
  for (int k = 0; k < kFrames; ++k) {
    const int in = E * (tid + kThreads * k), t = s0 + in;
    if (t >= V || t + E <= 0) continue;
    if (penalties || biased) {
      const CVec c = *reinterpret_cast<const CVec*>(counts + in), b = *reinterpret_cast<const CVec*>(biases + in);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (c[e] == 0 && b[e] == (C)F::kNoBias) continue;
        float v = (float)x[k][e];
        if (c[e]) {
          v = v > 0.f ? v / rho : v * rho;
          const uint32_t n = c[e] & (F::kPrompt - 1);
          if (n) v = v - beta * (float)n - alpha;
        }
        if (b[e] != (C)F::kNoBias) {
          float sum = values[b[e] == (C)F::kSeveral ? 0 : b[e]];
          if (twice && b[e] == (C)F::kSeveral) {
            bool any = false;
            for (int i = 0; i < n_bias; ++i)
              if (ids[i] == t + e) sum = any ? sum + values[i] : values[i], any = true;
          }
          v += sum;
        }
        x[k][e] = (T)v;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!(bits[k] >> e & 1)) x[k][e] = (T)-INFINITY;
      if constexpr (!WRITE) {
        const uint32_t value = t + e >= 0 && t + e < V ? ordered((float)x[k][e]) : 0;
        if (value > best) best = value, best_at = t + e;
      }
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
    uint64_t key = largest_of_wave(keyed(best, best_at));
    if ((tid & 63) == 0) best_s[tid >> 6] = key;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kThreads / 64; ++w) key = best_s[w] > key ? best_s[w] : key;
      if (slices == 1) {
        tokens[r * token_stride] = token_of(key);
        s_last = 0;
      } else {
        // coherent across the XCDs' L2 caches
        __hip_atomic_store(&part[(int64_t)r * slices + slice], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        s_last = __hip_atomic_fetch_add(&counters[r], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
      }
    }
    __syncthreads();
    if (!s_last || tid >= 64) return;
    key = 0;
    for (int i = tid; i < slices; i += 64) {
      const uint64_t other = __hip_atomic_load(&part[(int64_t)r * slices + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      key = other > key ? other : key;
    }
    key = largest_of_wave(key);
    if (tid == 0) {
      tokens[r * token_stride] = token_of(key);
      __hip_atomic_store(&counters[r], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// Tokens of a workgroup: the history is gone through once for each slice of a row, so that slices are large
// where the rows are workgroups enough.
typedef Form<4096, 256, uint16_t> Small;
typedef Form<16384, 1024, uint16_t> Large;
typedef Form<8192, 512, uint32_t> Wide;

int64_t size_of(int dtype) { return dtype == 2 ? 4 : 2; }
// Slices of a row (one that begins inside a frame may need one more).
int64_t slices_of(int64_t V, int64_t size, bool aligned, int slice) {
  return (V + (aligned ? 0 : 16 / size - 1) + slice - 1) / slice;
}
// Whether the threads of a launch of this form pass no 2^32.
template <typename F>
bool fits(const Logits& f) {
  const int64_t rows = f.R < (1ll << 31) ? f.R : 1ll << 31;
  return rows * slices_of(f.V, size_of(f.dtype), false, F::kSlice) * F::kThreads < (1ll << 32);
}
bool wide(const Logits& f) { return f.L >= 1 << 15 || f.n_bias >= (1 << 16) - 1; }

template <typename T, bool WRITE, typename F>
hipError_t launch_form(const Logits& f, void* out, int64_t out_stride, int64_t* tokens, int64_t token_stride, void* ws,
                       hipStream_t stream) {
  const bool aligned = (uintptr_t)f.x % 16 == 0 && f.stride * sizeof(T) % 16 == 0;
  const int slices = (int)slices_of(f.V, sizeof(T), aligned, F::kSlice);
  hipLaunchKernelGGL((logits_kernel<T, WRITE, F>), dim3((unsigned)(f.R * slices)), dim3(F::kThreads), 0, stream, f,
                     (T*)out, out_stride, tokens, token_stride, (int*)ws,
                     WRITE ? nullptr : (uint64_t*)((char*)ws + kWsCounterBytes), slices);
  return hipGetLastError();
}

template <typename T, bool WRITE>
hipError_t launch_t(const Logits& f, void* out, int64_t out_stride, int64_t* tokens, int64_t token_stride, void* ws,
                    hipStream_t stream) {
  if (wide(f)) return launch_form<T, WRITE, Wide>(f, out, out_stride, tokens, token_stride, ws, stream);
  if (f.R * ((f.V + Large::kSlice - 1) / Large::kSlice) >= device_cu_count() && fits<Large>(f))
    return launch_form<T, WRITE, Large>(f, out, out_stride, tokens, token_stride, ws, stream);
  return launch_form<T, WRITE, Small>(f, out, out_stride, tokens, token_stride, ws, stream);
}

template <bool WRITE>
hipError_t launch(const Logits& f, void* out, int64_t out_stride, int64_t* tokens, int64_t token_stride, void* ws,
                  hipStream_t stream) {
  if (f.dtype == 0) return launch_t<f16, WRITE>(f, out, out_stride, tokens, token_stride, ws, stream);
  if (f.dtype == 1) return launch_t<__bf16, WRITE>(f, out, out_stride, tokens, token_stride, ws, stream);
  return launch_t<float, WRITE>(f, out, out_stride, tokens, token_stride, ws, stream);
}

}  // namespace

bool logits_launch_fits(const Logits& f) { return wide(f) ? fits<Wide>(f) : fits<Small>(f); }

hipError_t launch_process_logits(const Logits& f, void* out, int64_t out_stride, hipStream_t stream) {
  return launch<true>(f, out, out_stride, nullptr, 0, nullptr, stream);
}

size_t greedy_ws_bytes(int64_t R, int64_t V, int dtype) {
  return kWsCounterBytes + (size_t)(R * slices_of(V, size_of(dtype), false, Small::kSlice)) * 8;
}

hipError_t launch_greedy_tokens(const Logits& f, int64_t* tokens, int64_t token_stride, void* workspace,
                                hipStream_t stream) {
  return launch<false>(f, nullptr, 0, tokens, token_stride, workspace, stream);
}

}  // namespace pmi
