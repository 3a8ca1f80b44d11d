// 8-bit integer matrix product with a scale per token and per channel, and the
// quantisation of rows that feeds it.
//
//   code = round(x * 127 / amax),  scale = amax / 127     (per row of K values)
//   y[m, n] = sx[m] sw[n] sum_k cx[m, k] cw[n, k] (+ bias[n])
//
// The sum is exact in int32 (K <= 131072: 127^2 K < 2^31), so neither the order of the
// products nor a split of K changes a bit; the scales are applied in fp32 and y is
// rounded once. The reference only simulates this (its quantize_inputs path rounds the
// activations and multiplies in floating point, pare/layers/linear.py:120-138).
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "pmi_common.h"
#include "pmi_launch.h"
#include "w8a8.h"

namespace pmi {
namespace {

// Rows [M, K] that are not codes yet, of y's type.
struct W8A8Rows {
  const void* x;
  int64_t ld;
  int K, wide;  // wide: eight values may be read at once
};

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

// ---- quantisation of rows ----------------------------------------------------------

template <typename T>
PMI_DEV uint32_t abs_max8(const T* p, int n, bool wide, vec8<T>& v) {
  if (wide) {
    v = *reinterpret_cast<const vec8<T>*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (T)0.f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __builtin_bit_cast(uint32_t, (float)v[e]) & 0x7fffffffu);
  return m;
}

template <typename T>
PMI_DEV u32x2 codes_of8(const vec8<T>& v, float inv) {
  u32x2 w = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int q = (int)fminf(fmaxf(rintf((float)v[e] * inv), -127.f), 127.f);
    w[e >> 2] |= (uint32_t)(q & 255) << (8 * (e & 3));
  }
  return w;
}
// 127 / amax, finite for the smallest rows too; 0 of a row of zeros.
PMI_DEV float inverse_of(float amax) { return amax > 0.f ? fminf(127.f / amax, FLT_MAX) : 0.f; }

// Bound by the bytes (4099 x 4096 fp16: 13 us, 50 MB), a row alone by its launch (4.7 us).
// Codes of a row, zeros from K to ld. One workgroup of 256 threads per row, eight values a
// thread and step; the first kKeep steps (rows up to 8192) stay in registers between the
// maximum and the codes. |x| is compared as bits, where infinities and NaN are the largest.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t x_ld,
                                                            int8_t* __restrict__ codes, float* __restrict__ scales,
                                                            int K, int ld, int wide) {
  constexpr int kKeep = 4;
  __shared__ uint32_t red[4];
  const int tid = threadIdx.x;
  const T* row = x + (int64_t)blockIdx.x * x_ld;
  vec8<T> keep[kKeep];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int k = 8 * (tid + 256 * i);
    if (k < K) m = max(m, abs_max8(row + k, K - k, wide && k + 8 <= K, keep[i]));
  }
  for (int k = 8 * (tid + 256 * kKeep); k < K; k += 2048) {
    vec8<T> v;
    m = max(m, abs_max8(row + k, K - k, wide && k + 8 <= K, v));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  const float amax = __builtin_bit_cast(float, m);
  const float inv = inverse_of(amax);
  if (tid == 0) scales[blockIdx.x] = amax * (1.f / 127.f);
  int8_t* out = codes + (int64_t)blockIdx.x * ld;
  auto put = [&](int k, const vec8<T>& v) { *reinterpret_cast<u32x2*>(out + k) = codes_of8<T>(v, inv); };
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int k = 8 * (tid + 256 * i);
    if (k < K) put(k, keep[i]);
  }
  for (int k = 8 * (tid + 256 * kKeep); k < K; k += 2048) {
    vec8<T> v;
    abs_max8(row + k, K - k, wide && k + 8 <= K, v);
    put(k, v);
  }
  // (K <= 8 (tid + ..) < ld: at most one thread, the columns between K rounded up to 8 and to 16)
  const int tail = (K + 7) / 8 * 8;
  if (tid == 0 && tail < ld) *reinterpret_cast<u32x2*>(out + tail) = u32x2{0, 0};
}

// y of eight neighbouring columns n .. n + 7 of row m from their sums.
template <typename T>
PMI_DEV void store_row8(T* __restrict__ y, const int* sums, const float* sw, const float* bias, float sx, int m, int n,
                        int N, bool wide) {
  vec8<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (T)((float)sums[e] * sx * sw[e] + bias[e]);
  T* at = y + (int64_t)m * N + n;
  if (wide && n + 8 <= N) {
    *reinterpret_cast<vec8<T>*>(at) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < N) at[e] = o[e];
  }
}

// ---- many rows ---------------------------------------------------------------------
// BN weight rows x BM activation rows per workgroup of WN x WM waves, in steps of 128
// columns. Both operands' rows go from memory straight to LDS (two slots, one barrier a step; the
// copies of the next step fly while this one is multiplied); 16-byte chunk c of row r lies at
// chunk c ^ (r / 2 % 8), so that reads of 16 consecutive rows (two rows fill the 64 banks) do not
// meet in one. Products
// 32x32x32: the weights are the rows of the result, so that a wave reads (BN / WN + BM / WM) x
// 32 bytes for BN / WN x BM / WM / 1024 of them. Columns past ld and rows past the end are copied
// as zeros (from past the descriptor's end). The sums go through LDS (the second slot), 32
// activation rows at a time, to be written 16 bytes a lane. A workgroup stays for several tiles: the
// next one's first copies fly into the first slot meanwhile (4099 x 28672 x 4096: 490 us, a workgroup a
// tile 515; 4096 rows 453 and 473; 2000 x 6144 x 4096 65.5 and 68.3).
//
// What bounds it (4099 x 28672 x 4096 with 13 us of quantisation, 1.96e15 operations a second, 2.12e15 with
// 4096 rows, which fill their tiles): the products alone take about 290 us, the copies hold them up
// by some 120, the stores of y by 70 before they met the next tile's copies (measured with each
// left out). Four slots of 64 columns, three steps ahead: 545 us, twice the requests to L2 for
// half a line each.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void w8a8_tiles_kernel(W8A8 p, int grid_m, int grid_n, int chunk) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int kSlot = (BM + BN) * 128;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int c = l & 31, h = l >> 5;
  // Workgroup 8 k + x runs on XCD x and takes tiles x chunk + k, + gridDim / 8 and so on of the list:
  // blocks of eight tiles of activation rows, columns of weights inside, so that an XCD's tiles share
  // rows of both.
  const int tiles = min(chunk, grid_m * grid_n - (int)(blockIdx.x % 8) * chunk);  // of this XCD
  const int M = (int)p.M, N = (int)p.N, ld = (int)p.ld;
  int m0, n0;
  u32x4 dx, dw;
  auto find = [&](int k) {
    const int tile = (blockIdx.x % 8) * chunk + k;
    const int band = tile / (8 * grid_n), in_band = tile - band * 8 * grid_n;
    const int band_rows = min(8, grid_m - 8 * band);
    m0 = (8 * band + in_band % band_rows) * BM, n0 = in_band / band_rows * BN;
    dx = descriptor(p.x + (int64_t)m0 * ld, (uint32_t)min(BM, M - m0) * ld);
    dw = descriptor(p.w + (int64_t)n0 * ld, (uint32_t)min(BN, N - n0) * ld);
  };
  int mine = blockIdx.x / 8;
  if (mine >= tiles) return;
  find(mine);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

  // a copy: eight rows of 128 bytes, from row 8 (wave + NW i) on (NW is even)
  const int crow = l >> 3, ccol = 16 * ((l & 7) ^ ((crow >> 1) + 4 * (wave & 1)));
  int at_row[BN / 8 / NW > BM / 8 / NW ? BN / 8 / NW : BM / 8 / NW];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(at_row) / sizeof(int)); ++i) at_row[i] = (8 * (wave + NW * i) + crow) * ld + ccol;
  auto copy = [&](int kt, int slot) {
    const uint32_t to = lds0 + slot * kSlot + wave * 1024;
    // past the end of the rows (the last step): past the end of all, zeros
    const bool out = 128 * kt + ccol >= ld;
#pragma unroll
    for (int i = 0; i < BN / 8 / NW; ++i) dma16(dw, to + i * NW * 1024, out ? 0x7ffffff0 : at_row[i], 128 * kt);
#pragma unroll
    for (int i = 0; i < BM / 8 / NW; ++i)
      dma16(dx, to + BN * 128 + i * NW * 1024, out ? 0x7ffffff0 : at_row[i], 128 * kt);
  };

  const int steps = (ld + 127) / 128;
  constexpr int kRow = BN / WN + 4;  // words of a row of sums, rows 16 bytes apart in the banks
  constexpr int kLanes = BN / WN / 8, kStep = 64 / kLanes;  // lanes a row, rows a step
  int* buf = reinterpret_cast<int*>(lds + kSlot) + wave * 32 * kRow;
  const bool wide = N % 8 == 0 && (uintptr_t)p.y % (8 * sizeof(T)) == 0;
  copy(0, 0);
  while (true) {
    // the tile's scales, before any product: the loads of the end would wait for the next tile's copies
    const int n = n0 + wn * (BN / WN) + 8 * (l % kLanes), m_first = m0 + wm * (BM / WM) + l / kLanes;
    float sw[8], bias[8], sx[TM * 32 / kStep];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sw[e] = n + e < N ? p.sw[n + e] : 0.f;
      bias[e] = p.bias && n + e < N ? (float)((const T*)p.bias)[n + e] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < TM * 32 / kStep; ++r) sx[r] = p.sx[min(m_first + kStep * r, M - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(sw[e]), "+v"(bias[e]));
#pragma unroll
    for (int r = 0; r < TM * 32 / kStep; ++r) asm volatile("" : "+v"(sx[r]));

    i32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    for (int kt = 0; kt < steps; ++kt) {
      wait_vmcnt_lgkm0<0>();  // this wave's copies have arrived, its reads of the other slot are done
      barrier_only();
      const int slot = kt & 1;
      if (kt + 1 < steps) copy(kt + 1, slot ^ 1);
      const uint8_t* wb = lds + slot * kSlot + (wn * (BN / WN) + c) * 128;
      const uint8_t* xb = lds + slot * kSlot + BN * 128 + (wm * (BM / WM) + c) * 128;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const int at = 16 * ((2 * ks + h) ^ ((c >> 1) & 7));
        i32x4 wv[TN], xv[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) wv[i] = *reinterpret_cast<const i32x4*>(wb + 32 * 128 * i + at);
#pragma unroll
        for (int j = 0; j < TM; ++j) xv[j] = *reinterpret_cast<const i32x4*>(xb + 32 * 128 * j + at);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wv[i], xv[j], acc[i][j], 0, 0, 0);
      }
    }
    wait_lgkm0();
    barrier_only();  // every wave has read the last step: the slots are free
    // the next tile's first copies, to the first slot, while this one's sums go through the second
    mine += gridDim.x / 8;
    const bool more = mine < tiles;
    if (more) {
      find(mine);
      copy(0, 0);
    }

    // result 4 e + f of tile (i, j): weight row 32 i + 8 e + 4 h + f, activation row 32 j + c
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<i32x4*>(buf + c * kRow + 32 * i + 8 * e + 4 * h) =
              i32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
      // (one wave's own rows: ordered by its LDS counter alone)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int s = 0; s < 32; s += kStep) {
        const int m = m_first + 32 * j + s;
        const i32x4* at = reinterpret_cast<const i32x4*>(buf + (s + l / kLanes) * kRow + 8 * (l % kLanes));
        const i32x4 lo = at[0], hi = at[1];
        const int sums[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (m < M && n < N) store_row8((T*)p.y, sums, sw, bias, sx[(32 * j + s) / kStep], m, n, N, wide);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (!more) return;
  }
}

template <typename T, int BM, int BN, int WM, int WN>
hipError_t tiles(const W8A8& p, hipStream_t stream) {
  constexpr int kWaves = WM * WN, kOut = kWaves * 32 * (BN / WN + 4) * 4, kSlot = (BM + BN) * 128;
  constexpr int kLds = kSlot + (kOut > kSlot ? kOut : kSlot), kPerCu = 160 * 1024 / kLds;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  const void* fn = reinterpret_cast<const void*>(&w8a8_tiles_kernel<T, BM, BN, WM, WN>);
  if (!(allowed.load() & bit)) {
    if (hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024); e != hipSuccess)
      return e;
    allowed.fetch_or(bit);
  }
  const int gm = (int)((p.M + BM - 1) / BM), gn = (int)((p.N + BN - 1) / BN);
  const int chunk = (int)(((int64_t)gm * gn + 7) / 8);
  const int per_xcd = device_cu_count() * kPerCu / 8;  // workgroups that the CUs hold
  hipLaunchKernelGGL((w8a8_tiles_kernel<T, BM, BN, WM, WN>), dim3((unsigned)std::min(chunk, std::max(per_xcd, 1)) * 8),
                     dim3(64 * kWaves), kLds, stream, p, gm, gn, chunk);
  return hipGetLastError();
}

// ---- few rows ----------------------------------------------------------------------
// Up to 64 activation rows: bound by the bytes of the weights (1 x 128256 x 4096: 95 us with its
// quantisation, 5.5 TB/s; 37 x 14335 x 4096: 22.6 us, of which the weights' bytes are 10: four steps a
// wave are too few to hide their first loads, and twice the loads in flight, or a longer share of
// rows, changed it by 2 %). A workgroup takes 16 NT weight
// rows, its eight waves the steps of 128 columns in turn; both operands come straight from memory
// to registers (the activations from L2), 16x16x64 products, the weights the rows of the
// result. The waves' sums are added through LDS.
//
// ROWS: up to 4 rows (4 pieces of 4096 values) that are not codes yet. Every workgroup quantises
// them for itself into LDS, behind its first loads of weights: a launch less, and the codes
// are not read from L2.
constexpr int kPieces = 4;
template <typename T, int MT, int NT, bool ROWS>
__global__ __launch_bounds__(512, 2) void w8a8_few_kernel(W8A8 p, W8A8Rows rows) {
  constexpr int kFly = 10 / (MT + NT) < 1 ? 1 : 10 / (MT + NT);  // steps in flight
  __shared__ __attribute__((aligned(16))) int8_t codes[ROWS ? kPieces * (4096 + 128) : 16];
  __shared__ uint32_t red[ROWS ? kPieces * 8 : 1];
  __shared__ float row_scale[kPieces];
  __shared__ __attribute__((aligned(16))) int sums[16 * MT][16 * NT + 4];
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = l & 15, h = l >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const int M = (int)p.M, N = (int)p.N, ld = (int)p.ld;
  for (int i = tid; i < 16 * MT * (16 * NT + 4); i += 512) (&sums[0][0])[i] = 0;
  // rows past the end read the last one, and are not stored
  const int8_t* wrow[NT];
  const int8_t* xrow[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) wrow[i] = p.w + (int64_t)min(n0 + 16 * i + c, N - 1) * ld;
#pragma unroll
  for (int j = 0; j < MT; ++j) xrow[j] = ROWS ? nullptr : p.x + (int64_t)min(16 * j + c, M - 1) * ld;
  // pieces of a row, and its stride in LDS (rows half the banks apart)
  const int per_row = (ld + 4095) / 4096, x_row = 4096 * per_row + 128;
  i32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  // a step: 128 columns, a lane's 32 h .. 32 h + 31 of a row (whole lines of 128 bytes a row)
  const i32x4 zero = {0, 0, 0, 0};
  const int full = ld / 128;  // whole steps
  i32x4 wv[kFly][NT][2], xv[ROWS ? 1 : kFly][MT][2];
  auto load = [&](int f, int s) {  // step s, or (past the end) the first again
    const int k = 128 * (s < full ? s : 0) + 32 * h;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        wv[f][i][q] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(wrow[i] + k + 16 * q));
    if constexpr (!ROWS) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) xv[f][j][q] = *reinterpret_cast<const i32x4*>(xrow[j] + k + 16 * q);
    }
  };
  auto multiply = [&](int f, int s) {
    const int g = ROWS ? 0 : f;
    if constexpr (ROWS) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        xv[0][0][q] = *reinterpret_cast<const i32x4*>(codes + min(c, M - 1) * x_row + 128 * s + 32 * h + 16 * q);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[f][i][q], xv[g][j][q], acc[i][j], 0, 0, 0);
  };
  if constexpr (ROWS) {
    static_assert(MT == 1, "up to 4 rows");
    vec8<T> v[kPieces];
    uint32_t m[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int row = j / per_row, k = 4096 * (j - row * per_row) + 8 * tid;
      v[j] = {};
      m[j] = 0;
      if (row < M && k < rows.K)
        m[j] = abs_max8((const T*)rows.x + row * rows.ld + k, rows.K - k, rows.wide && k + 8 <= rows.K, v[j]);
    }
#pragma unroll
    for (int f = 0; f < kFly; ++f) load(f, wave + 8 * f);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m[j] = max(m[j], (uint32_t)__shfl_xor((int)m[j], o));
      if (l == 0) red[8 * j + wave] = m[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int row = j / per_row, piece = j - row * per_row;
      if (row >= M) continue;
      uint32_t top = 0;
      for (int i = 8 * row * per_row; i < 8 * (row + 1) * per_row; ++i) top = max(top, red[i]);
      const float amax = __builtin_bit_cast(float, top);
      if (tid == 0) row_scale[row] = amax * (1.f / 127.f);
      *reinterpret_cast<u32x2*>(codes + row * x_row + 4096 * piece + 8 * tid) = codes_of8<T>(v[j], inverse_of(amax));
    }
    __syncthreads();
  }
  if (wave < full) {
    int s = wave;
    if constexpr (!ROWS) {
#pragma unroll
      for (int f = 0; f < kFly; ++f) load(f, s + 8 * f);
    }
    for (; s + 8 * kFly < full; s += 8 * kFly) {
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        multiply(f, s + 8 * f);
        load(f, s + 8 * (f + kFly));
      }
    }
#pragma unroll
    for (int f = 0; f < kFly; ++f)
      if (s + 8 * f < full) multiply(f, s + 8 * f);
  }
  if (wave == full % 8 && ld % 128) {  // the columns behind the last whole step: a multiple of 16
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = 128 * full + 32 * h + 16 * q;
#pragma unroll
      for (int i = 0; i < NT; ++i) wv[0][i][q] = k < ld ? *reinterpret_cast<const i32x4*>(wrow[i] + k) : zero;
      if constexpr (!ROWS) {
#pragma unroll
        for (int j = 0; j < MT; ++j) xv[0][j][q] = k < ld ? *reinterpret_cast<const i32x4*>(xrow[j] + k) : zero;
      }
    }
    multiply(0, full);
  }
  __syncthreads();  // sums are cleared
  // result e of tile (i, j): weight row 16 i + 4 h + e, activation row 16 j + c; kept at 16 i + 4 e + h
  // of the row, so that the 64 lanes of an addition are in 64 banks
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) atomicAdd(&sums[16 * j + c][16 * i + 4 * e + h], acc[i][j][e]);
  __syncthreads();
  const bool wide = N % 8 == 0 && (uintptr_t)p.y % (8 * sizeof(T)) == 0;
  for (int u = tid; u < M * 2 * NT; u += 512) {
    const int m = u / (2 * NT), n = n0 + 8 * (u % (2 * NT));
    if (n >= N) continue;
    float sw[8], bias[8];
    int v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = sums[m][((n - n0) & ~15) + 4 * (e & 3) + ((n - n0) >> 2 & 3) + (e >> 2)];
      sw[e] = n + e < N ? p.sw[n + e] : 0.f;
      bias[e] = p.bias && n + e < N ? (float)((const T*)p.bias)[n + e] : 0.f;
    }
    store_row8((T*)p.y, v, sw, bias, ROWS ? row_scale[m] : p.sx[m], m, n, N, wide);
  }
}

template <typename T, int MT, bool ROWS = false>
hipError_t few(const W8A8& p, hipStream_t stream, const W8A8Rows& rows = {}) {
  // More weight rows a workgroup read the activations less often (a quarter of them with 64), as
  // long as there are workgroups for the CUs. M x N x K, 16 / 32 / 64 weight rows (us with the
  // quantisation): 1 x 128256 x 4096 120 / 124 / 95, 8 x 14336 x 4096 22.8 / 23.4 / 19.4, 64 x 28672 x 4096
  // 72 / 54 / 48, 17 x 6144 x 4096 20.0 / 14.3 / 19.2, 1 x 4096 x 4096 10.1 / 13.1 / 16.5, 64 x 4096 x 14336
  // 42 / 50 / 69; the products alone where the rule is not the best: 1 x 6144 x 4096 9.0 / 10.2 / 12.9, 8 x 18944
  // x 3584 23.7 / 22.1 / 24.7, 64 x 18944 x 3584 49 / 33 / 37.
  const int64_t cus = device_cu_count();
  const dim3 block(512);
  if (p.N >= 48 * cus)
    hipLaunchKernelGGL((w8a8_few_kernel<T, MT, 4, ROWS>), dim3((unsigned)((p.N + 63) / 64)), block, 0, stream, p, rows);
  else if (p.N >= 20 * cus)
    hipLaunchKernelGGL((w8a8_few_kernel<T, MT, 2, ROWS>), dim3((unsigned)((p.N + 31) / 32)), block, 0, stream, p, rows);
  else
    hipLaunchKernelGGL((w8a8_few_kernel<T, MT, 1, ROWS>), dim3((unsigned)((p.N + 15) / 16)), block, 0, stream, p, rows);
  return hipGetLastError();
}

template <typename T>
hipError_t product(const W8A8& p, hipStream_t stream) {
  if (p.M <= 16) return few<T, 1>(p, stream);
  if (p.M <= 32) return few<T, 2>(p, stream);
  if (p.M <= 48) return few<T, 3>(p, stream);
  if (p.M <= 64) return few<T, 4>(p, stream);
  // 256 x 256 tiles where they fill the CUs, else 128 x 128 (the products alone, us, 256 / 128: 4096 x 4096 x
  // 4096 65 / 74, 256 x 128256 x 4096 157 / 184, 1024 x 4096 x 4096, 64 big tiles, 47 / 27; near the border
  // 300 x 28672 x 4096, 224 of them half filled, 55 / 54, 2000 x 6144 x 4096, 192, 55 / 58, 1024 x 14336 x
  // 4096, 224, 59 / 69; half filled, 128 x 128256 x 4096, 148 / 135)
  const int64_t big = ((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (big >= device_cu_count()) return tiles<T, 256, 256, 2, 4>(p, stream);
  return tiles<T, 128, 128, 2, 2>(p, stream);
}

}  // namespace

hipError_t launch_quantize_rows(const void* x, int x_dtype, int64_t x_ld, int8_t* codes, float* scales, int64_t M,
                                int64_t K, int64_t ld, hipStream_t stream) {
  const dim3 grid((unsigned)M), block(256);
  const int size = x_dtype == 2 ? 4 : 2;
  const int wide = (uintptr_t)x % (8 * size) == 0 && x_ld % 8 == 0;
  if (x_dtype == 0)
    hipLaunchKernelGGL(quantize_rows_kernel<f16>, grid, block, 0, stream, (const f16*)x, x_ld, codes, scales, (int)K,
                       (int)ld, wide);
  else if (x_dtype == 1)
    hipLaunchKernelGGL(quantize_rows_kernel<__bf16>, grid, block, 0, stream, (const __bf16*)x, x_ld, codes, scales,
                       (int)K, (int)ld, wide);
  else
    hipLaunchKernelGGL(quantize_rows_kernel<float>, grid, block, 0, stream, (const float*)x, x_ld, codes, scales,
                       (int)K, (int)ld, wide);
  return hipGetLastError();
}

hipError_t launch_w8a8_rows(const W8A8& p, const void* x, int64_t x_ld, int64_t K, hipStream_t stream) {
  // One launch for up to 4 rows while a CU has at most one workgroup, which quantise them again
  // (M x N x K in one launch / two, us, in a graph: 1 x 4096 x 4096 7.7 / 9.9, 4 x 4096 x 4096 10.0 /
  // 10.5, 1 x 14336 x 4096 17.1 / 18.9, 1 x 4096 x 14336 19.9 / 19.2, 4 x 28672 x 4096 30.7 / 30.2,
  // 1 x 128256 x 4096 107 / 97; a call from the host 5 us less), from 1024 columns on, so that every
  // wave has a step to load, and unless y is written over the x that other workgroups still read.
  const int size = p.dtype == 2 ? 4 : 2;
  const uintptr_t x0 = (uintptr_t)x, x1 = x0 + ((p.M - 1) * x_ld + K) * size, y0 = (uintptr_t)p.y, y1 = y0 + p.M * p.N * size;
  if (p.N <= 64 * (int64_t)device_cu_count() && p.M * ((p.ld + 4095) / 4096) <= kPieces && p.ld >= 1024 && (x1 <= y0 || y1 <= x0)) {
    const W8A8Rows rows = {x, x_ld, (int)K, (uintptr_t)x % (8 * size) == 0 && x_ld % 8 == 0};
    if (p.dtype == 0) return few<f16, 1, true>(p, stream, rows);
    if (p.dtype == 1) return few<__bf16, 1, true>(p, stream, rows);
    return few<float, 1, true>(p, stream, rows);
  }
  if (hipError_t e = launch_quantize_rows(x, p.dtype, x_ld, const_cast<int8_t*>(p.x), const_cast<float*>(p.sx), p.M, K,
                                          p.ld, stream);
      e != hipSuccess)
    return e;
  return launch_w8a8(p, stream);
}

hipError_t launch_w8a8(const W8A8& p, hipStream_t stream) {
  if (p.dtype == 0) return product<f16>(p, stream);
  if (p.dtype == 1) return product<__bf16>(p, stream);
  return product<float>(p, stream);
}

}  // namespace pmi
