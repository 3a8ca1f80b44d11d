// Host path of calls that the host would bound (CPython extension): the checks, the output
// allocation and the library call that pare_amd otherwise makes from Python.
//   matmul: pmi_matmul_w4a16, of pare_amd.kernels and pare_amd.linear. Calls at decode sizes take
//     3-15 us on the GPU, and the Python path issued one every 20 us (QuantizedLinear at one
//     row); this one every 7.
//   logits: pmi_process_logits and pmi_greedy_tokens, of pare_amd.logits, with up to eleven tensors to
//     check (one row: 6 us on the GPU; a call every 12.4 us from Python, every 5.0 from here).
//   fork_tables, release_tables, compact_tables, shared_prefixes: the entry points of pare_amd.paged for pages of
//     several requests (3-5 us on the GPU; a call every 10 to 20 us from Python, every 4.3 to 6.2 from here).
//   copy_pages: pmi_copy_kv_pages, of pare_amd.paged, with four tensors a layer (32 layers: 9 us on the GPU;
//     a call every 57 us from Python, every 6.4 from here).
//
// Only plain calls are taken: dense tensors of the expected types on the current
// device. For everything else, and where the library refuses, they return
// None and the caller's general path runs, with its own conversions and errors.
// Nothing is kept between calls, and no HIP header is needed: the library's entry
// points arrive as addresses, the stream as its handle.
#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <vector>

namespace py = pybind11;

namespace {

using MatmulFn = int (*)(const void*, int, const uint8_t*, const float*, const void*, int, const int32_t*,
                         const uint16_t*, const float*, const uint8_t*, const uint8_t*, void*, int, int64_t,
                         int64_t, int64_t, int64_t, void*, size_t, void*);
using ChoiceFn = int (*)(int64_t, int64_t, int64_t, int64_t, int);
using WorkspaceFn = size_t (*)(int64_t, int64_t, int64_t, int64_t, int);
using RouteFn = int (*)(int64_t, int64_t, int64_t, int64_t, int, int, size_t);

using ProcessFn = int (*)(const void*, int, int64_t, const int32_t*, int64_t, int64_t, const int32_t*, const int32_t*,
                          const float*, const float*, const float*, const int32_t*, const float*, int64_t,
                          const int32_t*, int64_t, int64_t, const int32_t*, void*, int64_t, int64_t, int64_t, void*);
using GreedyFn = int (*)(const void*, int, int64_t, const int32_t*, int64_t, int64_t, const int32_t*, const int32_t*,
                         const float*, const float*, const float*, const int32_t*, const float*, int64_t,
                         const int32_t*, int64_t, int64_t, const int32_t*, int64_t*, int64_t, int64_t, int64_t, void*,
                         size_t, void*);
using GreedyWorkspaceFn = size_t (*)(int64_t, int64_t, int);
using CopyFn = int (*)(const int32_t*, const int32_t*, const int32_t*, int64_t, void* const*, void* const*,
                       float* const*, float* const*, int64_t, int64_t, int64_t, int64_t, int64_t, void*);

using ForkFn = int (*)(int32_t*, int64_t, int32_t*, const int32_t*, const int32_t*, const int32_t*, int32_t*, int32_t*,
                       int32_t*, int32_t*, int32_t*, int64_t, int64_t, int64_t, int64_t, void*);
using ReleaseFn = int (*)(const int32_t*, int64_t, int32_t*, const uint8_t*, int32_t*, int32_t*, int32_t*, int64_t,
                          int64_t, int64_t, int64_t, void*, size_t, void*);
using CompactFn = int (*)(int32_t*, int64_t, const int32_t*, int32_t*, int32_t*, int32_t*, int32_t*, int32_t*, int32_t*,
                          int64_t, int64_t, int64_t, int64_t, void*, size_t, void*);
using RunsFn = int (*)(const int32_t*, int64_t, const int32_t*, const int32_t*, int32_t*, int32_t*, int32_t*, int64_t,
                       int64_t, int64_t, int64_t, void*, size_t, void*);
using BytesFn = size_t (*)(int64_t);

ForkFn g_fork = nullptr;
ReleaseFn g_release = nullptr;
CompactFn g_compact = nullptr;
RunsFn g_runs = nullptr;
BytesFn g_release_bytes = nullptr, g_compact_bytes = nullptr, g_runs_bytes = nullptr;
ProcessFn g_process = nullptr;
GreedyFn g_greedy = nullptr;
GreedyWorkspaceFn g_greedy_workspace = nullptr;
CopyFn g_copy = nullptr;
MatmulFn g_matmul = nullptr;
ChoiceFn g_choice = nullptr;
WorkspaceFn g_workspace = nullptr;
RouteFn g_route = nullptr;

constexpr int kF16 = 0, kBf16 = 1, kU8 = 3;  // PMI_F16, PMI_BF16, PMI_U8
constexpr int kChoiceTiled = 1, kChoicePerm = 2, kChoiceGm = 4;

void bind(uintptr_t matmul, uintptr_t choice, uintptr_t workspace, uintptr_t route) {
  g_matmul = reinterpret_cast<MatmulFn>(matmul);
  g_choice = reinterpret_cast<ChoiceFn>(choice);
  g_workspace = reinterpret_cast<WorkspaceFn>(workspace);
  g_route = reinterpret_cast<RouteFn>(route);
}

void bind_tables(uintptr_t fork, uintptr_t release, uintptr_t release_bytes, uintptr_t compact, uintptr_t compact_bytes,
                 uintptr_t runs, uintptr_t runs_bytes) {
  g_fork = reinterpret_cast<ForkFn>(fork);
  g_release = reinterpret_cast<ReleaseFn>(release);
  g_release_bytes = reinterpret_cast<BytesFn>(release_bytes);
  g_compact = reinterpret_cast<CompactFn>(compact);
  g_compact_bytes = reinterpret_cast<BytesFn>(compact_bytes);
  g_runs = reinterpret_cast<RunsFn>(runs);
  g_runs_bytes = reinterpret_cast<BytesFn>(runs_bytes);
}

void bind_serving(uintptr_t process, uintptr_t greedy, uintptr_t greedy_workspace, uintptr_t copy) {
  g_process = reinterpret_cast<ProcessFn>(process);
  g_greedy = reinterpret_cast<GreedyFn>(greedy);
  g_greedy_workspace = reinterpret_cast<GreedyWorkspaceFn>(greedy_workspace);
  g_copy = reinterpret_cast<CopyFn>(copy);
}

bool plain(const at::Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() &&
         !at::isTensorSubclassLike(t);
}

// A buffer the kernels read in place.
bool buffer(const at::Tensor& t, const at::Device& dev, at::ScalarType dtype, int64_t numel, size_t align) {
  return plain(t) && t.device() == dev && t.scalar_type() == dtype && t.numel() == numel && t.is_contiguous() &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % align == 0;
}

// [N] (one group), [N, G] or [N, G, 1].
bool per_group(const at::Tensor& t, int64_t N, int64_t G) {
  const int64_t d = t.dim();
  return d >= 1 && d <= 3 && t.size(0) == N && (d > 1 ? t.size(1) == G : G == 1) && (d < 3 || t.size(2) == 1);
}

template <typename T>
const T* ptr(const std::optional<at::Tensor>& t) {
  return t ? static_cast<const T*>(t->const_data_ptr()) : nullptr;
}

// x [.., K] @ dequant(w [N, K/2])^T (+ bias) -> [.., N]. cast: other dtypes of x
// are computed in fp16 and converted back (without it they are not taken). bf16:
// x in bf16 is computed in bf16. build_tiled: the caller could make the tiled
// copy that it has not; calls that would run on it are then left to it.
// workspace_fn(nbytes) gives the stream's workspace.
py::object matmul(const at::Tensor& x, const at::Tensor& w, const at::Tensor& scales, const at::Tensor& zeros,
                  int64_t gs, const std::optional<at::Tensor>& perm, const std::optional<at::Tensor>& perm16,
                  const std::optional<at::Tensor>& s_gm, const std::optional<at::Tensor>& z_gm,
                  const std::optional<at::Tensor>& w_tiled, bool build_tiled, bool cast, bool bf16,
                  const std::optional<at::Tensor>& bias, int64_t device, uintptr_t stream,
                  const py::function& workspace_fn) {
  if (!g_matmul || !plain(x) || !plain(w) || x.dim() < 1 || w.dim() != 2 || gs <= 0) return py::none();
  const at::Device dev = x.device();
  const int64_t N = w.size(0), K = 2 * w.size(1);
  if (dev.index() != device || x.size(-1) != K || K == 0 || N == 0 || K % gs != 0 || x.numel() == 0)
    return py::none();
  const at::ScalarType in = x.scalar_type();
  const bool native = in == at::kBFloat16 && bf16;
  if (!native && in != at::kHalf && !(cast && (in == at::kBFloat16 || in == at::kFloat))) return py::none();
  const int64_t M = x.numel() / K, G = K / gs;
  if (!buffer(w, dev, at::kByte, N * (K / 2), 16) || !buffer(scales, dev, at::kFloat, N * G, 4) ||
      !buffer(zeros, dev, at::kByte, N * G, 1) || !per_group(scales, N, G) || !per_group(zeros, N, G))
    return py::none();
  if (perm && !buffer(*perm, dev, at::kInt, K, 4)) return py::none();
  if (perm16 && (!perm || !buffer(*perm16, dev, at::kShort, K, 16))) return py::none();
  if (s_gm.has_value() != z_gm.has_value()) return py::none();
  if (s_gm && (!buffer(*s_gm, dev, at::kFloat, N * G, 4) || !buffer(*z_gm, dev, at::kByte, N * G, 4) ||
               s_gm->dim() != 2 || s_gm->size(0) != G || z_gm->dim() != 2 || z_gm->size(0) != G))
    return py::none();
  if (w_tiled && !buffer(*w_tiled, dev, at::kByte, (N + 63) / 64 * 64 * (K / 2), 16)) return py::none();
  const int act = perm ? kChoicePerm : 0;
  if (!w_tiled && build_tiled && !(native && perm)) {
    const int c = g_choice(M, N, K, gs, kChoiceTiled | act);
    if (c == 5 || c == 6) return py::none();
  }
  const size_t need = g_workspace(M, N, K, gs, perm ? 1 : 0);
  if (!w_tiled && build_tiled && native &&
      g_route(M, N, K, gs, kBf16, kChoiceTiled | act, need) != g_route(M, N, K, gs, kBf16, kChoiceGm | act, need))
    return py::none();
  at::Tensor ws;
  if (need) {
    ws = workspace_fn(need).cast<at::Tensor>();
    if (!plain(ws) || ws.device() != dev) return py::none();
  }
  // other threads run meanwhile: a launch waits where the stream's queue is full
  std::optional<py::gil_scoped_release> unlocked(std::in_place);
  at::Tensor xc = native || in == at::kHalf ? x : x.to(at::kHalf);
  xc = xc.contiguous();
  if (reinterpret_cast<uintptr_t>(xc.const_data_ptr()) % 16) xc = xc.clone();
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, at::TensorOptions().dtype(xc.scalar_type()).device(dev));

  const int code = native ? kBf16 : kF16;
  const int rc = g_matmul(xc.const_data_ptr(), code, static_cast<const uint8_t*>(w.const_data_ptr()),
                          static_cast<const float*>(scales.const_data_ptr()), zeros.const_data_ptr(), kU8,
                          ptr<int32_t>(perm), ptr<uint16_t>(perm16), ptr<float>(s_gm), ptr<uint8_t>(z_gm),
                          ptr<uint8_t>(w_tiled), y.mutable_data_ptr(), code, M, N, K, gs,
                          need ? ws.mutable_data_ptr() : nullptr, need ? (size_t)ws.numel() : 0,
                          reinterpret_cast<void*>(stream));
  if (rc == 0 && y.scalar_type() != in) y = y.to(in);
  if (rc == 0 && bias) y = y + *bias;
  unlocked.reset();
  return rc == 0 ? py::cast(y) : py::none();
}

using Maybe = std::optional<at::Tensor>;

// No tensor, or a buffer of these sizes.
bool none_or(const Maybe& t, const at::Device& dev, at::ScalarType dtype, at::IntArrayRef sizes) {
  return !t || (plain(*t) && t->device() == dev && t->scalar_type() == dtype && t->sizes() == sizes && t->is_contiguous());
}

// Rows of a 2-D tensor that are contiguous and do not overlap; their stride.
bool rows(const at::Tensor& t, int64_t& stride) {
  stride = t.stride(0) > t.size(1) ? t.stride(0) : t.size(1);
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}

// A tensor whose gradient, or whose tangent, somebody waits for.
bool differentiated(const at::Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

// The processed logits, or with `greedy` their tokens: the arguments of pare_amd.process_logits and
// pare_amd.greedy_tokens in their order.
py::object logits(bool greedy, const at::Tensor& x, const Maybe& history, const Maybe& history_lens,
                  const Maybe& prompt_lens, const Maybe& repetition, const Maybe& presence, const Maybe& frequency,
                  const Maybe& bias_ids, const Maybe& bias, const Maybe& allowed, const Maybe& allowed_rows,
                  const Maybe& out, int64_t device, uintptr_t stream, const py::function& workspace_fn) {
  if (!g_process || !plain(x) || x.dim() != 2) return py::none();
  const at::Device dev = x.device();
  const at::ScalarType type = x.scalar_type();
  const int64_t R = x.size(0), V = x.size(1);
  if (dev.index() != device || R == 0 || V == 0 ||
      (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat))
    return py::none();
  const int code = type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : 2;
  int64_t stride, history_stride = 0, L = 0, n_bias = 0, masks = 0, words = 0;
  if (!rows(x, stride)) return py::none();
  if (history) {
    if (!plain(*history) || history->device() != dev || history->scalar_type() != at::kInt || history->dim() != 2 ||
        history->size(0) != R || !rows(*history, history_stride))
      return py::none();
    L = history->size(1);
  } else if (history_lens || prompt_lens || repetition || presence || frequency) {
    return py::none();
  }
  for (const Maybe* t : {&history_lens, &prompt_lens})
    if (!none_or(*t, dev, at::kInt, {R})) return py::none();
  for (const Maybe* t : {&repetition, &presence, &frequency})
    if (!none_or(*t, dev, at::kFloat, {R})) return py::none();
  if (bias_ids.has_value() != bias.has_value()) return py::none();
  if (bias_ids) {
    if (bias_ids->dim() != 2) return py::none();
    n_bias = bias_ids->size(1);
    if (!none_or(bias_ids, dev, at::kInt, {R, n_bias}) || !none_or(bias, dev, at::kFloat, {R, n_bias}))
      return py::none();
  }
  if (allowed) {
    if (allowed->dim() != 2) return py::none();
    masks = allowed->size(0), words = (V + 31) / 32;
    if (!none_or(allowed, dev, at::kInt, {masks, words}) || (!allowed_rows && masks != R)) return py::none();
  }
  if (!none_or(allowed_rows, dev, at::kInt, {R}) || (allowed_rows && !allowed)) return py::none();
  if (!greedy) {
    if (differentiated(x)) return py::none();
    for (const Maybe* t : {&repetition, &presence, &frequency, &bias, &out})
      if (*t && differentiated(**t)) return py::none();
  }
  at::Tensor y, ws;
  int64_t out_stride = greedy ? 1 : V;
  if (out) {
    y = *out;
    if (!plain(y) || y.device() != dev) return py::none();
    if (greedy) {
      if (y.scalar_type() != at::kLong || y.dim() < 1 || y.size(0) != R || y.numel() != R) return py::none();
      out_stride = R > 1 ? y.stride(0) : 1;
    } else if (y.scalar_type() != type || y.sizes() != x.sizes() || !rows(y, out_stride)) {
      return py::none();
    }
  }
  const size_t need = greedy ? g_greedy_workspace(R, V, code) : 0;
  if (need) {
    ws = workspace_fn(need).cast<at::Tensor>();
    if (!plain(ws) || ws.device() != dev) return py::none();
  }
  std::optional<py::gil_scoped_release> unlocked(std::in_place);
  if (!out) {
    const at::TensorOptions options = at::TensorOptions().device(dev);
    y = greedy ? at::empty({R}, options.dtype(at::kLong)) : at::empty({R, V}, options.dtype(type));
  }
  const auto call = [&](auto fn, auto... rest) {
    return fn(x.const_data_ptr(), code, stride, ptr<int32_t>(history), history_stride, L, ptr<int32_t>(history_lens),
              ptr<int32_t>(prompt_lens), ptr<float>(repetition), ptr<float>(presence), ptr<float>(frequency),
              ptr<int32_t>(bias_ids), ptr<float>(bias), n_bias, ptr<int32_t>(allowed), masks, words,
              ptr<int32_t>(allowed_rows), rest..., reinterpret_cast<void*>(stream));
  };
  const int rc = greedy ? call(g_greedy, static_cast<int64_t*>(y.mutable_data_ptr()), out_stride, R, V,
                               need ? ws.mutable_data_ptr() : nullptr, need ? (size_t)ws.numel() : (size_t)0)
                        : call(g_process, y.mutable_data_ptr(), out_stride, R, V);
  unlocked.reset();
  return rc == 0 ? py::cast(y) : py::none();
}

// Block tables, and the sizes that go with them.
struct Tables {
  at::Device dev = at::kCPU;
  int64_t R, width, stride;
  int32_t* at;
  bool of(const at::Tensor& t, int64_t device) {
    if (!plain(t) || t.dim() != 2 || t.scalar_type() != at::kInt || t.device().index() != device || !rows(t, stride))
      return false;
    dev = t.device(), R = t.size(0), width = t.size(1), at = t.mutable_data_ptr<int32_t>();
    return R > 0;
  }
  bool ints(const Maybe& t, int64_t n) const { return none_or(t, dev, at::kInt, {n}); }
  bool pool_of(const at::Tensor& free, const at::Tensor& pool, const Maybe& shares) const {
    return free.dim() == 1 && ints(free, free.size(0)) && ints(pool, 4) && ints(shares, free.size(0));
  }
};
int32_t* out(const Maybe& t) { return t ? t->mutable_data_ptr<int32_t>() : nullptr; }

// pare_amd.fork_block_tables: (src, dst).
py::object fork_tables(const at::Tensor& tables, const at::Tensor& kv_lens, const at::Tensor& parents,
                       const at::Tensor& free, const at::Tensor& pool, const at::Tensor& shares, const Maybe& lengths,
                       int64_t ps, int64_t device, uintptr_t stream) {
  Tables t;
  if (!g_fork || !t.of(tables, device) || !t.ints(kv_lens, t.R) || !t.ints(parents, t.R) || !t.ints(lengths, t.R) ||
      !t.pool_of(free, pool, shares))
    return py::none();
  const at::Tensor all = at::empty({3, t.R}, at::TensorOptions().dtype(at::kInt).device(t.dev));
  int32_t* p = all.mutable_data_ptr<int32_t>();
  int rc;
  {
    py::gil_scoped_release unlocked;
    rc = g_fork(t.at, t.stride, out(kv_lens), ptr<int32_t>(parents), ptr<int32_t>(lengths), ptr<int32_t>(free),
                out(pool), out(shares), p, p + t.R, p + 2 * t.R, t.R, t.width, free.size(0), ps,
                reinterpret_cast<void*>(stream));
  }
  return rc == 0 ? py::object(py::make_tuple(all.select(0, 0), all.select(0, 1))) : py::none();
}

// pare_amd.release_block_tables with shares: whether it was done.
bool release_tables(const at::Tensor& tables, const at::Tensor& kv_lens, const at::Tensor& done, const at::Tensor& free,
                    const at::Tensor& pool, const at::Tensor& shares, int64_t ps, int64_t device, uintptr_t stream) {
  Tables t;
  if (!g_release || !t.of(tables, device) || !t.ints(kv_lens, t.R) || !none_or(done, t.dev, at::kBool, {t.R}) ||
      !t.pool_of(free, pool, shares))
    return false;
  const size_t bytes = g_release_bytes(free.size(0));
  const at::Tensor scratch = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(t.dev));
  py::gil_scoped_release unlocked;
  return g_release(t.at, t.stride, out(kv_lens), reinterpret_cast<const uint8_t*>(done.const_data_ptr()), out(free),
                   out(pool), out(shares), t.R, t.width, free.size(0), ps, scratch.mutable_data_ptr(), bytes,
                   reinterpret_cast<void*>(stream)) == 0;
}

// pare_amd.compact_block_tables: (src, dst, count).
py::object compact_tables(const at::Tensor& tables, const at::Tensor& kv_lens, const at::Tensor& free,
                          const at::Tensor& pool, const Maybe& shares, int64_t ps, int64_t device, uintptr_t stream) {
  Tables t;
  if (!g_compact || !t.of(tables, device) || !t.ints(kv_lens, t.R) || !t.pool_of(free, pool, shares)) return py::none();
  const int64_t pages = free.size(0), half = pages / 2;
  if (pages == 0) return py::none();
  const size_t bytes = g_compact_bytes(pages);
  const at::Tensor all =
      at::empty({2 * half + 1 + (int64_t)(bytes / 4)}, at::TensorOptions().dtype(at::kInt).device(t.dev));
  int32_t* p = all.mutable_data_ptr<int32_t>();
  int rc;
  {
    py::gil_scoped_release unlocked;
    rc = g_compact(t.at, t.stride, ptr<int32_t>(kv_lens), out(free), out(pool), out(shares), p, p + half, p + 2 * half,
                   t.R, t.width, pages, ps, p + 2 * half + 1, bytes, reinterpret_cast<void*>(stream));
  }
  if (rc != 0) return py::none();
  return py::make_tuple(all.narrow(0, 0, half), all.narrow(0, half, half), all.narrow(0, 2 * half, 1));
}

// pare_amd.shared_prefixes: (starts, lens, runs).
py::object shared_prefixes(const at::Tensor& tables, const at::Tensor& kv_lens, const Maybe& q_starts, int64_t ps,
                           int64_t least_pages, int64_t device, uintptr_t stream, const py::function& workspace_fn) {
  Tables t;
  if (!g_runs || !t.of(tables, device) || !t.ints(kv_lens, t.R) || !t.ints(q_starts, t.R + 1)) return py::none();
  const size_t need = g_runs_bytes(t.R);
  if (!need) return py::none();
  const at::Tensor ws = workspace_fn(need).cast<at::Tensor>();
  if (!plain(ws) || ws.device() != t.dev) return py::none();
  const at::Tensor all = at::empty({6 * t.R + 1}, at::TensorOptions().dtype(at::kInt).device(t.dev));
  int32_t* p = all.mutable_data_ptr<int32_t>() + 4 * t.R;
  int rc;
  {
    py::gil_scoped_release unlocked;
    rc = g_runs(t.at, t.stride, ptr<int32_t>(kv_lens), ptr<int32_t>(q_starts), p, p + t.R + 1, p - 4 * t.R, t.R, t.width,
                ps, least_pages, ws.mutable_data_ptr(), (size_t)ws.numel(), reinterpret_cast<void*>(stream));
  }
  if (rc != 0) return py::none();
  return py::make_tuple(all.narrow(0, 4 * t.R, t.R + 1), all.narrow(0, 5 * t.R + 1, t.R),
                        all.narrow(0, 0, 4 * t.R).view({t.R, 4}));
}

// The layers' buffers of one kind: a sequence of tensors of the same sizes and type, or one tensor with the
// layers first. `first` is the first layer's.
bool layers(const py::object& all, const at::Device& dev, std::vector<void*>& at_layers, at::Tensor& first) {
  if (THPVariable_Check(all.ptr())) {
    const at::Tensor& t = THPVariable_Unpack(all.ptr());
    if (!plain(t) || t.device() != dev || t.dim() < 1 || t.size(0) == 0 || !t.is_contiguous()) return false;
    first = t.select(0, 0);
    for (int64_t i = 0; i < t.size(0); ++i)
      at_layers.push_back(static_cast<char*>(t.mutable_data_ptr()) + i * first.numel() * t.element_size());
    return true;
  }
  if (!PyList_Check(all.ptr()) && !PyTuple_Check(all.ptr())) return false;
  PyObject** items = PySequence_Fast_ITEMS(all.ptr());
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(all.ptr()); ++i) {
    if (!THPVariable_Check(items[i])) return false;
    const at::Tensor& t = THPVariable_Unpack(items[i]);
    if (i == 0) first = t;
    if (!plain(t) || t.device() != dev || t.scalar_type() != first.scalar_type() || t.sizes() != first.sizes() ||
        !t.is_contiguous())
      return false;
    at_layers.push_back(t.mutable_data_ptr());
  }
  return !at_layers.empty();
}

// pare_amd.copy_kv_pages: whether it was done.
bool copy_pages(const at::Tensor& src, const at::Tensor& dst, const Maybe& count, const py::object& k_caches,
                const py::object& v_caches, const py::object& k_scales, const py::object& v_scales, int64_t device,
                uintptr_t stream) {
  if (!g_copy || !plain(src)) return false;
  const at::Device dev = src.device();
  const int64_t n = src.numel();
  if (dev.index() != device || !none_or(src, dev, at::kInt, {n}) || !none_or(dst, dev, at::kInt, {n}) ||
      !none_or(count, dev, at::kInt, {1}))
    return false;
  std::vector<void*> kp, vp, ksp, vsp;
  at::Tensor k, v, ks, vs;
  if (!layers(k_caches, dev, kp, k) || !layers(v_caches, dev, vp, v) || !layers(k_scales, dev, ksp, ks) ||
      !layers(v_scales, dev, vsp, vs) || vp.size() != kp.size() || ksp.size() != kp.size() || vsp.size() != kp.size())
    return false;
  if (k.dim() != 4 || (k.scalar_type() != at::kChar && k.scalar_type() != at::kFloat8_e4m3fn) ||
      v.scalar_type() != k.scalar_type() || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat)
    return false;
  const int64_t pages = k.size(0), KV = k.size(1), ps = k.size(2), D = k.size(3);
  if (KV == 0 || ps % 16 || v.sizes() != at::IntArrayRef{pages, KV, ps / 16, D, 16} ||
      ks.sizes() != at::IntArrayRef{pages, KV} || vs.sizes() != ks.sizes())
    return false;
  py::gil_scoped_release unlocked;
  return g_copy(src.const_data_ptr<int32_t>(), dst.const_data_ptr<int32_t>(), ptr<int32_t>(count), n, kp.data(),
                vp.data(), reinterpret_cast<float* const*>(ksp.data()), reinterpret_cast<float* const*>(vsp.data()),
                (int64_t)kp.size(), pages, ps, KV, D, reinterpret_cast<void*>(stream)) == 0;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("bind", &bind);
  m.def("bind_serving", &bind_serving);
  m.def("bind_tables", &bind_tables);
  m.def("logits", &logits);
  m.def("fork_tables", &fork_tables);
  m.def("release_tables", &release_tables);
  m.def("compact_tables", &compact_tables);
  m.def("shared_prefixes", &shared_prefixes);
  m.def("copy_pages", &copy_pages);
  m.def("matmul", &matmul);
}
