"""A paged cache of 8-bit keys and values: serving sequences of different lengths.

The caller side of a serving loop, next to the fixed-length fp16 cache of
``decoder``: block tables and slot maps built on the device from request lengths
(``extend_block_tables``, ``release_block_tables``), the write of new tokens with
RoPE (``rope_append_kv``), attention of one or many new tokens per request
(``paged_attention``) and the read of whole pages (``read_kv_pages``).
``PagedKVCache`` holds the buffers of a model's layers and makes these calls.

The cache: codes int8 or float8_e4m3fn, code * scale = value,
  k_cache [pages, KV, page_size, D], v_cache [pages, KV, page_size / 16, D, 16]
  (token 16 b + j of a page at [b, :, j]), k_scale and v_scale fp32 [pages, KV].
page_size 16, 32, 64, 128 or 256, D 64 or 128. No call waits for the device, and all
of them can be captured into a graph. None has a reference counterpart: the
reference serves through HuggingFace's cache (pare/eval/throughput.py:84-126).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .kernels import _DeviceGuard, _raw_stream, _workspace

_CODES = {torch.int8: _lib.PMI_I8, torch.float8_e4m3fn: _lib.PMI_F8}
_VALUES = {torch.float16: _lib.PMI_F16, torch.bfloat16: _lib.PMI_BF16, torch.float32: _lib.PMI_F32}


class BatchPlan(NamedTuple):
    """What ``extend_block_tables`` says about a step (all int32, on the device)."""

    q_starts: torch.Tensor   # [R + 1] where each request's new tokens begin
    kv_lens: torch.Tensor    # [R] lengths with the new tokens
    first: torch.Tensor      # [R] position of its first new token, -1 if refused
    fresh: torch.Tensor      # [R + 1] pages that the requests before each one took
    positions: torch.Tensor  # [total] position of each new token
    slots: torch.Tensor      # [total] page * page_size + offset, -1: not stored
    pool: torch.Tensor       # [4] head and count of the free ring, requests refused, 0


def _hip(t: torch.Tensor, fn: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{fn} requires HIP (cuda) tensors.")
    return t.device


def _ints(dev: torch.device, n: int | None = None, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
        assert (t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous() and (n is None or t.numel() == n)), (
            f"{name} must be a contiguous int32 [{'n' if n is None else n}] tensor")


def _tables(tables: torch.Tensor, dev: torch.device, R: int) -> None:
    if tables.device != dev:
        raise RuntimeError(f"block_tables is on {tables.device}, expected {dev}")
    assert (tables.dtype == torch.int32 and tables.dim() == 2 and tables.shape[0] == R
            and (tables.shape[1] <= 1 or tables.stride(1) == 1)
            and (R <= 1 or tables.stride(0) >= tables.shape[1])), (
        f"block_tables must be an int32 [{R}, width] tensor with contiguous rows")


def _row_stride(tables: torch.Tensor) -> int:
    return max(tables.stride(0), tables.shape[1])


def _cache(dev: torch.device, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
           v_scale: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(pages, KV, page_size, D, code) of a cache, after its checks."""
    assert k_cache.dim() == 4 and v_cache.dim() == 5, (
        "k_cache must be [pages, KV, page_size, D] and v_cache [pages, KV, page_size / 16, D, 16]")
    pages, KV, ps, D = k_cache.shape
    assert KV > 0 and D > 0, "the caches must hold at least one head"
    assert tuple(v_cache.shape) == (pages, KV, ps // 16, D, 16) and ps % 16 == 0, (
        f"v_cache must be [{pages}, {KV}, {ps // 16}, {D}, 16], got {tuple(v_cache.shape)}")
    assert k_cache.dtype in _CODES and v_cache.dtype == k_cache.dtype, (
        "the caches must both be int8 or both float8_e4m3fn")
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "the caches must be contiguous"
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        assert t.dtype == torch.float32 and tuple(t.shape) == (pages, KV) and t.is_contiguous(), (
            f"{name} must be a contiguous float32 [{pages}, {KV}] tensor")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale)):
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
    return pages, KV, ps, D, _CODES[k_cache.dtype]


def extend_block_tables(block_tables: torch.Tensor, kv_lens: torch.Tensor, new_lens: torch.Tensor,
                        free_pages: torch.Tensor, pool: torch.Tensor, page_size: int, total: int, *,
                        kv_lens_out: torch.Tensor | None = None, pool_out: torch.Tensor | None = None,
                        max_len: int | None = None) -> BatchPlan:
    """Pages, slots and positions of a step in which request r gets ``new_lens[r]``
    more tokens, in one or two launches and without the host knowing the lengths.

    ``block_tables`` int32 [R, width] (its fresh entries are written), ``kv_lens`` and
    ``new_lens`` int32 [R], ``free_pages`` int32 [pages of the cache], the ring of free
    pages whose first entry and count are ``pool[0]`` and ``pool[1]`` (int32 [4];
    ``pool[2]`` counts refused requests), ``total`` the number of new tokens of all
    requests (fewer in fact: the rest get slot -1). A request whose table row is too
    short, that would be longer than ``max_len``, whose tokens pass ``total``, or that needs
    pages when the needs up to it exceed the pool, is refused: it keeps its length and its
    tokens get slot -1.
    ``kv_lens_out`` and ``pool_out`` may be ``kv_lens`` and ``pool``: the step is then taken
    in place."""
    dev = _hip(block_tables, "extend_block_tables")
    R = block_tables.shape[0]
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens, new_lens=new_lens)
    _ints(dev, free_pages=free_pages)
    _ints(dev, 4, pool=pool)
    if kv_lens_out is not None:
        _ints(dev, R, kv_lens_out=kv_lens_out)
    if pool_out is not None:
        _ints(dev, 4, pool_out=pool_out)
    assert max_len is None or max_len >= 0, "max_len may not be negative"
    cut = [R + 1, R, R + 1, total, total, R if kv_lens_out is None else 0, 4 if pool_out is None else 0]
    q_starts, first, fresh, positions, slots, lens, state = torch.empty(
        sum(cut), dtype=torch.int32, device=dev).split(cut)
    kv_lens_out = lens if kv_lens_out is None else kv_lens_out
    pool_out = state if pool_out is None else pool_out
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_extend_block_tables_upto(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), new_lens.data_ptr(),
            free_pages.data_ptr(), pool.data_ptr(), q_starts.data_ptr(), kv_lens_out.data_ptr(), first.data_ptr(),
            fresh.data_ptr(), positions.data_ptr(), slots.data_ptr(), pool_out.data_ptr(), R, block_tables.shape[1],
            free_pages.numel(), page_size, (1 << 31) - 1 if max_len is None else max_len, total, _raw_stream(dev)),
            "pmi_extend_block_tables")
    return BatchPlan(q_starts, kv_lens_out, first, fresh, positions, slots, pool_out)


def release_block_tables(block_tables: torch.Tensor, kv_lens: torch.Tensor, done: torch.Tensor,
                         free_pages: torch.Tensor, pool: torch.Tensor, page_size: int) -> None:
    """Gives the pages of the requests with ``done[r]`` (bool [R]) back to the ring of
    free pages, in request order, and sets their ``kv_lens`` to 0."""
    dev = _hip(block_tables, "release_block_tables")
    R = block_tables.shape[0]
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens)
    _ints(dev, free_pages=free_pages)
    _ints(dev, 4, pool=pool)
    assert (done.dtype == torch.bool and done.dim() == 1 and done.numel() == R and done.is_contiguous()
            and done.device == dev), (
        f"done must be a contiguous bool [{R}] tensor on {dev}")
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_release_block_tables(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), done.data_ptr(),
            free_pages.data_ptr(), pool.data_ptr(), R, block_tables.shape[1], free_pages.numel(), page_size,
            _raw_stream(dev)), "pmi_release_block_tables")


def rope_append_kv(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                   slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor) -> torch.Tensor:
    """Rotated q [T, H, D] of the fused rows ``qkv`` [T, (H + 2 KV) * D] (fp16 or bf16);
    the rotated k and the v of token t are quantised into slot ``slots[t]``.

    ``cos``, ``sin`` fp32 [L, D/2], indexed by ``positions`` int32 [T] (one outside the
    table takes its first or last row). Tokens with
    consecutive slots of one page form a run, and a page may be in one run only (as
    ``extend_block_tables`` makes them). A run raises its page's scale to what its values
    need; the page's older codes are rounded again to the new scale. Slots outside the
    cache are skipped. An infinity or NaN makes its page and head NaN."""
    dev = _hip(qkv, "rope_append_kv")
    pages, KV, ps, D, code = _cache(dev, k_cache, v_cache, k_scale, v_scale)
    assert qkv.dim() == 2 and qkv.dtype in (torch.float16, torch.bfloat16), (
        "qkv must be float16 or bfloat16 [T, (H + 2 KV) * D]")
    T, width = qkv.shape
    H = width // D - 2 * KV
    assert width % D == 0 and H > 0 and H % KV == 0, (
        f"qkv has {width} columns, expected (H + 2 * {KV}) * {D}")
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.stride(0) < width or qkv.data_ptr() % 16:
        qkv = torch.empty(T, width, dtype=qkv.dtype, device=dev).copy_(qkv)
    _ints(dev, T, positions=positions, slots=slots)
    for name, t in (("cos", cos), ("sin", sin)):
        assert (t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == D // 2 and t.is_contiguous()
                and t.device == dev and t.shape == cos.shape), (
            f"{name} must be a contiguous float32 [L, {D // 2}] tensor on {dev}")
    q = torch.empty(T, H, D, dtype=qkv.dtype, device=dev)
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_rope_append_kv(
            qkv.data_ptr(), _VALUES[qkv.dtype], max(qkv.stride(0), width), cos.data_ptr(), sin.data_ptr(),
            cos.shape[0], positions.data_ptr(), slots.data_ptr(), q.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), code, pages, ps, T, H, KV, D,
            _raw_stream(dev)), "pmi_rope_append_kv")
    return q


def read_kv_pages(pages: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, dtype: torch.dtype = torch.float16):
    """(k, v) [n, KV, page_size, D] of the n pages ``pages`` (int32), as values of ``dtype``
    (fp16, bf16 or fp32); zeros for a page number outside the cache."""
    dev = _hip(k_cache, "read_kv_pages")
    n_pages, KV, ps, D, code = _cache(dev, k_cache, v_cache, k_scale, v_scale)
    _ints(dev, pages=pages)
    assert dtype in _VALUES, "dtype must be float16, bfloat16 or float32"
    k = torch.empty(pages.numel(), KV, ps, D, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_read_kv_pages(
            pages.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), code,
            n_pages, ps, k.data_ptr(), v.data_ptr(), _VALUES[dtype], pages.numel(), KV, D, _raw_stream(dev)),
            "pmi_read_kv_pages")
    return k, v


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor,
                    q_starts: torch.Tensor | None = None, *, scale: float, window: int = 0,
                    max_q_len: int | None = None, max_kv_len: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention [T, H, D] of the queries ``q`` [T, H, D] (fp16 or bf16, any token and head
    strides) over the cache.

    Request r has the queries ``q_starts[r] .. q_starts[r + 1] - 1`` (int32 [R + 1]; None:
    one query each) and ``kv_lens[r]`` keys (int32 [R]), its own among them: query i of n
    sees positions up to ``kv_lens[r] - n + i``, with ``window`` > 0 the last ``window`` of
    those. A query that sees nothing gives zeros; rows behind the last request's are
    left as they were (``out``) or undefined. ``max_q_len`` and ``max_kv_len`` bound what
    a request has (default: all of q, the table's width): tighter bounds make the call
    faster, and queries and keys past them are left out.
    ``scale`` multiplies q . k."""
    dev = _hip(q, "paged_attention")
    pages, KV, ps, D, code = _cache(dev, k_cache, v_cache, k_scale, v_scale)
    assert q.dim() == 3 and q.shape[2] == D and q.dtype in (torch.float16, torch.bfloat16), (
        f"q must be float16 or bfloat16 [T, H, {D}]")
    T, H = q.shape[0], q.shape[1]
    R = kv_lens.numel()
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens)
    if q_starts is not None:
        _ints(dev, R + 1, q_starts=q_starts)
    else:
        assert T == R, f"without q_starts there is one query per request: q has {T}, kv_lens {R}"
        max_q_len = 1
    max_q = T if max_q_len is None else min(max_q_len, T)
    assert max_q >= 0 and window >= 0, "max_q_len and window may not be negative"
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = torch.empty(T, H, D, dtype=q.dtype, device=dev).copy_(q)
    if out is None:
        out = torch.empty(T, H, D, dtype=q.dtype, device=dev)
    else:
        assert (out.dtype == q.dtype and tuple(out.shape) == (T, H, D) and out.is_contiguous()
                and out.device == dev and out.data_ptr() % 16 == 0), (
            f"out must be a contiguous, 16-byte aligned [{T}, {H}, {D}] tensor of q's type")
    width = block_tables.shape[1]
    max_kv = width * ps if max_kv_len is None else min(max_kv_len, width * ps)
    assert max_kv >= 0, "max_kv_len may not be negative"
    L = _lib.lib()
    with _DeviceGuard(dev):
        stream = _raw_stream(dev)
        nbytes = L.pmi_paged_attention_workspace_bytes(T, R, H, KV, D, max_q, max_kv, window)
        ws = _workspace(dev, stream, nbytes)
        _lib.check(L.pmi_paged_attention(
            q.data_ptr(), _VALUES[q.dtype], q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), code, pages, ps, block_tables.data_ptr(),
            _row_stride(block_tables), kv_lens.data_ptr(), q_starts.data_ptr() if q_starts is not None else None,
            out.data_ptr(), T, R, width, H, KV, D, max_q, max_kv, window, scale,
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream),
            "pmi_paged_attention")
    return out


class PagedKVCache:
    """The paged 8-bit cache of a model's layers, with one block table for all of them.

    ``requests`` rows of up to ``max_len`` tokens share ``pages`` pages (default: enough
    for all of them at full length). ``extend`` makes room for a step's new tokens (never
    past ``max_len``, so RoPE tables of as many positions do),
    ``append`` writes them layer by layer, ``attend`` reads, ``release`` gives a finished
    request's pages back. ``pool[2]`` counts requests that ``extend`` refused."""

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, device, *,
                 page_size: int = 64, pages: int | None = None, dtype: torch.dtype = torch.int8) -> None:
        if dtype not in _CODES:
            raise ValueError("the cache holds int8 or float8_e4m3fn codes")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {page_size}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if layers < 0 or min(requests, max_len, kv_heads) < 1 or (pages is not None and pages < 1):
            raise ValueError("requests, max_len, kv_heads and pages must be positive, layers not negative")
        dev = torch.device(device)
        width = -(-max_len // page_size)
        pages = requests * width if pages is None else pages
        self.page_size, self.max_len = page_size, max_len
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=torch.uint8, device=dev).view(dtype) for _ in range(layers)]
        self.v = [torch.zeros(pages, kv_heads, page_size // 16, head_dim, 16, dtype=torch.uint8,
                              device=dev).view(dtype) for _ in range(layers)]
        self.k_scale = [torch.zeros(pages, kv_heads, device=dev) for _ in range(layers)]
        self.v_scale = [torch.zeros(pages, kv_heads, device=dev) for _ in range(layers)]
        self.block_tables = torch.full((requests, width), -1, dtype=torch.int32, device=dev)
        self.kv_lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=dev)
        self.pool = torch.tensor([0, pages, 0, 0], dtype=torch.int32, device=dev)

    def reset(self) -> None:
        """An empty cache: every page free."""
        pages = self.free_pages.numel()
        self.kv_lens.zero_()
        torch.arange(pages, out=self.free_pages)
        self.pool.zero_()
        self.pool[1:2].fill_(pages)  # (from the host's memory it would wait for the device)

    def extend(self, new_lens: torch.Tensor, total: int) -> BatchPlan:
        """``extend_block_tables`` in place."""
        return extend_block_tables(self.block_tables, self.kv_lens, new_lens, self.free_pages, self.pool,
                                   self.page_size, total, kv_lens_out=self.kv_lens, pool_out=self.pool,
                                   max_len=self.max_len)

    def release(self, done: torch.Tensor) -> None:
        release_block_tables(self.block_tables, self.kv_lens, done, self.free_pages, self.pool, self.page_size)

    def append(self, layer: int, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               plan: BatchPlan) -> torch.Tensor:
        return rope_append_kv(qkv, cos, sin, plan.positions, plan.slots, self.k[layer], self.v[layer],
                              self.k_scale[layer], self.v_scale[layer])

    def attend(self, layer: int, q: torch.Tensor, plan: BatchPlan, *, scale: float, window: int = 0,
               max_q_len: int | None = None, max_kv_len: int | None = None) -> torch.Tensor:
        return paged_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                               self.block_tables, plan.kv_lens, plan.q_starts, scale=scale, window=window,
                               max_q_len=max_q_len, max_kv_len=max_kv_len)
