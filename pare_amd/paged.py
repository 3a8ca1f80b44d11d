"""A paged cache of 8-bit keys and values: serving sequences of different lengths.

The caller side of a serving loop, next to the fixed-length fp16 cache of
``decoder``: block tables and slot maps built on the device from request lengths
(``extend_block_tables``, ``release_block_tables``), the write of new tokens with
RoPE (``rope_append_kv``), attention of one or many new tokens per request
(``paged_attention``) and the read of whole pages (``read_kv_pages``).
``PagedKVCache`` holds the buffers of a model's layers and makes these calls.

Requests may own pages together (``shares``, int32 [pages], counts a page's owners beyond
the first): ``fork_block_tables`` lets a request begin with another one's tokens,
``release_block_tables`` gives back what nobody else owns, ``compact_block_tables`` moves the
live pages to the cache's front, ``copy_kv_pages`` copies what both say. ``shared_prefixes``
finds the requests of a step whose first pages are the same, and ``paged_attention`` then
reads those once for all of them.

The cache: codes int8 or float8_e4m3fn, code * scale = value,
  k_cache [pages, KV, page_size, D], v_cache [pages, KV, page_size / 16, D, 16]
  (token 16 b + j of a page at [b, :, j]), k_scale and v_scale fp32 [pages, KV].
page_size 16, 32, 64, 128 or 256, D 64 or 128. No call waits for the device, and all
of them can be captured into a graph. None has a reference counterpart: the
reference serves through HuggingFace's cache (pare/eval/throughput.py:84-126).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

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


class PageMoves(NamedTuple):
    """Pages to be copied: ``src[i]`` to ``dst[i]`` (int32 [n], -1: none), of the first
    ``count[0]`` (int32 [1], on the device) if there is one."""

    src: torch.Tensor
    dst: torch.Tensor
    count: torch.Tensor | None


class SharedPrefixes(NamedTuple):
    """Runs of neighbouring requests that begin with the same pages (``shared_prefixes``)."""

    starts: torch.Tensor  # int32 [R + 1] the first request of each run, R behind the last
    lens: torch.Tensor    # int32 [R] positions that the members of a request's run share
    runs: torch.Tensor    # int32 [R, 4] first request, first query, queries and positions shared of each, or zeros


def _hip(t: torch.Tensor, fn: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{fn} requires HIP (cuda) tensors.")
    return t.device


def _here() -> tuple[int, int]:
    """The current device and its stream, for the calls of the host extension: it takes plain calls on
    that device, and leaves all others to the path behind it."""
    here = torch._C._cuda_getDevice()
    return here, torch._C._cuda_getCurrentRawStream(here)


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
                         free_pages: torch.Tensor, pool: torch.Tensor, page_size: int, *,
                         shares: torch.Tensor | None = None) -> None:
    """Gives the pages of the requests with ``done[r]`` (bool [R]) back to the ring of
    free pages, in request order, and sets their ``kv_lens`` to 0. With ``shares`` (int32
    [pages]) a page loses an owner for each of them, and goes back when it has none left,
    in the order of the pages' numbers."""
    dev = _hip(block_tables, "release_block_tables")
    if shares is not None and _lib.host().release_tables(block_tables, kv_lens, done, free_pages, pool, shares,
                                                         page_size, *_here()):
        return
    R = block_tables.shape[0]
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens)
    _ints(dev, free_pages=free_pages)
    _ints(dev, 4, pool=pool)
    assert (done.dtype == torch.bool and done.dim() == 1 and done.numel() == R and done.is_contiguous()
            and done.device == dev), (
        f"done must be a contiguous bool [{R}] tensor on {dev}")
    if shares is not None:
        _ints(dev, free_pages.numel(), shares=shares)
        L = _lib.lib()
        nbytes = L.pmi_release_shared_scratch_bytes(free_pages.numel())
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with _DeviceGuard(dev):
            _lib.check(L.pmi_release_shared_block_tables(
                block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), done.data_ptr(),
                free_pages.data_ptr(), pool.data_ptr(), shares.data_ptr(), R, block_tables.shape[1],
                free_pages.numel(), page_size, scratch.data_ptr(), nbytes, _raw_stream(dev)),
                "pmi_release_shared_block_tables")
        return
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_release_block_tables(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), done.data_ptr(),
            free_pages.data_ptr(), pool.data_ptr(), R, block_tables.shape[1], free_pages.numel(), page_size,
            _raw_stream(dev)), "pmi_release_block_tables")


def fork_block_tables(block_tables: torch.Tensor, kv_lens: torch.Tensor, parents: torch.Tensor,
                      free_pages: torch.Tensor, pool: torch.Tensor, shares: torch.Tensor, page_size: int, *,
                      lengths: torch.Tensor | None = None) -> PageMoves:
    """Request r begins with the first ``lengths[r]`` (int32 [R]; None, or more than there are: all)
    tokens of request ``parents[r]`` (int32 [R]; itself, or none of 0 .. R - 1: nothing
    happens), in place and without the host knowing any length.

    Their whole pages are owned by both from now on (``shares`` int32 [pages] counts a page's
    owners beyond the first); a last page that they do not fill is copied to a page from the ring:
    the returned moves ([R]) are for ``copy_kv_pages``, on the same stream. The copy is of the whole
    page with its scales, so a fork that ends inside a page reads its tokens as its parent does, bit for
    bit: as coarse as larger tokens behind them in that page have made them, and as NaN where
    one of those is an infinity or NaN (their own codes were lost with it). A parent is what it was
    before the call. Refused, and counted in ``pool[2]``, is a request that holds tokens, or that
    needs a page when the needs up to it exceed the pool."""
    dev = _hip(block_tables, "fork_block_tables")
    here, stream = _here()
    moves = _lib.host().fork_tables(block_tables, kv_lens, parents, free_pages, pool, shares, lengths, page_size, here,
                                    stream)
    if moves is not None:
        return PageMoves(*moves, None)
    R, width = block_tables.shape[0], block_tables.shape[1] if block_tables.dim() == 2 else 0
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens, parents=parents)
    _ints(dev, free_pages=free_pages)
    _ints(dev, free_pages.numel(), shares=shares)
    _ints(dev, 4, pool=pool)
    if lengths is not None:
        _ints(dev, R, lengths=lengths)
    src, dst, scratch = torch.empty(3, R, dtype=torch.int32, device=dev)
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_fork_block_tables(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), parents.data_ptr(),
            lengths.data_ptr() if lengths is not None else None, free_pages.data_ptr(), pool.data_ptr(),
            shares.data_ptr(), src.data_ptr(), dst.data_ptr(), scratch.data_ptr(), R, width, free_pages.numel(),
            page_size, _raw_stream(dev)), "pmi_fork_block_tables")
    return PageMoves(src, dst, None)


def compact_block_tables(block_tables: torch.Tensor, kv_lens: torch.Tensor, free_pages: torch.Tensor,
                         pool: torch.Tensor, shares: torch.Tensor | None, page_size: int) -> PageMoves:
    """Makes the n pages that the requests hold (by ``kv_lens`` and ``block_tables``) pages
    0 .. n - 1, in place: those from n on, in order, take the places of the free ones before it, in order.
    Pages n, n + 1, .. are the ring's free ones afterwards, in that order, also pages that
    neither a request nor the ring held. The returned moves ([pages / 2], as many as ``count``
    says) are for ``copy_kv_pages``, on the same stream. It is for between two steps: slots of a plan made
    before are of the old places. ``shares``: as in ``fork_block_tables``, or
    None."""
    dev = _hip(block_tables, "compact_block_tables")
    moves = _lib.host().compact_tables(block_tables, kv_lens, free_pages, pool, shares, page_size, *_here())
    if moves is not None:
        return PageMoves(*moves)
    R, width = block_tables.shape[0], block_tables.shape[1] if block_tables.dim() == 2 else 0
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens)
    _ints(dev, free_pages=free_pages)
    pages = free_pages.numel()
    _ints(dev, 4, pool=pool)
    if shares is not None:
        _ints(dev, pages, shares=shares)
    L = _lib.lib()
    nbytes = L.pmi_compact_scratch_bytes(pages)
    src, dst, count, scratch = torch.empty(2 * (pages // 2) + 1 + nbytes // 4, dtype=torch.int32, device=dev).split(
        [pages // 2, pages // 2, 1, nbytes // 4])
    with _DeviceGuard(dev):
        if pages == 0:
            count.zero_()
        _lib.check(L.pmi_compact_block_tables(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(), free_pages.data_ptr(),
            pool.data_ptr(), shares.data_ptr() if shares is not None else None, src.data_ptr(), dst.data_ptr(),
            count.data_ptr(), R, width, pages, page_size, scratch.data_ptr(), nbytes, _raw_stream(dev)),
            "pmi_compact_block_tables")
    return PageMoves(src, dst, count)


def copy_kv_pages(moves: PageMoves, k_caches: Sequence[torch.Tensor] | torch.Tensor,
                  v_caches: Sequence[torch.Tensor] | torch.Tensor, k_scales: Sequence[torch.Tensor] | torch.Tensor,
                  v_scales: Sequence[torch.Tensor] | torch.Tensor) -> None:
    """Copies the pages of ``moves``, codes and scales, in the caches of all layers (sequences of as
    many tensors each, all of the same sizes and type, or tensors with the layers first), in one
    launch per 64 layers. Pairs with a page that the cache does not have are left out; no page may be
    copied to twice, or be copied from and to."""
    _hip(moves.src, "copy_kv_pages")
    if _lib.host().copy_pages(*moves, k_caches, v_caches, k_scales, v_scales, *_here()):
        return
    k_caches, v_caches, k_scales, v_scales = (list(t) for t in (k_caches, v_caches, k_scales, v_scales))
    n = len(k_caches)
    assert len(v_caches) == n and len(k_scales) == n and len(v_scales) == n, (
        "the caches and scales must be sequences of one tensor a layer")
    dev = _hip(moves.src, "copy_kv_pages")
    _ints(dev, moves.src.numel(), src=moves.src, dst=moves.dst)
    if moves.count is not None:
        _ints(dev, 1, count=moves.count)
    if n == 0:
        return
    sizes = None
    for layer in zip(k_caches, v_caches, k_scales, v_scales):
        mine = _cache(dev, *layer)
        assert sizes is None or mine == sizes, "the caches of all layers must have the same sizes and type"
        sizes = mine
    pages, KV, ps, D, _ = sizes
    pointers = [(ctypes.c_void_p * n)(*[t.data_ptr() for t in ts]) for ts in (k_caches, v_caches, k_scales, v_scales)]
    with _DeviceGuard(dev):
        _lib.check(_lib.lib().pmi_copy_kv_pages(
            moves.src.data_ptr(), moves.dst.data_ptr(), moves.count.data_ptr() if moves.count is not None else None,
            moves.src.numel(), *pointers, n, pages, ps, KV, D, _raw_stream(dev)), "pmi_copy_kv_pages")


def shared_prefixes(block_tables: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor | None,
                    page_size: int, *, least: int = 256) -> SharedPrefixes:
    """Which neighbouring requests of a step begin with the same pages, for ``paged_attention``.

    ``kv_lens`` int32 [R] with the new tokens that ``q_starts`` int32 [R + 1] counts (None: one
    each). A request joins the run of the request with new tokens before it if at least
    ``least`` positions of theirs, in whole pages before their new tokens, lie in the same pages;
    the members of a run share what all of them have in common. Where groups of requests share more with
    each other than with their neighbours (a document each, behind one system prompt), ``least`` has to be
    above what all have in common for each group to be a run; else they are one run, which
    shares that alone."""
    dev = _hip(block_tables, "shared_prefixes")
    here, stream = _here()
    runs = _lib.host().shared_prefixes(block_tables, kv_lens, q_starts, page_size, -(-least // max(page_size, 1)), here,
                                       stream, lambda nbytes: _workspace(dev, stream, nbytes))
    if runs is not None:
        return SharedPrefixes(*runs)
    R, width = block_tables.shape[0], block_tables.shape[1] if block_tables.dim() == 2 else 0
    _tables(block_tables, dev, R)
    _ints(dev, R, kv_lens=kv_lens)
    if q_starts is not None:
        _ints(dev, R + 1, q_starts=q_starts)
    assert least >= 1, "least must be at least one position"
    runs, starts, lens = torch.empty(6 * R + 1, dtype=torch.int32, device=dev).split([4 * R, R + 1, R])
    L = _lib.lib()
    with _DeviceGuard(dev):
        stream = _raw_stream(dev)
        if R == 0:
            starts.zero_()
        ws = _workspace(dev, stream, L.pmi_shared_prefixes_workspace_bytes(R))
        _lib.check(L.pmi_shared_prefixes(
            block_tables.data_ptr(), _row_stride(block_tables), kv_lens.data_ptr(),
            q_starts.data_ptr() if q_starts is not None else None, starts.data_ptr(), lens.data_ptr(),
            runs.data_ptr(), R, width, page_size, -(-least // max(page_size, 1)),
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream),
            "pmi_shared_prefixes")
    return SharedPrefixes(starts, lens, runs.view(R, 4))


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
                    out: torch.Tensor | None = None, shared: SharedPrefixes | None = None) -> torch.Tensor:
    """Attention [T, H, D] of the queries ``q`` [T, H, D] (fp16 or bf16, any token and head
    strides) over the cache.

    Request r has the queries ``q_starts[r] .. q_starts[r + 1] - 1`` (int32 [R + 1]; None:
    one query each) and ``kv_lens[r]`` keys (int32 [R]), its own among them: query i of n
    sees positions up to ``kv_lens[r] - n + i``, with ``window`` > 0 the last ``window`` of
    those. A query that sees nothing gives zeros; rows behind the last request's are
    left as they were (``out``) or undefined. ``max_q_len`` and ``max_kv_len`` bound what
    a request has (default: all of q, the table's width): tighter bounds make the call
    faster, and queries and keys past them are left out.
    ``scale`` multiplies q . k.

    ``shared``: what ``shared_prefixes`` says of the same tables, lengths and queries. The result
    is the same but for roundings; keys that a run of requests shares are read once for all of it
    where that pays: from 2048 keys (``max_kv_len``) and 2^27 bytes of all requests' keys and values on, up
    to 32 query rows a request (``max_q_len`` H / KV), without a window. The bounds decide for the whole
    call, whatever the requests hold: with ``q_starts`` and no ``max_q_len`` the one is all of q, and one
    request of many new tokens among single ones takes the sharing from all."""
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
    if shared is not None:
        _ints(dev, R, lens=shared.lens)
        assert shared.runs.is_contiguous(), "runs must be contiguous"
        _ints(dev, 4 * R, runs=shared.runs.view(-1))
        with _DeviceGuard(dev):
            stream = _raw_stream(dev)
            ws = _workspace(dev, stream, L.pmi_paged_attention_shared_workspace_bytes(T, R, H, KV, D, max_q, max_kv,
                                                                                      window))
            _lib.check(L.pmi_paged_attention_shared(
                q.data_ptr(), _VALUES[q.dtype], q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), code, pages, ps, block_tables.data_ptr(),
                _row_stride(block_tables), kv_lens.data_ptr(), q_starts.data_ptr() if q_starts is not None else None,
                shared.runs.data_ptr(), shared.lens.data_ptr(), out.data_ptr(), T, R, width, H, KV, D, max_q,
                max_kv, window, scale, ws.data_ptr() if ws is not None else None,
                ws.numel() if ws is not None else 0, stream), "pmi_paged_attention_shared")
        return out
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
    request's pages back. ``pool[2]`` counts requests that ``extend`` and ``fork`` refused.

    With ``sharing`` requests may begin as forks of others (``fork``), whose whole pages they then
    own together; ``shared_prefixes`` tells ``attend`` which those are. ``compact`` moves the
    live pages to the front, ``resize`` changes how many pages there are."""

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, device, *,
                 page_size: int = 64, pages: int | None = None, dtype: torch.dtype = torch.int8,
                 sharing: bool = False) -> None:
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
        self.shares = torch.zeros(pages, dtype=torch.int32, device=dev) if sharing else None

    def reset(self) -> None:
        """An empty cache: every page free."""
        pages = self.free_pages.numel()
        self.kv_lens.zero_()
        if self.shares is not None:
            self.shares.zero_()
        torch.arange(pages, out=self.free_pages)
        self.pool.zero_()
        self.pool[1:2].fill_(pages)  # (from the host's memory it would wait for the device)

    def extend(self, new_lens: torch.Tensor, total: int) -> BatchPlan:
        """``extend_block_tables`` in place."""
        return extend_block_tables(self.block_tables, self.kv_lens, new_lens, self.free_pages, self.pool,
                                   self.page_size, total, kv_lens_out=self.kv_lens, pool_out=self.pool,
                                   max_len=self.max_len)

    def release(self, done: torch.Tensor) -> None:
        release_block_tables(self.block_tables, self.kv_lens, done, self.free_pages, self.pool, self.page_size,
                             shares=self.shares)

    def fork(self, parents: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """``fork_block_tables`` in place, with the copies of all layers; not between a step's ``extend`` and its
        last ``append``, when the parents' lengths count tokens that are not there to be copied."""
        if self.shares is None:
            raise RuntimeError("fork needs a cache made with sharing=True")
        self._copy(fork_block_tables(self.block_tables, self.kv_lens, parents, self.free_pages, self.pool, self.shares,
                                     self.page_size, lengths=lengths))

    def compact(self) -> None:
        """``compact_block_tables`` in place, with the copies of all layers; not between a step's ``extend``
        and its last ``append``, whose plan has the old slots."""
        self._copy(compact_block_tables(self.block_tables, self.kv_lens, self.free_pages, self.pool, self.shares,
                                        self.page_size))

    def _copy(self, moves: PageMoves) -> None:
        copy_kv_pages(moves, self.k, self.v, self.k_scale, self.v_scale)

    def resize(self, pages: int) -> None:
        """A cache of ``pages`` pages with the same requests, after ``compact``. The buffers are new
        ones (a graph captured before writes to the old ones), and the call waits for the device."""
        if pages < 1:
            raise ValueError("pages must be positive")
        self.compact()
        old, dev = self.free_pages.numel(), self.free_pages.device
        live = old - int(self.pool[1])
        if pages < live:
            raise ValueError(f"the requests hold {live} pages, more than {pages}")
        for buffers in (self.k, self.v, self.k_scale, self.v_scale):
            for i, t in enumerate(buffers):
                raw = t.view(torch.uint8) if t.dtype != torch.float32 else t
                new = torch.zeros(pages, *t.shape[1:], dtype=raw.dtype, device=dev)
                new[:live] = raw[:live]
                buffers[i] = new.view(t.dtype)
        if self.shares is not None:
            shares = torch.zeros(pages, dtype=torch.int32, device=dev)
            shares[:live] = self.shares[:live]
            self.shares = shares
        self.free_pages = ((torch.arange(pages, device=dev) + live) % pages).to(torch.int32)
        self.pool[1:2].fill_(pages - live)

    def shared_prefixes(self, plan: BatchPlan, least: int = 256) -> SharedPrefixes:
        """Which of the plan's requests begin with the same pages, for ``attend``: once a step."""
        return shared_prefixes(self.block_tables, plan.kv_lens, plan.q_starts, self.page_size, least=least)

    def append(self, layer: int, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               plan: BatchPlan) -> torch.Tensor:
        return rope_append_kv(qkv, cos, sin, plan.positions, plan.slots, self.k[layer], self.v[layer],
                              self.k_scale[layer], self.v_scale[layer])

    def attend(self, layer: int, q: torch.Tensor, plan: BatchPlan, *, scale: float, window: int = 0,
               max_q_len: int | None = None, max_kv_len: int | None = None,
               shared: SharedPrefixes | None = None) -> torch.Tensor:
        return paged_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                               self.block_tables, plan.kv_lens, plan.q_starts, scale=scale, window=window,
                               max_q_len=max_q_len, max_kv_len=max_kv_len, shared=shared)
