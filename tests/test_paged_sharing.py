"""Pages of the cache that several requests own, and attention that reads them once, against
plain implementations (oracle/sharing_oracle.py, oracle/serving_oracle.py): forks, releases,
compaction, copies, runs, refusals, capture."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
import torch

import pare_amd as P
from oracle import serving_oracle as S
from oracle import sharing_oracle as O
from pare_amd import _lib

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
CODES = [torch.int8, torch.float8_e4m3fn]
P8 = 0x1000  # an aligned address that is never read: validation comes first
BAD = (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# --- the oracle, refusals (CPU) -----------------------------------------------------------

def test_oracle_by_hand():
    t = [[4, 2, 9], [-1, -1, -1], [-1, -1, -1], [7, -1, -1]]
    got = O.fork(t, [40, 0, 0, 16], [-1, 0, 0, 0], [0, 40, 35, 3], [5, 6, 1, 0, 0, 0, 0, 0, 0, 0], [1, 2, 0, 0], [0] * 10, 16)
    assert got[0] == [[4, 2, 9], [4, 2, 6], [4, 2, 1], [7, -1, -1]] and got[1] == [40, 40, 35, 16]
    assert got[2] == [3, 0, 1, 0] and got[3] == [0, 0, 2, 0, 2] + [0] * 5  # request 3 holds tokens
    assert got[4:] == ([-1, 9, 9, -1], [-1, 6, 1, -1])
    lens, free, pool, shares = O.release(got[0], got[1], [1, 1, 0, 0], [0] * 10, [3, 0, 0, 0], got[3], 16)
    assert lens == [0, 0, 35, 16] and free[3:5] == [6, 9] and pool[1] == 2 and shares == [0] * 10
    tables, free, pool, shares, src, dst = O.compact(got[0], lens, [3, 2, 1, 0], [0] * 10, 16)
    # pages 1, 2, 4 and 7 are live: 4 and 7 take the places of 0 and 3
    assert tables[2:] == [[0, 2, 1], [3, -1, -1]] and free[:3] == [4, 5, 6] and pool == [0, 6, 1, 0]
    assert (src, dst) == ([4, 7, -1, -1, -1], [0, 3, -1, -1, -1])
    assert O.runs([[1, 2, 3], [1, 2, 4], [1, 2, 3], [5, 2, 3]], [48, 48, 0, 33], None, 16, 32) == \
        ([0, 3, 4, 4, 4], [32, 32, 0, 0], [[0, 0, 3, 32]] + [[0] * 4] * 3)


def _fork_args(**kw):
    a = dict(t=P8, stride=4, lens=P8, parents=P8, lengths=P8, free=P8, pool=P8, shares=P8, src=P8, dst=P8, scratch=P8,
             R=2, width=4, ring=8, ps=16)
    a.update(kw)
    return [*a.values(), None]


def _release_args(**kw):
    a = dict(t=P8, stride=4, lens=P8, done=P8, free=P8, pool=P8, shares=P8, R=2, width=4, ring=8, ps=16, scratch=P8,
             nbytes=1 << 20)
    a.update(kw)
    return [*a.values(), None]


def _compact_args(**kw):
    a = dict(t=P8, stride=4, lens=P8, free=P8, pool=P8, shares=P8, src=P8, dst=P8, moves=P8, R=2, width=4, ring=8,
             ps=16, scratch=P8, nbytes=1 << 20)
    a.update(kw)
    return [*a.values(), None]


def _copy_args(layers=2, **kw):
    one = (ctypes.c_void_p * 2)(P8, P8)
    a = dict(src=P8, dst=P8, count=None, n=3, k=one, v=one, ks=one, vs=one, layers=layers, pages=4, ps=16, KV=2, D=64)
    a.update(kw)
    return [*a.values(), None]


def _runs_args(**kw):
    a = dict(t=P8, stride=4, lens=P8, starts=P8, out=P8, shared=P8, runs=P8, R=2, width=4, ps=16, least=1, ws=P8, nbytes=1 << 20)
    a.update(kw)
    return [*a.values(), None]


SIZES = [dict(R=-1), dict(R=4097), dict(width=-1), dict(stride=3), dict(ps=24), dict(width=1 << 30, stride=1 << 30)]
RING = [dict(ring=-1), dict(ring=1 << 30), dict(free=None), dict(pool=None)]


@pytest.mark.parametrize("change", SIZES + RING + [dict(t=None), dict(lens=None), dict(parents=None), dict(shares=None),
                                                   dict(src=None), dict(dst=None), dict(scratch=None)])
def test_fork_refuses(change):
    assert _lib.lib().pmi_fork_block_tables(*_fork_args(**change)) in BAD


@pytest.mark.parametrize("change", SIZES + RING + [dict(t=None), dict(lens=None), dict(done=None), dict(shares=None),
                                                   dict(scratch=None), dict(nbytes=4), dict(scratch=P8 + 2)])
def test_release_refuses(change):
    assert _lib.lib().pmi_release_shared_block_tables(*_release_args(**change)) in BAD


@pytest.mark.parametrize("change", SIZES + RING + [dict(t=None), dict(lens=None), dict(src=None), dict(dst=None),
                                                   dict(moves=None), dict(scratch=None), dict(nbytes=60),
                                                   dict(scratch=P8 + 2)])
def test_compact_refuses(change):
    assert _lib.lib().pmi_compact_block_tables(*_compact_args(**change)) in BAD


@pytest.mark.parametrize("change", [dict(n=-1), dict(n=1 << 31), dict(layers=-1), dict(src=None), dict(dst=None), dict(k=None),
                                    dict(vs=None), dict(k=(ctypes.c_void_p * 2)(P8, None)),
                                    dict(v=(ctypes.c_void_p * 2)(P8, P8 + 8)), dict(D=96), dict(ps=17), dict(KV=0),
                                    dict(pages=-1)])
def test_copy_refuses(change):
    assert _lib.lib().pmi_copy_kv_pages(*_copy_args(**change)) in BAD


@pytest.mark.parametrize("change", SIZES + [dict(t=None), dict(lens=None), dict(out=None), dict(shared=None),
                                            dict(runs=None), dict(runs=P8 + 4), dict(least=0), dict(least=1 << 31), dict(ws=None), dict(ws=P8 + 16),
                                            dict(nbytes=100)])
def test_shared_prefixes_refuses(change):
    assert _lib.lib().pmi_shared_prefixes(*_runs_args(**change)) in BAD


def _attention_args(**kw):
    a = dict(q=P8, dtype=_lib.PMI_F16, stride=512, head=128, k=P8, v=P8, ks=P8, vs=P8, code=_lib.PMI_I8, pages=4, ps=16,
             tables=P8, tstride=4, lens=P8, starts=P8, runs=P8, shared=P8, out=P8, T=2, R=2, width=4, H=4, KV=1, D=128,
             max_q=2, max_kv=64, window=0, scale=1.0, ws=P8, ws_bytes=1 << 40)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("change", [dict(runs=None), dict(runs=P8 + 8), dict(shared=None), dict(dtype=_lib.PMI_F32), dict(D=80), dict(ps=48),
                                    dict(H=65), dict(scale=float("nan")), dict(ws=None), dict(ws_bytes=1 << 16),
                                    dict(ws=P8 + 16), dict(lens=None), dict(tables=None), dict(max_q=-1),
                                    dict(T=1 << 25, max_q=64, H=64, KV=64, R=1 << 25, starts=None)])
def test_shared_attention_refuses(change):
    assert _lib.lib().pmi_paged_attention_shared(*_attention_args(**change)) in BAD


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert L.pmi_fork_block_tables(*_fork_args(R=0, t=None, lens=None, src=None)) == _lib.PMI_OK
    assert L.pmi_release_shared_block_tables(*_release_args(R=0, t=None)) == _lib.PMI_OK
    assert L.pmi_release_shared_block_tables(*_release_args(ring=0, scratch=None)) == _lib.PMI_OK
    assert L.pmi_compact_block_tables(*_compact_args(ring=0, free=None, scratch=None)) == _lib.PMI_OK
    assert L.pmi_copy_kv_pages(*_copy_args(n=0, src=None)) == _lib.PMI_OK
    assert L.pmi_copy_kv_pages(*_copy_args(layers=0)) == _lib.PMI_OK
    assert L.pmi_copy_kv_pages(*_copy_args(pages=0)) == _lib.PMI_OK
    assert L.pmi_shared_prefixes(*_runs_args(R=0, t=None, ws=None)) == _lib.PMI_OK
    assert L.pmi_paged_attention_shared(*_attention_args(T=0, R=0, starts=None)) == _lib.PMI_OK


def test_cpu_tensors_raise():
    t, i = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: P.fork_block_tables(t, i[:1], i[:1], i, i, i, 16),
                 lambda: P.compact_block_tables(t, i[:1], i, i, i, 16),
                 lambda: P.shared_prefixes(t, i[:1], None, 16),
                 lambda: P.copy_kv_pages(P.PageMoves(i, i, None), [], [], [], [])):
        with pytest.raises(RuntimeError):
            call()


# --- tables ---------------------------------------------------------------------------------

class _Pool:
    """A consistent cache's tables on the host: requests, some of them with pages in common."""

    def __init__(self, rng, R, ps, longest, parents, children, spare, width=None):
        lens = [rng.randint(1, longest) if r < parents else 0 for r in range(R)]
        self.ps, self.R = ps, R
        self.width = width or -(-longest // ps) + 2
        need = sum(-(-n // ps) for n in lens) + 3 * children
        self.pages = need + spare
        order = list(range(self.pages))
        rng.shuffle(order)
        self.tables = [[rng.randint(-1, self.pages) for _ in range(self.width)] for _ in range(R)]
        self.shares = [0] * self.pages
        for r in range(parents):
            for j in range(-(-lens[r] // ps)):
                self.tables[r][j] = order.pop()
        for r in range(parents, parents + children):
            p = rng.randrange(r)
            n = rng.randint(0, max(lens[p], 0))
            for j in range(n // ps):
                self.tables[r][j] = self.tables[p][j]
                self.shares[self.tables[p][j]] += 1
            own = min(rng.randint(1, 3), self.width - n // ps)
            for j in range(n // ps, n // ps + own):
                self.tables[r][j] = order.pop()
            lens[r] = max(0, ps * (n // ps + own) - rng.randrange(ps))
        self.lens = lens
        head = rng.randrange(self.pages)
        self.free = [rng.randint(-3, self.pages) for _ in range(self.pages)]
        for i, p in enumerate(order):
            self.free[(head + i) % self.pages] = p
        self.pool = [head, len(order), rng.randint(0, 5), 0]

    def device(self):
        t = torch.full((self.R, self.width + 3), 77, dtype=torch.int32, device=DEV)
        view = t[:, :self.width]  # rows of a wider buffer
        view.copy_(_ints(self.tables).view(self.R, self.width))
        return view, _ints(self.lens), _ints(self.free), _ints(self.pool), _ints(self.shares)


@gpu
@pytest.mark.parametrize("R,ps,longest,parents,spare", [(1, 16, 40, 1, 0), (5, 16, 200, 2, 1), (40, 32, 3000, 7, 20),
                                                        (600, 64, 9000, 30, 300), (4096, 16, 300, 96, 2500)])
@pytest.mark.parametrize("given", [False, True])
def test_fork(R, ps, longest, parents, spare, given):
    rng = random.Random(R + given)
    for _ in range(3):
        c = _Pool(rng, R, ps, longest, parents, 0, spare)
        want_of = [rng.randrange(-1, R + 1) if rng.random() < 0.2 else rng.randrange(parents) for _ in range(R)]
        lengths = [rng.choice([0, -3, ps, 10 ** 6, rng.randint(0, longest)]) for _ in range(R)] if given else None
        t, lens, free, pool, shares = c.device()
        moves = P.fork_block_tables(t, lens, _ints(want_of), free, pool, shares, ps,
                                    lengths=_ints(lengths) if given else None)
        want = O.fork(c.tables, c.lens, want_of, lengths, c.free, c.pool, c.shares, ps)
        for g, w in zip((t, lens, pool, shares, moves.src, moves.dst), want):
            assert g.tolist() == w
        assert free.tolist() == c.free and moves.count is None
        if t.stride(0) > c.width:
            assert (t._base[:, c.width:] == 77).all()


@gpu
def test_fork_of_strange_states():
    """Negative lengths, lengths past the table, entries outside the cache, a pool that no cache has."""
    t = _ints([[5, -1, 99], [0, 0, 0], [0, 0, 0], [3, 3, 3]]).view(4, 3)
    lens, shares = _ints([1000, -7, 0, -2]), _ints([0] * 6)
    for pool in ([0, 6, 0, 0], [-5, 100, 2, 9]):
        tt, ll, ss, pp = t.clone(), lens.clone(), shares.clone(), _ints(pool)
        m = P.fork_block_tables(tt, ll, _ints([1, 0, 3, 2]), _ints([1, 2, 3, 4, 5, 0]), pp, ss, 16)
        # 0 holds tokens; 1 takes its whole row (48 tokens); 2 and 3 begin empty
        assert ll.tolist() == [1000, 48, 0, 0] and tt.tolist()[1] == [5, -1, 99] and ss.tolist() == [0, 0, 0, 0, 0, 1]
        assert m.src.tolist() == [-1] * 4 and pp.tolist() == [0, 6, pool[2] + 1, 0]
    none = P.fork_block_tables(t[:0], lens[:0], lens[:0], shares, _ints([0, 6, 0, 0]), shares, 16)
    assert none.src.numel() == 0
    empty = torch.zeros(0, dtype=torch.int32, device=DEV)  # a cache of no pages
    pool = _ints([0, 0, 0, 0])
    ll = _ints([5, 0, 0, 0])
    P.fork_block_tables(t, ll, _ints([0, 0, 0, 3]), empty, pool, empty, 16)
    assert ll.tolist() == [5, 0, 0, 0] and pool.tolist() == [0, 0, 2, 0]


@gpu
@pytest.mark.parametrize("R,ps,longest,parents,children,spare", [(1, 16, 40, 1, 0, 0), (9, 16, 200, 2, 7, 3),
                                                                 (60, 32, 3000, 10, 50, 20), (300, 16, 3000, 40, 200, 9000),
                                                                 (4096, 16, 100, 2000, 2096, 5), (6, 16, 200, 3, 3, 16330),
                                                                 (6, 16, 200, 3, 3, 16400)])
def test_release_of_shared_pages(R, ps, longest, parents, children, spare):
    rng = random.Random(R)
    for share in (0.3, 1.0, 0.0):
        c = _Pool(rng, R, ps, longest, parents, children, spare)
        done = [rng.random() < share for _ in range(R)]
        t, lens, free, pool, shares = c.device()
        P.release_block_tables(t, lens, torch.tensor(done, device=DEV), free, pool, ps, shares=shares)
        want = O.release(c.tables, c.lens, done, c.free, c.pool, c.shares, ps)
        for g, w in zip((lens, free, pool, shares), want):
            assert g.tolist() == w
        assert t.tolist() == c.tables
        if share == 1.0:
            assert pool.tolist()[1] == c.pages and not any(shares.tolist())


@gpu
@pytest.mark.parametrize("R,ps,longest,parents,children,spare", [(1, 16, 40, 1, 0, 0), (9, 16, 200, 2, 7, 3),
                                                                 (60, 32, 3000, 10, 50, 900), (300, 16, 3000, 40, 200, 9000),
                                                                 (4096, 16, 100, 2000, 2096, 5), (3, 16, 20, 0, 0, 5000),
                                                                 (6, 16, 200, 3, 3, 16330), (6, 16, 200, 3, 3, 16400),
                                                                 (2, 256, 100, 1, 0, 0)])
@pytest.mark.parametrize("shared", [True, False])
def test_compact(R, ps, longest, parents, children, spare, shared):
    rng = random.Random(R)
    for lost in (0.0, 0.5):
        c = _Pool(rng, R, ps, longest, parents, children if shared else 0, spare)
        for r in range(R):  # requests that are gone, and pages that nobody knows of
            if rng.random() < lost:
                c.lens[r] = rng.choice([0, -4])
        t, lens, free, pool, shares = c.device()
        moves = P.compact_block_tables(t, lens, free, pool, shares if shared else None, ps)
        want = O.compact(c.tables, c.lens, c.pool, c.shares, ps)
        for g, w in zip((t, free, pool, shares, moves.src, moves.dst), want):
            if g is not shares or shared:
                assert g.tolist() == w
        assert moves.count.tolist() == [sum(x >= 0 for x in want[4])] and lens.tolist() == c.lens


@gpu
def test_compact_without_requests_or_pages():
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    pool = _ints([0, 0, 3, 0])
    m = P.compact_block_tables(_ints([[1]]).view(1, 1), _ints([0]), e, pool, None, 16)
    assert m.count.tolist() == [0] and m.src.numel() == 0
    free, pool = _ints([2, 1, 0, 9, 9]), _ints([1, 2, 3, 0])
    m = P.compact_block_tables(_ints([[1]])[:0].view(0, 1), e, free, pool, None, 16)
    assert free.tolist() == [0, 1, 2, 3, 4] and pool.tolist() == [0, 5, 3, 0] and m.src.tolist() == [-1, -1]


@gpu
@pytest.mark.parametrize("layers,pages,KV,ps,D", [(1, 5, 1, 16, 64), (3, 40, 8, 64, 128), (70, 9, 3, 32, 64), (2, 7, 5, 256, 128)])
@pytest.mark.parametrize("code", CODES)
def test_copy(layers, pages, KV, ps, D, code):
    g = torch.Generator(device=DEV).manual_seed(pages)
    rand = lambda *s: torch.randint(0, 256, s, dtype=torch.uint8, generator=g, device=DEV)  # noqa: E731
    k = [rand(pages, KV, ps, D).view(code) for _ in range(layers)]
    v = [rand(pages, KV, ps // 16, D, 16).view(code) for _ in range(layers)]
    s = [[torch.rand(pages, KV, generator=g, device=DEV) for _ in range(layers)] for _ in range(2)]
    src, dst = [0, -1, pages - 1, 2, 0, pages, 0, 4], [1, 2, 3, -1, pages, 4, -5, 4 if pages < 6 else 5]
    for count in (None, 1, 0, 100, -3):
        before = [[t.clone() for t in group] for group in (k, v, *s)]
        P.copy_kv_pages(P.PageMoves(_ints(src), _ints(dst), None if count is None else _ints([count])), k, v, *s)
        todo = list(zip(src, dst))[:len(src) if count is None else max(count, 0)]
        for group, old in zip((k, v, *s), before):
            for t, o in zip(group, old):
                want = o.view(torch.uint8).clone()
                for a, b in todo:
                    if 0 <= a < pages and 0 <= b < pages:
                        want[b] = o.view(torch.uint8)[a]
                assert torch.equal(t.view(torch.uint8), want)
    P.copy_kv_pages(P.PageMoves(_ints(src), _ints(dst), None), [], [], [], [])
    # the layers in one tensor each
    whole = [torch.stack([t.view(torch.uint8) for t in group]).view(group[0].dtype) for group in (k, v, *s)]
    moves = P.PageMoves(_ints([1, 0]), _ints([3, 2]), None)
    P.copy_kv_pages(moves, *whole)
    P.copy_kv_pages(moves, tuple(k), v, *s)
    for t, group in zip(whole, (k, v, *s)):
        assert torch.equal(t.view(torch.uint8), torch.stack([x.view(torch.uint8) for x in group]))
        assert torch.equal(t.view(torch.uint8)[:, 3], t.view(torch.uint8)[:, 1])
    with pytest.raises(AssertionError):
        P.copy_kv_pages(P.PageMoves(_ints(src), _ints(dst), None), k, v, s[0], s[1][:-1])
    with pytest.raises(AssertionError):
        P.copy_kv_pages(P.PageMoves(_ints(src), _ints(dst[:-1]), None), k, v, *s)
    if layers > 1:
        with pytest.raises(AssertionError):
            P.copy_kv_pages(P.PageMoves(_ints(src), _ints(dst), None), [k[0], k[1][1:]] + k[2:], v, *s)


@gpu
@pytest.mark.parametrize("R,ps,longest,least", [(1, 16, 100, 16), (7, 16, 400, 16), (33, 32, 9000, 100), (300, 16, 20000, 256),
                                                (4096, 64, 700, 64)])
def test_shared_prefixes(R, ps, longest, least):
    rng = random.Random(R + least)
    for mode in range(4):
        width = -(-longest // ps) + 1
        family = [[rng.randint(0, 1 << 20) for _ in range(width)] for _ in range(max(1, R // 6))]
        tables, lens, new, f, row = [], [], [], 0, None
        for r in range(R):
            if row is None or rng.random() < 0.15:
                f = rng.randrange(len(family))
            at = rng.choice([0, width, rng.randint(0, width), rng.randint(0, width)])
            row = family[f][:at] + [rng.randint(-1, 1 << 20) for _ in range(width - at)]
            if rng.random() < 0.1:
                row[rng.randrange(width)] = -1
            tables.append(row)
            lens.append(rng.choice([0, -1]) if mode == 2 and rng.random() < 0.4 else rng.randint(1, longest + ps))
            new.append(rng.randint(0, 9) if mode == 3 else 1)
        starts = None if mode in (0, 2) else np.concatenate([[0], np.cumsum(new)]).tolist()
        got = P.shared_prefixes(_ints(tables).view(R, width), _ints(lens), _ints(starts) if starts else None, ps, least=least)
        want = O.runs(tables, lens, starts, ps, least)
        assert got.starts.tolist() == want[0] and got.lens.tolist() == want[1] and got.runs.tolist() == want[2]
    none = P.shared_prefixes(_ints([[1]]).view(1, 1)[:0], _ints([1])[:0], None, 16)
    assert none.starts.tolist() == [0] and none.lens.numel() == 0


# --- attention -------------------------------------------------------------------------------

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _case(code, dtype, H, KV, D, ps, runs, seed=0, extra=2, share=True):
    """runs: per run (shared tokens in whole pages, [(tokens behind, new tokens), ..]). The tables are as wide as
    it takes for the call to read shared pages once (by its bounds: 2048 keys, 2^27 bytes of all requests)."""
    rng = np.random.default_rng(seed)
    lens, new, rows, at = [], [], [], 0
    for pages, members in runs:
        first = list(range(at, at + pages))
        at += pages
        for behind, n in members:
            lens.append(pages * ps + behind + n if n or behind >= 0 else 0)
            new.append(n)
            own = -(-max(lens[-1], 0) // ps) - pages if lens[-1] > 0 else 0
            rows.append((first if lens[-1] > 0 else []) + list(range(at, at + max(own, 0))))
            at += max(own, 0)
    c = S.Cache(at + 3, KV, ps, D, code)
    c.fill(rng)
    name = rng.permutation(at + 3)
    wide = -(-max(2048, (1 << 27) // (len(lens) * KV * 2 * D) + 1) // ps) if share else 0
    width = max(max(map(len, rows)) + extra, wide)
    tables = rng.integers(0, at + 3, (len(lens), width)).astype(np.int32)
    for r, row in enumerate(rows):
        tables[r, :len(row)] = name[row]
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), H, D)) * 2.0).to(dtype)
    return c, tables, lens, starts, q


def _run(case, least=1, decode=None, shared=True, **kw):
    c, tables, lens, starts, q = case
    k, v, ks, vs = c.tensors(DEV)
    new = np.diff(starts)
    if decode is None:
        decode = bool((new == 1).all())
    t, n = torch.from_numpy(tables).to(DEV), _ints(lens)
    s = None if decode else torch.from_numpy(starts).to(DEV)
    runs = P.shared_prefixes(t, n, s, c.ps, least=least) if shared is True else shared
    kw.setdefault("max_q_len", int(max(new)))
    return P.paged_attention(q.to(DEV), k, v, ks, vs, t, n, s, scale=1 / q.shape[-1] ** 0.5, shared=runs, **kw), runs


def _check(got, case, dtype, **kw):
    """Half a step of the type, and of the probabilities, which the kernels hold in fp16 from scores whose
    fp32 sums are off by less than 2^-13, twice for numerator and sum, as without sharing; the joins'
    fp32 roundings are 2^-13 of those."""
    c, tables, lens, starts, q = case
    o, weight = S.attention(q.double().numpy(), c.values(0), c.values(1), tables, lens, starts, c.ps,
                            1 / q.shape[-1] ** 0.5, **kw)
    err = np.abs(got.double().cpu().numpy() - o)
    tol = HALF[dtype] * np.abs(o) + (2.0 ** -11 + 2.0 ** -12) * 1.001 * weight + 2.0 ** -25
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} off, at most {err.max():.3e} at {np.argwhere(err > tol)[0]}"


HEADS = [(1, 1, 64, 16), (4, 1, 128, 64), (32, 8, 128, 64), (7, 1, 128, 128), (8, 8, 64, 32), (14, 2, 64, 256),
         (16, 1, 128, 16), (40, 2, 128, 64), (64, 1, 64, 32)]


@gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D,ps", HEADS)
def test_single_tokens_of_shared_pages(code, dtype, H, KV, D, ps):
    """Runs of two to many requests, of one page and of several, requests of their own among them."""
    p = max(1, 300 // ps)
    case = _case(code, dtype, H, KV, D, ps, [(p, [(0, 1), (5, 1), (ps, 1)]), (0, [(40, 1)]), (2 * p + 1, [(ps - 1, 1), (70, 1)]),
                                             (1, [(i, 1) for i in range(21)]), (0, [(0, 1)])], seed=H + D + ps)
    got, runs = _run(case)
    want = [0, 3, 4, 6, 27]
    assert runs.starts.tolist()[:5] == want and runs.lens.tolist()[0] == p * ps
    _check(got, case, dtype)
    assert torch.equal(_run(case)[0], got)


@gpu
@pytest.mark.parametrize("H,KV,D,ps,shared,members", [(32, 8, 128, 64, 70, 40), (28, 4, 128, 128, 9, 70),
                                                      (16, 2, 64, 16, 500, 33), (4, 4, 64, 16, 129, 300),
                                                      (8, 2, 128, 64, 41, 11), (32, 2, 64, 16, 300, 3),
                                                      (8, 2, 128, 64, 33, 4)])
def test_long_prefixes_in_several_ranges(H, KV, D, ps, shared, members):
    code, dtype = (CODES[0], torch.float16) if H == 32 else (CODES[1], torch.bfloat16)
    case = _case(code, dtype, H, KV, D, ps, [(shared, [(i % 7 * 20, 1) for i in range(members)]), (3, [(9, 1), (0, 1)])])
    got, runs = _run(case)
    assert runs.lens.tolist()[:members] == [shared * ps] * members
    few = list(range(0, members, max(1, members // 6))) + [members, members + 1]
    c, tables, lens, _, q = case
    sub = (c, tables[few], [lens[i] for i in few], np.arange(len(few) + 1).astype(np.int32), q[few])
    _check(got[few], sub, dtype)
    plain = _run(case, shared=None)[0]
    weight = np.abs(c.values(1)).max()
    err = (got.double() - plain.double()).abs().cpu().numpy()
    assert (err <= 2 * HALF[dtype] * np.abs(plain.double().cpu().numpy()) + 2 * (2.0 ** -11 + 2.0 ** -12) * weight).all()


@gpu
@pytest.mark.parametrize("H,KV,D", [(8, 2, 128), (8, 1, 64), (16, 8, 64)])
def test_several_tokens_a_request(H, KV, D):
    """Ragged new tokens, some of none; a run's rows are those of all its members."""
    new = [3, 1, 0, 7, 5, 8, 2, 0, 1, 6, 8, 8, 1, 4]
    runs = [(20, [(i, n) for i, n in enumerate(new)]), (0, [(0, 8), (90, 1)]), (6, [(31, 2), (0, 8), (1, 1)])]
    for code, dtype in ((CODES[0], torch.bfloat16), (CODES[1], torch.float16)):
        case = _case(code, dtype, H, KV, D, 32, runs, seed=H)
        got, found = _run(case)
        assert found.starts.tolist()[:4] == [0, 14, 15, 16]
        _check(got, case, dtype)


@gpu
def test_finished_requests_in_the_middle_and_rows_behind_the_last():
    """Requests without tokens and keys interrupt no run; rows behind the last request stay."""
    case = _case(CODES[0], torch.float16, 4, 2, 64, 16, [(9, [(-1, 0), (3, 2), (-1, 0), (20, 1), (-1, 0), (0, 3), (-1, 0)])])
    c, tables, lens, starts, q = case
    assert lens.count(0) == 4
    wide = torch.cat([q, torch.full((3, 4, 64), float("nan"), dtype=q.dtype)])
    out = torch.full((9, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    got, runs = _run((c, tables, lens, starts, wide), out=out, max_q_len=3)
    assert got is out and (out[6:] == 7).all() and runs.starts.tolist()[:2] == [1, 7]
    assert runs.lens.tolist() == [0, 144, 0, 144, 0, 144, 0]
    _check(out[:6], case, torch.float16)
    # the same in strides of another layout
    view = torch.full((9, 8, 72), 3.0, dtype=torch.float16)[:, ::2, :64]
    view[:6] = q
    c2 = _run((c, tables, lens, starts, view), max_q_len=3)[0]
    assert torch.equal(c2[:6], out[:6])


@gpu
@pytest.mark.parametrize("max_kv", [0, 5, 64, 150, 2048, 2099, 2304, 2310, 2400])
def test_keys_past_the_bound_are_left_out(max_kv):
    """A bound inside of the shared pages, at their end and behind it."""
    case = _case(CODES[0], torch.float16, 8, 8, 64, 256, [(9, [(i, 1) for i in range(65)])])
    _check(_run(case, max_kv_len=max_kv)[0], case, torch.float16, max_kv=max_kv)


@gpu
def test_calls_that_do_not_share():
    """A window, requests of many rows, one request, few bytes: the same values as without runs, bit for bit."""
    case = _case(CODES[0], torch.float16, 8, 1, 64, 16, [(9, [(3, 1), (5, 1), (0, 1)])], share=False)
    assert torch.equal(_run(case)[0], _run(case, shared=None)[0])
    case = _case(CODES[0], torch.float16, 8, 1, 64, 16, [(9, [(3, 9), (5, 1), (0, 4)])])
    assert torch.equal(_run(case)[0], _run(case, shared=None)[0])       # 72 rows
    case = _case(CODES[0], torch.float16, 8, 1, 64, 16, [(9, [(3, 1), (5, 1), (0, 1)])])
    assert torch.equal(_run(case, window=30)[0], _run(case, shared=None, window=30)[0])
    _check(_run(case, window=30)[0], case, torch.float16, window=30)
    alone = _case(CODES[0], torch.float16, 8, 1, 64, 16, [(9, [(3, 1)])])
    assert torch.equal(_run(alone)[0], _run(alone, shared=None)[0])


@gpu
def test_requests_that_share_nothing_are_as_without_runs():
    """Nothing is joined: the bits of the call without runs (few rows are dealt as there)."""
    case = _case(CODES[1], torch.bfloat16, 8, 2, 128, 32, [(0, [(n, 1)]) for n in (5, 700, 64, 33, 1200)])
    got, runs = _run(case)
    assert runs.lens.tolist() == [0] * 5 and torch.equal(got, _run(case, shared=None)[0])


@gpu
def test_runs_of_another_batch_stay_inside_the_buffers():
    """Runs and lengths that no batch has lead nowhere else: what is read and written is this
    call's (requests whose members' rows are right have right results)."""
    case = _case(CODES[0], torch.float16, 4, 2, 64, 16, [(9, [(3, 1), (20, 1)]), (0, [(50, 1)])])
    def runs(lens, *rows):
        return P.SharedPrefixes(_ints([0] * 4), _ints(lens), _ints(list(rows) + [[0] * 4] * (3 - len(rows))))

    right, found = _run(case)
    assert found.runs.tolist() == [[0, 0, 2, 144], [0] * 4, [0] * 4]
    assert torch.equal(_run(case, shared=runs([144, 144, 0], [0, 0, 2, 144]))[0], right)
    big = (1 << 31) - 1
    strange = ([-5, 0, 2, 144], [3, 0, 2, 144], [0, -1, 2, 144], [0, 0, 4, 144], [0, 3, 1, 144], [0, 1, big, 144],
               [big, big, big, big], [0, 0, -2, 144], [0, 0, 2, -9], [2, 2, 1, big])
    for lens in ([0, 0, 0], [-8, -8, 1 << 30]):
        for row in strange:
            out = torch.full((3, 4, 64), 7.0, dtype=torch.float16, device=DEV)
            _check(_run(case, shared=runs(lens, row), out=out)[0], case, torch.float16)
    # positions that are said to be shared, of no such run: those requests' rows mean nothing, the others' are right
    for row in strange + ([2, 2, 1, 48], [1, 1, 1, 144]):
        assert torch.equal(_run(case, shared=runs([144, 144, 0], row))[0][2], right[2])


@gpu
@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_a_page_that_is_not_finite(bad, which, where):
    """What sees it is NaN, its head of all queries of the run or of its own request; the rest is right."""
    for members in (3, 40):
        case = _case(CODES[0], torch.float16, 4, 2, 64, 16, [(9, [(40, 1)] * members), (2, [(7, 1), (9, 1)])])
        c, tables, lens, starts, q = case
        clean = _run(case)[0]
        page = int(tables[1, 4 if where == "shared" else 10])
        c.scales[which][page, 1] = bad
        got = _run(case)[0]
        hit = torch.zeros(members + 2, 4, dtype=torch.bool, device=DEV)
        hit[:members, 2:] = where == "shared"
        hit[1, 2:] = True
        assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


@gpu
def test_what_lies_behind_a_request_leaves_no_trace():
    """NaN codes and scales in the pages behind a request's last one, NaN codes behind its last token."""
    case = _case(CODES[1], torch.float16, 4, 1, 128, 32, [(5, [(3, 1), (40, 1), (0, 1)])], extra=4)
    c, tables, lens, starts, q = case
    clean = _run(case)[0]
    used = set()
    for r, n in enumerate(lens):
        used |= {int(p) for p in tables[r, :-(-n // 32)]}
        if n % 32:
            for i in range(2):
                c.codes[i][tables[r, n // 32], :, n % 32:] = 0x7F
    for page in set(range(c.codes[0].shape[0])) - used:
        for i in range(2):
            c.codes[i][page] = 0xFF
            c.scales[i][page] = np.nan
    assert torch.equal(_run(case)[0], clean)


@gpu
@pytest.mark.parametrize("large", ["shared", "own"])
def test_scores_far_apart_between_the_parts(large):
    """One part's scores above all of the other's by more than fp16's range: it alone remains."""
    case = _case(CODES[0], torch.float16, 4, 1, 64, 16, [(6, [(30, 1)] * 5)])
    c, tables, lens, starts, q = case
    pages = tables[0, :6] if large == "shared" else np.unique(tables[:, 6:8])
    for p in pages:
        c.scales[0][p] *= 40
    _check_peaked(_run(case)[0], case)


def _check_peaked(got, case):
    """Scores up to 40 times as large: the fp32 sums' errors grow with them (2^-13 40 < 2^-7), and the probabilities'
    relative errors with those, twice."""
    c, tables, lens, starts, q = case
    o, weight = S.attention(q.double().numpy(), c.values(0), c.values(1), tables, lens, starts, c.ps, 1 / 8)
    err = np.abs(got.double().cpu().numpy() - o)
    assert (err <= 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2.0 ** -6) * weight + 2.0 ** -25).all()


@gpu
def test_many_requests_and_runs():
    """More requests than lanes, runs of all sizes, short and long."""
    rng = random.Random(5)
    runs = [(rng.choice([0, 1, 5, 30]), [(rng.randint(0, 60), 1) for _ in range(rng.choice([1, 2, 3, 25]))]) for _ in range(60)]
    case = _case(CODES[1], torch.float16, 4, 2, 64, 16, runs)
    got, found = _run(case, least=32)
    assert max(found.lens.tolist()) == 480
    _check(got, case, torch.float16)


@gpu
@pytest.mark.parametrize("H,KV,D,runs,members", [(8, 8, 64, 40, 20), (16, 8, 64, 35, 35), (16, 16, 128, 20, 20)])
def test_more_runs_than_workgroups(H, KV, D, runs, members):
    """Runs that fill the CUs unsplit, of up to 64 rows and of more: one part a row, or one a half."""
    rng = random.Random(runs)
    case = _case(CODES[0], torch.float16, H, KV, D, 16, [(rng.randint(2, 9), [(rng.randint(0, 20), 1) for _ in range(members)])
                                                        for _ in range(runs)])
    got, found = _run(case)
    assert found.starts.tolist()[:runs + 1] == [members * i for i in range(runs + 1)]
    c, tables, lens, _, q = case
    few = sorted(rng.sample(range(len(lens)), 60))
    _check(got[few], (c, tables[few], [lens[i] for i in few], np.arange(61).astype(np.int32), q[few]), torch.float16)
    plain = _run(case, shared=None)[0]
    weight = np.abs(c.values(1)).max()
    err = (got.double() - plain.double()).abs().cpu().numpy()
    tol = 2 * HALF[torch.float16] * np.abs(plain.double().cpu().numpy()) + 2 * (2.0 ** -11 + 2.0 ** -12) * weight
    assert (err <= tol).all() and not torch.equal(got, plain)


@gpu
def test_more_than_the_parts_hold_is_done_without_them():
    """A call of too many requests x KV heads for parts: as without runs, not refused."""
    L = _lib.lib()
    R, KV = 1 << 18, 16
    args = (R, R, KV, KV, 64, 1, 4096, 0)
    assert L.pmi_paged_attention_shared_workspace_bytes(*args) == L.pmi_paged_attention_workspace_bytes(*args)
    assert L.pmi_paged_attention_shared_workspace_bytes(64, 64, 32, 8, 128, 1, 8192, 0) > \
        L.pmi_paged_attention_workspace_bytes(64, 64, 32, 8, 128, 1, 8192, 0)


@gpu
def test_pages_past_32_bits_of_bytes():
    """Copies, and shared pages, whose offsets pass 2^32 bytes."""
    pages, KV, ps, D = 17000, 8, 256, 128
    k = torch.zeros(pages, KV, ps, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(pages, KV, ps // 16, D, 16, dtype=torch.int8, device=DEV)
    ks, vs = torch.full((pages, KV), 0.01, device=DEV), torch.full((pages, KV), 0.01, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    top = pages - 1
    for t in (k, v):
        t[top - 8:] = torch.randint(-127, 128, t[top - 8:].shape, generator=g, device=DEV, dtype=torch.int8)
    P.copy_kv_pages(P.PageMoves(_ints([top, top - 8]), _ints([3, 16500]), None), [k], [v], [ks], [vs])
    for t in (k, v):
        assert torch.equal(t[3], t[top]) and torch.equal(t[16500], t[top - 8]) and not t[2].any() and not t[4].any()
    # 40 requests of eight pages at the end of the cache, and the same ones at its front
    rows = torch.arange(top - 8, top, dtype=torch.int32, device=DEV)
    wide = -(-max(2048, (1 << 27) // (40 * KV * 2 * D) + 1) // ps)
    q = torch.randn(40, 16, D, generator=g, device=DEV).half()
    out = []
    for at in (rows, rows - (top - 8) + 8):
        P.copy_kv_pages(P.PageMoves(rows, at.contiguous(), None), [k], [v], [ks], [vs])
        tables = torch.zeros(40, max(wide, 9), dtype=torch.int32, device=DEV)
        tables[:, :8] = at
        tables[:, 8] = torch.arange(100, 140, device=DEV)
        lens = torch.full((40,), 8 * ps + 5, dtype=torch.int32, device=DEV)
        shared = P.shared_prefixes(tables, lens, None, ps)
        assert shared.lens.tolist() == [8 * ps] * 40
        out.append(P.paged_attention(q, k, v, ks, vs, tables, lens, scale=0.01, shared=shared))
    assert torch.equal(*out) and out[0].any()


@gpu
def test_shared_attention_captured():
    """Lengths grow and a request ends between the replays; each equals the eager call."""
    case = _case(CODES[0], torch.float16, 8, 2, 128, 32, [(20, [(1, 1)] * 9), (3, [(0, 1)] * 2)], extra=6)
    c, tables, lens, starts, q = case
    k, v, ks, vs = c.tensors(DEV)
    t, n, x = torch.from_numpy(tables).to(DEV), _ints(lens), q.to(DEV)

    def step():
        runs = P.shared_prefixes(t, n, None, 32, least=64)
        return P.paged_attention(x, k, v, ks, vs, t, n, scale=0.1, shared=runs)

    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    torch.cuda.current_stream().wait_stream(s)
    last = None
    for i in range(5):
        n += 3
        if i == 2:
            n[4] = 0
        x.normal_()
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (last is None or not torch.equal(want, last))
        last = want.clone()


@gpu
def test_python_checks():
    case = _case(CODES[0], torch.float16, 4, 2, 64, 16, [(9, [(3, 1), (20, 1)])])
    starts = _ints([0, 2, 2])
    for lens, runs in ((_ints([0]), _ints([[0] * 4] * 2)), (_ints([0, 0]), _ints([[0] * 4])),
                       (_ints([0, 0]), _ints([[0] * 4] * 2).long()), (_ints([0, 0]).long(), _ints([[0] * 4] * 2))):
        with pytest.raises(AssertionError):
            _run(case, shared=P.SharedPrefixes(starts, lens, runs))
    with pytest.raises(RuntimeError):
        _run(case, shared=P.SharedPrefixes(starts, _ints([0, 0]), _ints([[0] * 4] * 2).cpu()))
    t = _ints([[1, 2], [3, 4]]).view(2, 2)
    two, four, free = _ints([0, 0]), _ints([0, 5, 0, 0]), _ints([0] * 5)
    for bad in (lambda: P.fork_block_tables(t, two, two.long(), free, four, free, 16),
                lambda: P.fork_block_tables(t, two, two[:1], free, four, free, 16),
                lambda: P.fork_block_tables(t, two, two, free, four, free[:4], 16),
                lambda: P.fork_block_tables(t, two, two, free, free, free, 16),
                lambda: P.fork_block_tables(t, two, two, free, four, free, 16, lengths=two[:1]),
                lambda: P.fork_block_tables(t.t(), two, two, free, four, free, 16),
                lambda: P.release_block_tables(t, two, two.bool(), free, four, 16, shares=two),
                lambda: P.compact_block_tables(t, two, free, four, two, 16),
                lambda: P.shared_prefixes(t, two, two, 16),
                lambda: P.shared_prefixes(t, two, None, 16, least=0)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(_lib.PmiError):
        P.fork_block_tables(t, two, two, free, four, free, 24)
    with pytest.raises(RuntimeError):
        P.PagedKVCache(1, 2, 64, 1, 64, DEV).fork(two)


def test_runs_in_other_strides_are_refused(monkeypatch):
    """Their address is handed over as that of R rows of 4: rows that lie apart, or one that stands for all, would be
    read as others, and past their memory. (Checks come before anything of the device's.)"""
    monkeypatch.setattr(P.paged, "_hip", lambda t, fn: t.device)
    k, s = torch.zeros(4, 1, 16, 64, dtype=torch.int8), torch.zeros(4, 1)
    args = (torch.zeros(3, 1, 64, dtype=torch.float16), k, k.view(4, 1, 1, 64, 16), s, s,
            torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    rows = torch.zeros(3, 8, dtype=torch.int32)
    for runs in (rows[:, :4], rows[:1, :4].expand(3, 4), torch.zeros(4, 3, dtype=torch.int32).t()):
        shared = P.SharedPrefixes(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), runs)
        with pytest.raises(AssertionError, match="runs must be contiguous"):
            P.paged_attention(*args, scale=0.125, shared=shared)


@gpu
def test_runs_whose_row_tiles_pass_32_bits_stay_inside_the_buffers():
    """Runs that no batch has, each of all queries: 2^28 + 2 row tiles of 16 KV heads, 2^32 + 32 together, which are
    not the 32 that 32 bits say (16 ranges each would be written past the parts). No request is said to share anything:
    the bits are those without runs."""
    R, KV, H, D, ps = 100000, 16, 64, 64, 16
    g = torch.Generator(device=DEV).manual_seed(0)
    k = torch.randint(-127, 128, (4, KV, ps, D), generator=g, device=DEV, dtype=torch.int8)
    scale = torch.full((4, KV), 0.01, device=DEV)
    tables = torch.randint(0, 4, (R, 2048 // ps), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(1, 2 * ps, (R,), generator=g, device=DEV, dtype=torch.int32)
    q = torch.randn(R, H, D, generator=g, device=DEV).half()
    args = (q, k, k.view(4, KV, 1, D, 16), scale, scale, tables, lens)
    tiles = -(-R * (H // KV) // 128)
    n = 2 ** 28 // tiles
    runs = torch.zeros(R, 4, dtype=torch.int32, device=DEV)
    runs[:n, 2], runs[:n, 3] = R, ps
    last = 2 ** 28 + 2 - n * tiles
    runs[n, 2], runs[n, 3] = last * 128 // (H // KV), ps
    assert 0 < last <= tiles and n * tiles + last == 2 ** 28 + 2 and n < R
    sizes, L = (R, R, H, KV, D, 1, 2048, 0), _lib.lib()
    assert L.pmi_paged_attention_shared_workspace_bytes(*sizes) > L.pmi_paged_attention_workspace_bytes(*sizes)
    want = P.paged_attention(*args, scale=0.125)
    got = P.paged_attention(*args, scale=0.125, shared=P.SharedPrefixes(runs[:, 0], torch.zeros_like(lens), runs))
    assert torch.equal(got, want)
