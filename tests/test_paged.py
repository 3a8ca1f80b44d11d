"""The paged 8-bit cache against plain implementations (oracle/serving_oracle.py): block
tables and slots, the write with RoPE, the read, attention, refusals, capture."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
import torch

import pare_amd as P
from oracle import serving_oracle as S
from pare_amd import _lib

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
CODES = [torch.int8, torch.float8_e4m3fn]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# --- the oracle itself (CPU) ---------------------------------------------------------

def test_oracle_append_error_is_half_a_code():
    """Values written in one run are within half a code of what they were."""
    rng = np.random.default_rng(0)
    for dtype in CODES:
        c = S.Cache(2, 1, 16, 64, dtype)
        x = rng.standard_normal((16, 3 * 64)).astype(np.float32)
        ones, zeros = np.ones((16, 32), np.float32), np.zeros((16, 32), np.float32)
        c.append(x, ones, zeros, np.arange(16), np.arange(16, 32), 1)
        for i in range(2):
            want = x[:, 64 * (1 + i):64 * (2 + i)]
            scale = c.scales[i][1, 0]
            step = 1.0 if dtype == torch.int8 else np.maximum(np.abs(want) / scale * 2 ** -3, 2.0 ** -9)
            assert (np.abs(c.values(i)[1, 0] - want) <= 0.5001 * scale * step).all()


def test_oracle_tables_by_hand():
    t, starts, lens, first, pos, slots, pool = S.extend_tables(
        [[7, -1], [-1, -1], [3, -1]], [15, 0, 3], [2, 17, 1], [0, 1, 2], [2, 2, 0, 0], 16, 22)
    assert t == [[7, 2], [-1, -1], [3, -1]]     # request 1 needs two pages, one is left
    assert (starts, lens, first) == ([0, 2, 19, 20], [17, 0, 4], [15, -1, 3])
    # pages 7 and 3 are not of a cache of three pages
    assert slots == [-1, 32] + [-1] * 20 and pool == [0, 1, 1, 0]
    assert pos[:2] == [15, 16] and pos[19] == 3
    t, starts, lens, first, pos, slots, pool = S.extend_tables(
        [[7, -1], [-1, -1], [3, -1]], [15, 0, 3], [2, 17, 1], [0, 1, 2, 9, 9, 9, 9, 9], [1, 2, 0, 0], 16, 22)
    assert slots == [7 * 16 + 15, 16] + [-1] * 17 + [51, -1, -1] and pool == [2, 1, 1, 0]


# --- refusals of the C ABI (CPU) -----------------------------------------------------

P8 = 0x1000  # a 16-byte aligned address that is never read: validation comes first


def _append_args(**kw):
    a = dict(qkv=P8, dtype=_lib.PMI_F16, stride=6 * 128, cos=P8, sin=P8, L=8, positions=P8, slots=P8, q=P8, k=P8,
             v=P8, ks=P8, vs=P8, code=_lib.PMI_I8, pages=4, ps=16, T=2, H=4, KV=1, D=128)
    a.update(kw)
    return [*a.values(), None]


def _attention_args(**kw):
    a = dict(q=P8, dtype=_lib.PMI_F16, stride=512, head=128, k=P8, v=P8, ks=P8, vs=P8, code=_lib.PMI_I8, pages=4, ps=16,
             tables=P8, tstride=4, lens=P8, starts=P8, out=P8, T=2, R=1, width=4, H=4, KV=1, D=128, max_q=2,
             max_kv=64, window=0, scale=1.0, ws=P8, ws_bytes=1 << 40)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("change", [dict(dtype=_lib.PMI_F32), dict(code=_lib.PMI_U8), dict(ps=24), dict(ps=0),
                                    dict(ps=512), dict(D=96), dict(H=5, KV=2), dict(KV=0), dict(stride=760),
                                    dict(stride=772), dict(L=0), dict(T=-1), dict(T=1 << 31), dict(qkv=None),
                                    dict(k=None), dict(v=P8 + 8), dict(q=P8 + 2), dict(pages=-1),
                                    dict(pages=1 << 40), dict(slots=None), dict(L=1 << 40)])
def test_append_refuses(change):
    rc = _lib.lib().pmi_rope_append_kv(*_append_args(**change))
    assert rc in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED) and "pmi_rope_append_kv" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(dtype=_lib.PMI_F32), dict(code=_lib.PMI_F16), dict(ps=48), dict(D=80),
                                    dict(H=6, KV=4), dict(H=65, KV=1), dict(stride=513), dict(head=4), dict(T=-1),
                                    dict(R=-1), dict(width=5), dict(max_q=-1), dict(max_kv=-1), dict(window=-1),
                                    dict(starts=None), dict(T=1 << 40), dict(width=1 << 40, tstride=1 << 40),
                                    dict(max_kv=1 << 40), dict(q=None), dict(q=P8 + 8),
                                    dict(out=None), dict(lens=None), dict(tables=None), dict(k=None),
                                    dict(window=1 << 40), dict(R=1 << 40)])
def test_attention_refuses(change):
    rc = _lib.lib().pmi_paged_attention(*_attention_args(**change))
    assert rc in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED) and "pmi_paged_attention" in _lib.last_error()


def test_attention_without_its_workspace_is_refused():
    L = _lib.lib()
    need = L.pmi_paged_attention_workspace_bytes(2, 2, 4, 1, 128, 1, 100000, 0)
    if need:
        args = dict(starts=None, T=2, R=2, max_q=1, max_kv=100000, width=10000, tstride=10000)
        for bad in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=P8 + 16)):
            assert L.pmi_paged_attention(*_attention_args(**args, **bad)) == _lib.PMI_ERR_INVALID


@pytest.mark.parametrize("change", [dict(R=-1), dict(R=4097), dict(width=9), dict(ring=-1), dict(ps=8), dict(total=-1),
                                    dict(total=1 << 31), dict(width=1 << 40, stride=1 << 40), dict(ring=1 << 40),
                                    dict(tables=None), dict(pool=None), dict(slots=None), dict(free=None)])
def test_tables_refuse(change):
    a = dict(tables=P8, stride=8, lens=P8, new=P8, free=P8, pool=P8, starts=P8, out=P8, first=P8, fresh=P8, positions=P8,
             slots=P8, pool_out=P8, R=2, width=8, ring=16, ps=16, total=2)
    a.update(change)
    rc = _lib.lib().pmi_extend_block_tables(*a.values(), None)
    assert rc in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED)
    if not {"total", "slots"} & set(change):
        a = dict(tables=P8, stride=8, lens=P8, done=P8, free=P8, pool=P8, R=2, width=8, ring=16, ps=16)
        a.update(change)
        rc = _lib.lib().pmi_release_block_tables(*a.values(), None)
        assert rc in (_lib.PMI_ERR_INVALID, _lib.PMI_ERR_UNSUPPORTED)


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert L.pmi_rope_append_kv(*_append_args(T=0, qkv=None)) == _lib.PMI_OK
    assert L.pmi_paged_attention(*_attention_args(T=0)) == _lib.PMI_OK
    assert L.pmi_paged_attention(*_attention_args(max_q=0)) == _lib.PMI_OK
    assert L.pmi_read_kv_pages(None, P8, P8, P8, P8, _lib.PMI_I8, 4, 16, None, None, _lib.PMI_F16, 0, 1, 64,
                               None) == _lib.PMI_OK
    assert L.pmi_release_block_tables(P8, 8, P8, P8, P8, P8, 0, 8, 16, 16, None) == _lib.PMI_OK
    assert L.pmi_read_kv_pages(P8, P8, P8, P8, P8, _lib.PMI_I8, 4, 16, P8, P8, _lib.PMI_U8, 1, 1, 64,
                               None) == _lib.PMI_ERR_INVALID


def test_cpu_tensors_raise():
    i = torch.zeros(1, dtype=torch.int32)
    k, v, s = torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1, 1, 64, 16, dtype=torch.int8), torch.zeros(1, 1)
    with pytest.raises(RuntimeError, match="HIP"):
        P.paged_attention(torch.zeros(1, 1, 64).half(), k, v, s, s, i[None], i, scale=1.0)
    with pytest.raises(RuntimeError, match="HIP"):
        P.rope_append_kv(torch.zeros(1, 192).half(), s, s, i, i, k, v, s, s)
    with pytest.raises(RuntimeError, match="HIP"):
        P.read_kv_pages(i, k, v, s, s)
    with pytest.raises(RuntimeError, match="HIP"):
        P.extend_block_tables(i[None], i, i, i, torch.zeros(4, dtype=torch.int32), 16, 1)
    with pytest.raises(ValueError):
        P.PagedKVCache(1, 1, 16, 1, 64, "cpu", dtype=torch.float16)
    for args, kw in (((1, 1, 16, 1, 80, "cpu"), {}), ((1, 1, 16, 1, 64, "cpu"), dict(page_size=24)),
                     ((1, 1, 16, 1, 64, "cpu"), dict(page_size=512)), ((1, 0, 16, 1, 64, "cpu"), {}),
                     ((1, 1, 0, 1, 64, "cpu"), {}), ((1, 1, 16, 1, 64, "cpu"), dict(pages=0))):
        with pytest.raises(ValueError):
            P.PagedKVCache(*args, **kw)


# --- block tables --------------------------------------------------------------------

def _random_tables(rng, R, ps, longest, newest, spare, width=None):
    lens = [rng.choice([0, 1, ps - 1, ps, rng.randint(0, longest)]) for _ in range(R)]
    new = [rng.choice([0, 1, 1, rng.randint(0, newest)]) for _ in range(R)]
    held = [-(-n // ps) for n in lens]
    width = width or max([-(-(a + b) // ps) for a, b in zip(lens, new)] + [1])
    lens = [min(n, width * ps) for n in lens]
    held = [-(-n // ps) for n in lens]
    need = sum(-(-(a + b) // ps) - h for a, b, h in zip(lens, new, held))
    pages = sum(held) + max(0, need + spare)
    order = rng.sample(range(pages), pages)
    tables, at = [[-1] * width for _ in range(R)], 0
    for r, h in enumerate(held):
        tables[r][:h] = order[at:at + h]
        at += h
    ring = max(pages, 1)
    free, head = [0] * ring, rng.randrange(ring)
    for i, page in enumerate(order[at:]):
        free[(head + i) % ring] = page
    return tables, lens, new, free, [head, pages - at, 3, 0]


@gpu
@pytest.mark.parametrize("R,ps,longest,newest,spare,width", [
    (1, 16, 0, 1, 0, None), (1, 64, 500, 300, 0, None), (48, 64, 4000, 3, 5, None), (70, 16, 200, 90, 4, None),
    (70, 16, 200, 90, -20, None), (33, 32, 400, 900, -50, 12), (1025, 16, 40, 5, 0, None),
    (4096, 128, 3000, 2, -7, None), (300, 256, 1000, 700, 9, None)])
def test_extend_block_tables(R, ps, longest, newest, spare, width):
    """Every output against the oracle's integers: pools that are too small, rows that are
    too short, more tokens than one workgroup looks up, tokens behind the last request."""
    rng = random.Random(R * ps + newest)
    tables, lens, new, free, pool = _random_tables(rng, R, ps, longest, newest, spare, width)
    total = sum(new) + rng.randint(0, 5)
    want = S.extend_tables(tables, lens, new, free, pool, ps, total)
    wide = torch.full((R, len(tables[0]) + 3), -9, dtype=torch.int32, device=DEV)  # rows of a larger table
    t = wide[:, :len(tables[0])]
    t.copy_(_ints(tables))
    args = (_ints(lens), _ints(new), _ints(free), _ints(pool))
    plan = P.extend_block_tables(t, *args, ps, total)
    got = (t, plan.q_starts, plan.kv_lens, plan.first, plan.positions, plan.slots, plan.pool)
    for name, g, w in zip(("tables", "q_starts", "kv_lens", "first", "positions", "slots", "pool"), got, want):
        assert g.tolist() == w, name
    assert (wide[:, len(tables[0]):] == -9).all()
    assert args[0].tolist() == lens and args[3].tolist() == pool
    # in place
    t.copy_(_ints(tables))
    again = P.extend_block_tables(t, *args, ps, total, kv_lens_out=args[0], pool_out=args[3])
    assert args[0].tolist() == want[2] and args[3].tolist() == want[6]
    assert again.slots.tolist() == want[5] and t.tolist() == want[0]


@gpu
def test_extend_with_negative_lengths_and_strange_pools():
    """Lengths below zero count as zero; a head or count that no pool has, and table
    entries outside the cache, lead to no slot outside it."""
    t = _ints([[5, -1, 99], [-1, -1, -1]])
    plan = P.extend_block_tables(t, _ints([-4, 3]), _ints([2, -1]), _ints([1, 0, 2]), _ints([77, 50, 0, 0]), 16, 2)
    assert plan.q_starts.tolist() == [0, 2, 2] and plan.slots.tolist() == [16, 17]
    plan = P.extend_block_tables(t, _ints([33, 0]), _ints([1, 0]), _ints([1, 0, 2]), _ints([0, 3, 0, 0]), 16, 1)
    assert plan.slots.tolist() == [-1]  # its page is 99
    none = P.extend_block_tables(t[:0], _ints([]), _ints([]), _ints([]), _ints([0, 0, 0, 0]), 16, 3)
    assert none.slots.tolist() == [-1] * 3 and none.q_starts.tolist() == [0]


@gpu
@pytest.mark.parametrize("R,ps", [(1, 16), (37, 32), (1500, 16)])
def test_extend_and_release_keep_every_page_once(R, ps):
    """Requests that grow, end and start again: no page is ever held twice, and every
    page is in a table or in the ring."""
    rng = random.Random(R)
    c = P.PagedKVCache(0, R, 40 * ps, 1, 64, DEV, page_size=ps, pages=R * 12)
    pages = R * 12
    for step in range(12):
        new = [rng.choice([0, 1, rng.randint(0, 4 * ps)]) for _ in range(R)]
        c.extend(_ints(new), sum(new))
        done = torch.tensor([rng.random() < 0.3 for _ in range(R)], device=DEV)
        held_before = c.kv_lens.tolist()
        c.release(done)
        lens, pool = c.kv_lens.tolist(), c.pool.tolist()
        assert lens == [0 if d else n for n, d in zip(held_before, done.tolist())]
        rows, free = c.block_tables.tolist(), c.free_pages.tolist()
        held = [p for row, n in zip(rows, lens) for p in row[:-(-n // ps)]]
        loose = [free[(pool[0] + i) % pages] for i in range(pool[1])]
        assert sorted(held + loose) == list(range(pages)), step


# --- the write and the read ----------------------------------------------------------

def _rope(L, D):
    inv = 1.0 / 10000.0 ** (np.arange(0, D, 2) / D)
    a = np.arange(L)[:, None] * inv
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _check_cache(c, k, v, ks, vs, where=""):
    np.testing.assert_array_equal(ks.cpu().numpy(), c.scales[0], err_msg="k_scale " + where)
    np.testing.assert_array_equal(vs.cpu().numpy(), c.scales[1], err_msg="v_scale " + where)
    np.testing.assert_array_equal(k.cpu().view(torch.uint8).numpy(), c.codes[0], err_msg="k codes " + where)
    np.testing.assert_array_equal(S.token_major(v), c.codes[1], err_msg="v codes " + where)


@gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D,ps", [(1, 1, 64, 16), (8, 2, 128, 64), (7, 1, 128, 32), (4, 4, 64, 128),
                                       (6, 3, 128, 256)])
def test_append_equals_the_oracle_bit_for_bit(code, dtype, H, KV, D, ps):
    """Prompts of odd lengths, then single tokens whose values grow (the pages' older
    codes are rounded again), then a mix; refused tokens and slots outside the cache are
    skipped. Scales and codes are one IEEE operation after another: equal bits."""
    rng = np.random.default_rng(H * D + ps)
    pages = 14
    c = S.Cache(pages, KV, ps, D, code)
    for i in range(2):  # old bytes nobody wrote
        c.codes[i][:] = rng.integers(0, 127, c.codes[i].shape)
        c.scales[i][:] = rng.uniform(0.5, 1, c.scales[i].shape)
    k, v, ks, vs = c.tensors(DEV)
    cos, sin = _rope(4 * ps, D)
    tcos, tsin = torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV)
    perm = rng.permutation(pages)
    rows = perm[:12].reshape(3, 4)
    lens = [0, 0, 0]
    steps = [[ps + 5, 3, 0], [1, 1, 1], [1, 1, 1], [1, 0, 1], [ps - 6, 2, 17 if ps > 16 else 9], [1, 1, 1]]
    for step, new in enumerate(steps):
        positions = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)] + [[0, 0]]).astype(np.int32)
        slots = np.concatenate([rows[r][np.arange(a, a + n) // ps] * ps + np.arange(a, a + n) % ps
                                for r, (a, n) in enumerate(zip(lens, new))] + [[-1, pages * ps]]).astype(np.int32)
        lens = [a + n for a, n in zip(lens, new)]
        x = torch.from_numpy(rng.standard_normal((len(slots), (H + 2 * KV) * D)) * (1 + step)).to(dtype)
        wide = torch.zeros(len(slots), (H + 2 * KV) * D + 8, dtype=dtype, device=DEV)
        wide[:, :-8] = x.to(DEV)
        q = P.rope_append_kv(wide[:, :-8], tcos, tsin, torch.from_numpy(positions).to(DEV),
                             torch.from_numpy(slots).to(DEV), k, v, ks, vs)
        want = c.append(x.float().numpy(), cos, sin, positions, slots, H)
        assert torch.equal(q.cpu(), torch.from_numpy(want).to(dtype)), step
        _check_cache(c, k, v, ks, vs, f"step {step}")
    some = torch.tensor([int(perm[0]), pages, -1, int(perm[5])], dtype=torch.int32, device=DEV)
    for out in (torch.float16, torch.bfloat16, torch.float32):
        rk, rv = P.read_kv_pages(some, k, v, ks, vs, dtype=out)
        for got, i in ((rk, 0), (rv, 1)):
            val = (S.decode(c.codes[i], code) * c.scales[i][..., None, None])[[perm[0], perm[5]]]
            assert torch.equal(got[[0, 3]].cpu(), torch.from_numpy(val).to(out))
            assert (got[[1, 2]] == 0).all()


@gpu
@pytest.mark.parametrize("code", CODES)
def test_append_against_64_bits(code):
    """Codes times scales against the rotation in 64 bits: half a code, and 2^-20 of the
    largest for the fp32 rotation and division (a few roundings of 2^-24 each)."""
    H, KV, D, ps, T = 4, 2, 128, 64, 150
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(T, (H + 2 * KV) * D, generator=g).half()
    cos, sin = _rope(T, D)
    c = P.PagedKVCache(1, 1, T, KV, D, DEV, page_size=ps, dtype=code)
    plan = c.extend(_ints([T]), T)
    q = c.append(0, qkv.to(DEV), torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV), plan)
    x = qkv.double().numpy().reshape(T, H + 2 * KV, D)
    turned = S.rotate(x[:, :H + KV], cos.astype(np.float64), sin.astype(np.float64))
    assert np.abs(q.cpu().double().numpy() - turned[:, :H]).max() <= np.abs(turned).max() * (2 ** -11 + 2 ** -20)
    k, v = P.read_kv_pages(c.block_tables[0], c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], dtype=torch.float32)
    for got, want in ((k, turned[:, H:]), (v, x[:, H + KV:])):
        got = got.transpose(1, 2).reshape(-1, KV, D)[:T].cpu().double().numpy()
        for page in range(-(-T // ps)):
            a, b = got[page * ps:(page + 1) * ps], want[page * ps:min(T, (page + 1) * ps)]
            top = np.abs(b).max((0, 2), keepdims=True)
            half = top / 254 if code == torch.int8 else np.maximum(np.abs(b) * 2.0 ** -4, top / 448 * 2.0 ** -10)
            assert (np.abs(a[:len(b)] - b) <= half + top * 2.0 ** -20).all()


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_append_shows_infinities_and_nan_in_their_page_and_head_only(bad):
    KV, D, ps = 2, 64, 16
    c = P.PagedKVCache(1, 1, 48, KV, D, DEV, page_size=ps)
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv = torch.randn(40, 4 * KV * D // 2 * 1 + KV * D, generator=g, device=DEV).half()
    H = qkv.shape[1] // D - 2 * KV
    qkv[20, (H + KV) * D + 5] = bad  # v of head 0, second page
    cos, sin = (torch.from_numpy(t).to(DEV) for t in _rope(48, D))
    plan = c.extend(_ints([40]), 40)
    c.append(0, qkv, cos, sin, plan)
    page = c.block_tables[0].long()
    finite = torch.isfinite(c.v_scale[0][page])
    assert finite.tolist() == [[True, True], [False, True], [True, True]]
    assert torch.isfinite(c.k_scale[0]).all()


# --- attention -------------------------------------------------------------------------

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _attention_case(code, dtype, H, KV, D, ps, lens, new, window=0, seed=0, width=None, spread=2.0):
    """Inputs on the device, and (o, weight) in 64 bits."""
    rng = np.random.default_rng(seed)
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + 3
    c = S.Cache(pages, KV, ps, D, code)
    c.fill(rng)
    order = rng.permutation(pages)
    width = width or max(need + [1]) + 1
    tables = rng.integers(0, pages, (len(lens), width)).astype(np.int32)  # entries past a request's end: any page
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = order[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), H, D)) * spread).to(dtype)
    return c, tables, starts, q


def _tolerance(o, weight, dtype):
    """Half a step of the output's type, and of the probabilities': the kernels hold them
    in fp16 (2^-11), from scores whose fp32 sums over at most 128 products are off by less
    than 2^-13 here (|q| |k| scale sums to 14, times 130 2^-24), twice for numerator and sum."""
    return HALF[dtype] * np.abs(o) + (2.0 ** -11 + 2.0 ** -12) * weight + 2.0 ** -25


def _check(got, o, weight, dtype, what=""):
    err = np.abs(got.double().cpu().numpy() - o)
    bad = err > _tolerance(o, weight, dtype)
    assert not bad.any(), f"{what} {bad.sum()} of {bad.size} off, at most {err.max():.3e} at {np.argwhere(bad)[0]}"


def _run(c, tables, lens, starts, q, window=0, decode=None, **kw):
    k, v, ks, vs = c.tensors(DEV)
    new = np.diff(starts)
    if decode is None:
        decode = bool((new == 1).all())
    return P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                             None if decode else torch.from_numpy(starts).to(DEV), scale=1 / q.shape[-1] ** 0.5,
                             window=window, max_q_len=int(max(new)), **kw)


def _oracle(c, tables, lens, starts, q, window=0):
    return S.attention(q.double().numpy(), c.values(0), c.values(1), tables, lens, starts, c.ps,
                       1 / q.shape[-1] ** 0.5, window)


HEADS = [(1, 1, 64, 16), (4, 1, 128, 64), (32, 8, 128, 64), (7, 1, 128, 128), (8, 8, 64, 32), (14, 2, 64, 256),
         (16, 1, 128, 16), (40, 2, 128, 64), (64, 1, 64, 32)]


@gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D,ps", HEADS)
def test_decode_attention(code, dtype, H, KV, D, ps):
    """One token for each of a ragged batch: lengths of one, around a page, a tile and a
    split, and a request of length zero (whose row is zeros)."""
    lens = [1, 2, ps - 1, ps, ps + 1, 63, 64, 65, 255, 257, 0, 700]
    case = _attention_case(code, dtype, H, KV, D, ps, lens, [1] * len(lens), seed=H + D + ps)
    got = _run(case[0], case[1], lens, case[2], case[3])
    _check(got, *_oracle(case[0], case[1], lens, case[2], case[3]), dtype)
    assert (got[10] == 0).all()
    # the same with the starts given
    assert torch.equal(got, _run(case[0], case[1], lens, case[2], case[3], decode=False))


@gpu
@pytest.mark.parametrize("lens", [[5000], [20000, 3], [1023, 4097, 2048, 9001]])
def test_decode_attention_of_long_contexts(lens):
    """Several splits of one sequence, joined; bit-identical when repeated."""
    for code, dtype in ((CODES[0], torch.float16), (CODES[1], torch.bfloat16)):
        case = _attention_case(code, dtype, 8, 2, 128, 64, lens, [1] * len(lens), seed=sum(lens))
        got = _run(case[0], case[1], lens, case[2], case[3])
        _check(got, *_oracle(case[0], case[1], lens, case[2], case[3]), dtype)
        assert torch.equal(got, _run(case[0], case[1], lens, case[2], case[3]))


@gpu
@pytest.mark.parametrize("KV,D,lens", [(64, 64, [40000]), (64, 64, [33000]), (64, 64, [3000, 200, 9000]), (32, 128, [16000]),
                                       (16, 128, [64, 65, 4000] * 4), (2, 128, [8200] * 7), (1, 64, [70000, 1]),
                                       (8, 128, [500] * 130), (2, 64, [129] * 1100), (16, 128, [9000])])
def test_decode_attention_at_every_cut(KV, D, lens):
    """Numbers of tiles on both sides of every way to deal them out (pages used many times)."""
    rng = np.random.default_rng(len(lens) * KV)
    c = S.Cache(5, KV, 256, D, CODES[0])
    c.fill(rng)
    tables = rng.integers(0, 5, (len(lens), -(-max(lens) // 256))).astype(np.int32)
    starts = np.arange(len(lens) + 1).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((len(lens), KV, D))).half()
    few = sorted({0, 1, len(lens) // 2, len(lens) - 1} & set(range(len(lens))))  # (the oracle is slow)
    got = _run(c, tables, lens, starts, q)
    want = _oracle(c, tables[few], [lens[i] for i in few], np.arange(len(few) + 1), q[few])
    _check(got[few], *want, torch.float16)
    again = _run(c, tables, lens, starts, q)
    assert torch.equal(got, again)
    # the requests that the oracle skipped: the same keys one by one
    for i in range(0, len(lens), max(1, len(lens) // 8)):
        alone = _run(c, tables[i:i + 1], lens[i:i + 1], starts[:2], q[i:i + 1])
        err = (got[i].double() - alone[0].double()).abs().cpu().numpy()
        weight = np.abs(c.values(1)).max()
        assert (err <= 2 * _tolerance(alone[0].double().cpu().numpy(), weight, torch.float16)).all()


@gpu
@pytest.mark.parametrize("window", [1, 16, 63, 64, 65, 300, 5000])
def test_windows(window):
    lens = [1, 64, 130, 700, 0, 2000]
    case = _attention_case(CODES[0], torch.float16, 8, 2, 128, 32, lens, [1] * len(lens), seed=window)
    _check(_run(case[0], case[1], lens, case[2], case[3], window=window),
           *_oracle(case[0], case[1], lens, case[2], case[3], window), torch.float16)
    new = [1, 64, 30, 5, 0, 3]
    case = _attention_case(CODES[1], torch.float16, 8, 2, 64, 32, lens, new, seed=window)
    _check(_run(case[0], case[1], lens, case[2], case[3], window=window),
           *_oracle(case[0], case[1], lens, case[2], case[3], window), torch.float16)


@gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D,ps", HEADS)
def test_prompt_attention(code, dtype, H, KV, D, ps):
    """Prompts of odd lengths from nothing, behind a context, of no tokens, and (a refused
    request's shape) with fewer keys than queries, whose first rows see nothing."""
    new = [1, 17, 0, 64, 33, 20, 90]
    lens = [1, 17, 40, 64, 300, 7, 129]
    case = _attention_case(code, dtype, H, KV, D, ps, lens, new, seed=H * D + ps)
    got = _run(case[0], case[1], lens, case[2], case[3])
    _check(got, *_oracle(case[0], case[1], lens, case[2], case[3]), dtype)
    a = int(case[2][5])
    assert (got[a:a + 13] == 0).all() and (got[a + 13] != 0).any()


@gpu
@pytest.mark.parametrize("new,lens", [([300], [300]), ([257, 5], [1300, 4000]), ([3] * 5, [100, 3, 64, 2500, 65]),
                                      ([8, 2], [513, 6000])])
def test_longer_prompts_and_several_tokens(new, lens):
    """Tiles on and off the diagonal, a few tokens over long contexts."""
    for code, dtype in ((CODES[0], torch.bfloat16), (CODES[1], torch.float16)):
        case = _attention_case(code, dtype, 8, 2, 128, 64, lens, new, seed=sum(lens))
        _check(_run(case[0], case[1], lens, case[2], case[3]),
               *_oracle(case[0], case[1], lens, case[2], case[3]), dtype)


@gpu
@pytest.mark.parametrize("H,KV,D", [(8, 2, 128), (8, 1, 64)])
def test_prompts_among_single_tokens(H, KV, D):
    """Requests of few and of many query rows in one call, both in parts that are joined, many
    times over: no part of the one reaches the other's."""
    lens = [3000, 700, 1, 5000, 2500, 64, 1300, 900]
    new = [1, 200, 1, 1, 150, 8, 17, 1]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, H, KV, D, 64, lens, new)
    want = _oracle(c, tables, lens, starts, q)
    first = _run(c, tables, lens, starts, q)
    _check(first, *want, torch.float16)
    for _ in range(50):
        assert torch.equal(_run(c, tables, lens, starts, q), first)


@gpu
def test_attention_takes_strided_queries_and_leaves_rows_behind_the_last():
    lens, new = [70, 9], [5, 2]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 64, 16, lens, new)
    o, weight = _oracle(c, tables, lens, starts, q)
    k, v, ks, vs = c.tensors(DEV)
    wide = torch.full((10, 8, 72), 3.0, dtype=torch.float16, device=DEV)
    view = wide[:, ::2, :64]
    view[:7] = q.to(DEV)
    out = torch.full((10, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    args = (k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens), torch.from_numpy(starts).to(DEV))
    got = P.paged_attention(view, *args, scale=1 / 8, max_q_len=5, out=out)
    assert got is out and (out[7:] == 7).all()
    _check(out[:7], o, weight, torch.float16)
    # odd strides and an odd start go through a copy
    odd = torch.empty(7 * 4 * 67 + 1, dtype=torch.float16, device=DEV)[1:].view(7, 4, 67)[:, :, :64]
    odd.copy_(q.to(DEV))
    assert torch.equal(P.paged_attention(odd, *args, scale=1 / 8, max_q_len=5), out[:7])
    # heads first, as an attention of another framework lays them out
    first = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(P.paged_attention(first, *args, scale=1 / 8, max_q_len=5), out[:7])


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("code", CODES)
def test_attention_ignores_what_lies_behind_a_sequence(code, new):
    """Bytes that are NaN as e4m3, and scales that are infinite or NaN, in the tokens behind
    a sequence's end, in the pages behind it and in tokens before the window: no trace."""
    lens, ps = [50, 131, 64], 32
    c, tables, starts, q = _attention_case(code, torch.float16, 4, 1, 128, ps, lens, [min(new, n) for n in lens],
                                           width=8)
    clean = _run(c, tables, lens, starts, q, window=40)
    pages = c.codes[0].shape[0]
    used = {int(tables[r, p // ps]) for r, n in enumerate(lens) for p in range(max(0, n - new - 39), n)}
    for r, n in enumerate(lens):
        if n % ps:
            for i in range(2):
                c.codes[i][tables[r, n // ps], :, n % ps:] = 0x7F
    for page in set(range(pages)) - used:
        for i in range(2):
            c.codes[i][page] = 0xFF
            c.scales[i][page] = [np.nan, np.inf][page % 2]
    assert torch.equal(_run(c, tables, lens, starts, q, window=40), clean)


@gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 20, 1]])
def test_attention_skips_pages_outside_the_cache(new):
    """Table entries outside the cache (a request that was refused pages): their tokens are
    as if they were not there."""
    lens = [100, 300, 70]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 64, 32, lens, new)
    tables[0, 1], tables[1, 4], tables[1, 0] = -1, 1 << 30, c.codes[0].shape[0]
    tables[2, :3] = -5
    got = _run(c, tables, lens, starts, q)
    _check(got, *_oracle(c, tables, lens, starts, q), torch.float16)
    assert (got[int(starts[2]):] == 0).all()


@gpu
@pytest.mark.parametrize("new", [1, 24])
def test_attention_of_peaked_and_large_scores(new):
    """Scores of several hundred (one position takes all), a scale of zero (all alike) and
    pages whose values are 10^4 times another's."""
    lens = [200, 513]
    n = [min(new, x) for x in lens]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 128, 16, lens, n, spread=60.0)
    got = _run(c, tables, lens, starts, q)
    o, weight = _oracle(c, tables, lens, starts, q)
    # scores are 30 times the other tests': their fp32 sums are off by up to 30 * 2^-13
    err = np.abs(got.double().cpu().numpy() - o)
    # (below 2^-14 a step of fp16 is 2^-24, however small the value: half of it, as in _tolerance)
    assert (err <= HALF[torch.float16] * np.abs(o) + (2.0 ** -11 + 30 * 2.0 ** -12) * weight + 2.0 ** -25).all()
    k, v, ks, vs = c.tensors(DEV)
    c.scales[1][::2] *= np.float32(1e4)
    c.scales[1][1::5] = 0
    vs = torch.from_numpy(c.scales[1]).to(DEV)
    flat = P.paged_attention(q.to(DEV).float().clamp(-4, 4).half(), k, v, ks, vs, torch.from_numpy(tables).to(DEV),
                             _ints(lens), torch.from_numpy(starts).to(DEV), scale=0.0, max_q_len=max(n))
    o, weight = S.attention(np.zeros(q.shape), c.values(0), c.values(1), tables, lens, starts, 16, 0.0)
    fits = np.abs(o) < 65000
    err = np.abs(flat.double().cpu().numpy() - o)
    assert (err <= _tolerance(o, weight, torch.float16))[fits].all()


@gpu
@pytest.mark.parametrize("code", CODES)
def test_append_of_the_smallest_values(code):
    """Values whose scale has no finite inverse in fp32: still codes of the right sign and
    no larger than they should be, so off by at most themselves, top / FLT_MAX."""
    g = torch.Generator().manual_seed(1)
    qkv = (torch.randn(20, 3 * 64, generator=g) * 1e-38).to(torch.bfloat16)
    qkv[3:6] = 0
    cos, sin = _rope(20, 64)
    c = P.PagedKVCache(1, 1, 20, 1, 64, DEV, page_size=16, dtype=code)
    plan = c.extend(_ints([20]), 20)
    c.append(0, qkv.to(DEV), torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV), plan)
    want = S.Cache(2, 1, 16, 64, code)
    want.append(qkv.float().numpy(), cos, sin, np.arange(20), np.arange(20), 1)
    _check_cache(want, c.k[0], c.v[0], c.k_scale[0], c.v_scale[0])
    _, v = P.read_kv_pages(c.block_tables[0], c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], dtype=torch.float32)
    got = v.reshape(-1, 64)[:20].cpu().double()
    err = (got - qkv[:, 128:].double()).abs()
    assert err.max() <= (127 if code == torch.int8 else 448) / np.finfo(np.float32).max


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("code", CODES)
def test_attention_of_the_smallest_value_scales(code, new):
    """Value scales of 1e-38 and zero beside ordinary ones, seen by one request each."""
    lens = [40, 200, 130]
    c, tables, starts, q = _attention_case(code, torch.bfloat16, 8, 2, 64, 16, lens, [new] * 3)
    c.scales[1][tables[0, :3]] = 1e-38
    c.scales[1][tables[1, 1::2]] = 1e-38
    c.scales[1][tables[2, :8]] = 0
    got = _run(c, tables, lens, starts, q)
    _check(got, *_oracle(c, tables, lens, starts, q), torch.bfloat16)
    assert got[:new].abs().max() <= 1e-38 * (127 if code == torch.int8 else 448) * 1.01


@gpu
def test_shared_pages_and_bounds_that_are_too_large():
    """Two requests with a common prefix's pages, limits far above what is there."""
    lens, new = [100, 101], [1, 1]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 128, 64, lens, new, width=40)
    tables[1] = tables[0]
    want = _oracle(c, tables, lens, starts, q)
    for kw in (dict(), dict(max_kv_len=101), dict(max_kv_len=1 << 20)):
        _check(_run(c, tables, lens, starts, q, **kw), *want, torch.float16)
    k, v, ks, vs = c.tensors(DEV)
    got = P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                            torch.from_numpy(starts).to(DEV), scale=1 / 128 ** 0.5)
    _check(got, *want, torch.float16)
    got = P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                            torch.from_numpy(starts).to(DEV), scale=1 / 128 ** 0.5, max_q_len=1000)
    _check(got, *want, torch.float16)


@gpu
def test_without_bounds_everything_is_attended_to():
    lens, new = [100, 300, 7], [60, 1, 7]
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 128, 64, lens, new)
    k, v, ks, vs = c.tensors(DEV)
    got = P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                            torch.from_numpy(starts).to(DEV), scale=1 / 128 ** 0.5)
    _check(got, *_oracle(c, tables, lens, starts, q), torch.float16)


@gpu
def test_python_checks():
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 2, 64, 16, [20], [1])
    k, v, ks, vs = c.tensors(DEV)
    t, lens, q = torch.from_numpy(tables).to(DEV), _ints([20]), q.to(DEV)
    ok = dict(scale=0.1)
    for args in ((q.float(), k, v, ks, vs, t, lens), (q, k, v[:, :, :, :32], ks, vs, t, lens),
                 (q, k, v, ks[:1], vs, t, lens), (q, k, v.view(torch.uint8), ks, vs, t, lens),
                 (q, k, v, ks, vs, t.long(), lens), (q, k, v, ks, vs, t, lens.long()),
                 (q[..., :32], k, v, ks, vs, t, lens), (q.expand(2, 4, 64), k, v, ks, vs, t, lens)):
        with pytest.raises(AssertionError):
            P.paged_attention(*args, **ok)
    with pytest.raises(RuntimeError):
        P.paged_attention(q, k, v, ks, vs, t.cpu(), lens, **ok)
    with pytest.raises(AssertionError):
        P.paged_attention(q, k, v, ks, vs, t, lens, out=q[..., :32], **ok)
    with pytest.raises(AssertionError):
        P.extend_block_tables(t, lens, lens.long(), lens, _ints([0, 0, 0, 0]), 16, 1)
    with pytest.raises(_lib.PmiError):
        P.extend_block_tables(t, lens, lens, lens, _ints([0, 0, 0, 0]), 24, 1)


# --- extremes ----------------------------------------------------------------------------

def _check_finite(got, o, weight, dtype):
    """``_check``, and nothing is NaN where the definition is not."""
    assert got.isfinite().all(), f"{(~got.isfinite()).sum().item()} of {got.numel()} not finite"
    _check(got, o, weight, dtype)


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size,keys", [(1e-24, 1), (1e-27, 1), (1e-37, 1), (1e20, 1e-20)])
def test_attention_of_small_queries_and_small_keys(size, keys, new):
    """bf16 queries whose products with the keys' scales leave fp32's range on one side, over
    partial last tiles and pages of zero keys: finite, and right, in both forms."""
    lens, ps = [200, 513, 70], 32
    c, tables, starts, q = _attention_case(CODES[0], torch.bfloat16, 4, 1, 128, ps, lens, [new] * 3, spread=2 * size)
    c.scales[0] *= np.float32(keys)
    for page in (tables[0, 1], tables[1, 7], tables[1, 16]):
        c.codes[0][page] = 0
        c.scales[0][page] = 0
    _check_finite(_run(c, tables, lens, starts, q), *_oracle(c, tables, lens, starts, q), torch.bfloat16)
    k, v, ks, vs = c.tensors(DEV)
    flat = P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                             torch.from_numpy(starts).to(DEV), scale=0.0, max_q_len=new)
    _check_finite(flat, *S.attention(np.zeros(q.shape), c.values(0), c.values(1), tables, lens, starts, ps, 0.0),
                  torch.bfloat16)


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size,keys", [(0.9e38, 1e-38), (2e-39, 1e38)])
def test_attention_of_queries_at_the_ends_of_bf16(size, keys, new):
    """Queries of up to the largest bf16 and subnormal ones, with keys that make ordinary
    scores of them."""
    lens = [200, 513, 70]
    c, tables, starts, q = _attention_case(CODES[0], torch.bfloat16, 4, 1, 128, 32, lens, [new] * 3, spread=1.0)
    q = (q.double() * size).clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
    largest = q.abs().float().amax(-1)
    assert largest.isfinite().all() and (largest.max() > 2.0 ** 127 if size > 1 else largest.max() < 2.0 ** -126)
    c.scales[0] *= np.float32(keys)
    _check_finite(_run(c, tables, lens, starts, q), *_oracle(c, tables, lens, starts, q), torch.bfloat16)


def test_attention_accepts_one_long_request_among_many():
    """The count of tiles that must fit 32 bits is that of the requests of few query rows: a
    long prompt, or a chunk, among many requests is not refused (but for the workspace that
    is missing here), nor are loose bounds; a count that does not fit is."""
    L = _lib.lib()
    for kw in (dict(T=16384, R=256, max_q=8192, max_kv=32768, width=512), dict(T=8192, R=64, max_q=8192,
                                                                               max_kv=131072, width=2048),
               dict(T=34000, R=64, max_q=32768, max_kv=32768, width=512), dict(T=4096, R=4096, max_q=1, max_kv=131072,
                                                                               width=2048)):
        rc = L.pmi_paged_attention(*_attention_args(H=32, KV=8, ps=64, stride=4096, pages=1 << 16, ws=None,
                                                    tstride=kw["width"], **kw))
        assert rc == _lib.PMI_ERR_INVALID and "workspace" in _lib.last_error(), (kw, _lib.last_error())
    rc = L.pmi_paged_attention(*_attention_args(H=32, KV=8, ps=256, stride=4096, T=65536, R=4096, max_q=16, ws=None,
                                                max_kv=1 << 22, width=1 << 14, tstride=1 << 14))
    assert rc == _lib.PMI_ERR_UNSUPPORTED and "tiles" in _lib.last_error()


@gpu
def test_attention_with_bounds_far_above_a_ragged_batch():
    """A prompt and many single tokens without bounds, tables for half a million tokens."""
    lens, new = [200] + [20 + i for i in range(63)], [200] + [1] * 63
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 16, 2, 64, 64, lens, new, width=8400)
    k, v, ks, vs = c.tensors(DEV)
    rows = torch.zeros(6000, 16, 64, dtype=torch.float16, device=DEV)
    rows[:263] = q.to(DEV)
    got = P.paged_attention(rows, k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                            torch.from_numpy(starts).to(DEV), scale=1 / 8)
    _check_finite(got[:263], *_oracle(c, tables, lens, starts, q), torch.float16)


def test_launches_past_32_bits_are_refused():
    """Grids of 2^32 threads or more (whose sizes a launch counts in 32 bits)."""
    L = _lib.lib()
    n = 1 << 24
    assert L.pmi_read_kv_pages(P8, P8, P8, P8, P8, _lib.PMI_I8, 4, 16, P8, P8, _lib.PMI_F16, n // 4, 4, 64,
                               None) == _lib.PMI_ERR_UNSUPPORTED
    assert L.pmi_rope_append_kv(*_append_args(T=1 << 27, D=128, H=1, KV=1, stride=384)) == _lib.PMI_ERR_UNSUPPORTED
    rc = L.pmi_paged_attention(*_attention_args(H=2, KV=2, D=64, T=1 << 29, R=1 << 23, max_q=65, stride=128, head=64,
                                                max_kv=64, width=4))
    assert rc == _lib.PMI_ERR_UNSUPPORTED, rc


@gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_page_with_an_infinity_reads_as_nan(bad, code):
    """An infinite or NaN key or value makes its page and head NaN, as they are read and for
    every query that sees them; nothing else changes."""
    H, KV, D, ps, T = 4, 2, 64, 16, 40
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv = torch.randn(T, (H + 2 * KV) * D, generator=g, device=DEV).half()
    cos, sin = (torch.from_numpy(t).to(DEV) for t in _rope(48, D))
    for col, which in ((H * D + 5, 0), ((H + KV) * D + 5, 1)):
        caches = []
        for value in (1.0, bad):
            c = P.PagedKVCache(1, 1, 48, KV, D, DEV, page_size=ps, dtype=code)
            x = qkv.clone()
            x[20, col] = value  # second page, head 0
            q = c.append(0, x, cos, sin, c.extend(_ints([T]), T))
            caches.append(c)
        page = caches[1].block_tables[0]
        read = P.read_kv_pages(page, caches[1].k[0], caches[1].v[0], caches[1].k_scale[0], caches[1].v_scale[0])
        clean = P.read_kv_pages(page, caches[0].k[0], caches[0].v[0], caches[0].k_scale[0], caches[0].v_scale[0])
        assert read[which][1, 0].isnan().all()
        read[which][1, 0] = clean[which][1, 0]
        assert torch.equal(read[0], clean[0]) and torch.equal(read[1], clean[1])
        for queries in (q, -q, q[-1:], -q[-1:]):
            n = len(queries)
            want, got = (P.paged_attention(queries, c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], c.block_tables,
                                           c.kv_lens, _ints([0, n]), scale=0.125) for c in caches)
            sees = torch.arange(T - n, T, device=DEV) >= 16
            assert got[sees][:, :2].isnan().all()
            # (the largest value scale of a tile is the unit that probabilities are rounded in, of rows
            # that do not see its page too: both are within _tolerance of the same)
            assert torch.equal(got[:, 2:], want[:, 2:])
            a, b = (t[~sees].double().cpu().numpy() for t in (got, want))
            assert (np.abs(a - b) <= 2 * _tolerance(b, clean[1].abs().max().item(), torch.float16)).all()


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_over_a_scale_that_is_not_finite(bad, which, code, new):
    """What sees a page whose scale is infinite or NaN is NaN in every dimension, whatever its
    codes and the query's sign; other requests and heads are as without it."""
    lens = [100, 130, 64]
    c, tables, starts, q = _attention_case(code, torch.float16, 8, 2, 64, 32, lens, [new] * 3)
    clean = _run(c, tables, lens, starts, q)
    page = tables[1, 1]  # positions 32 to 63 of request 1
    c.codes[which][page, 0] = 0x81 if code == torch.int8 else 0xFE  # the most negative code: no 0 * inf
    c.scales[which][page, 0] = bad
    for sign in (1, -1):
        got = _run(c, tables, lens, starts, sign * q)
        a, b = int(starts[1]), int(starts[2])
        assert got[a:b, :4].isnan().all()
        if sign == 1:
            assert torch.equal(got[a:b, 4:], clean[a:b, 4:])
            assert torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:])


@gpu
@pytest.mark.parametrize("new,lens", [([9, 3], [5, 100]), ([40, 70], [30, 300])])
def test_the_largest_window_hides_nothing(new, lens):
    """Windows up to the largest int, also where there are more queries than keys."""
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 4, 1, 64, 16, lens, new)
    want = _run(c, tables, lens, starts, q)
    assert want[-1].isfinite().all() and (want[-1] != 0).any()
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 10 ** 6):
        assert torch.equal(_run(c, tables, lens, starts, q, window=window), want), window


@gpu
def test_requests_stop_at_max_len():
    """A request may not grow past ``max_len``, also where its last page has room."""
    c = P.PagedKVCache(1, 3, 100, 1, 64, DEV, page_size=64)
    plan = c.extend(_ints([100, 90, 0]), 190)
    assert c.kv_lens.tolist() == [100, 90, 0] and (plan.slots >= 0).all()
    plan = c.extend(_ints([1, 10, 101]), 112)
    assert plan.kv_lens.tolist() == [100, 100, 0] and c.pool[2].item() == 2
    assert plan.first.tolist() == [-1, 90, -1]
    slots = plan.slots.tolist()
    assert slots[0] == -1 and min(slots[1:11]) >= 0 and slots[11:] == [-1] * 101
    plan = c.extend(_ints([0, 1, 100]), 101)
    assert c.kv_lens.tolist() == [100, 100, 100] and c.pool.tolist()[1:3] == [0, 3]
    assert plan.slots.tolist()[0] == -1 and plan.positions.tolist()[1:] == list(range(100))
    # the function itself: no limit but the row, or the one that is given
    t, lens, free, pool = _ints([[0, -1]]), _ints([5]), _ints([0, 1, 2]), _ints([1, 2, 0, 0])
    for limit, want in ((None, 32), (32, 32), (31, 5)):
        plan = P.extend_block_tables(t.clone(), lens, _ints([27]), free, pool, 16, 27, max_len=limit)
        assert plan.kv_lens.tolist() == [want] and plan.pool[2].item() == int(want == 5)
    with pytest.raises(AssertionError):
        P.extend_block_tables(t, lens, _ints([1]), free, pool, 16, 1, max_len=-1)


def test_a_negative_max_len_is_refused():
    a = dict(tables=P8, stride=8, lens=P8, new=P8, free=P8, pool=P8, starts=P8, out=P8, first=P8, fresh=P8, positions=P8,
             slots=P8, pool_out=P8, R=2, width=8, ring=16, ps=16, max_len=-1, total=2)
    assert _lib.lib().pmi_extend_block_tables_upto(*a.values(), None) == _lib.PMI_ERR_INVALID
    assert "max_len" in _lib.last_error()


@gpu
def test_no_call_waits_for_the_device():
    """Every call of a cache, under torch's check for synchronising ones, and captured."""
    KV, D, T = 1, 64, 20
    c = P.PagedKVCache(1, 2, 64, KV, D, DEV, page_size=16)
    cos, sin = (torch.from_numpy(t).to(DEV) for t in _rope(64, D))
    qkv = torch.randn(T, 3 * D, device=DEV).half()
    new, done = _ints([13, 7]), torch.tensor([True, False], device=DEV)

    def step():
        c.reset()
        plan = c.extend(new, T)
        o = c.attend(0, c.append(0, qkv, cos, sin, plan), plan, scale=0.125, max_q_len=13)
        P.read_kv_pages(c.free_pages, c.k[0], c.v[0], c.k_scale[0], c.v_scale[0])
        c.release(done)
        return o

    step()
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        want = step()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    lens, pool, free = c.kv_lens.tolist(), c.pool.tolist(), c.free_pages.tolist()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        c.extend(_ints([30, 30]), 60)  # something for reset to undo
        graph.replay()
        assert torch.equal(got, want)
        assert (c.kv_lens.tolist(), c.pool.tolist(), c.free_pages.tolist()) == (lens, pool, free)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_a_scale_that_is_not_finite_is_refused(scale):
    rc = _lib.lib().pmi_paged_attention(*_attention_args(scale=scale))
    assert rc == _lib.PMI_ERR_INVALID and "scale" in _lib.last_error()


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [-0.1, 1e-6])
def test_negative_and_small_scales(scale, new):
    lens = [200, 65, 330]
    c, tables, starts, q = _attention_case(CODES[0], torch.bfloat16, 4, 1, 128, 32, lens, [new] * 3)
    k, v, ks, vs = c.tensors(DEV)
    got = P.paged_attention(q.to(DEV), k, v, ks, vs, torch.from_numpy(tables).to(DEV), _ints(lens),
                            torch.from_numpy(starts).to(DEV), scale=scale, max_q_len=new)
    _check_finite(got, *S.attention(q.double().numpy(), c.values(0), c.values(1), tables, lens, starts, 32, scale),
                  torch.bfloat16)


# --- forms that only larger calls take ----------------------------------------------------

@gpu
@pytest.mark.parametrize("code,dtype,ps", [(CODES[0], torch.float16, 16), (CODES[1], torch.bfloat16, 128),
                                           (CODES[1], torch.float16, 32), (CODES[0], torch.bfloat16, 256)])
def test_append_of_many_tokens_equals_the_oracle(code, dtype, ps):
    """More than 1024 tokens (several a workgroup, whose runs end in the next ones' tokens):
    ragged prompts behind contexts, refused requests among them, slots outside the cache."""
    H, KV, D = 2, 1, 64 if ps == 32 else 128
    rng = np.random.default_rng(ps)
    lens, new = [0, 5, ps, 3 * ps - 1, 0, 70], [ps + 3, 403, 1, 299, 333, 517]
    refused = 4
    need = [-(-(a + b) // ps) for a, b in zip(lens, new)]
    pages = sum(need)
    c = S.Cache(pages, KV, ps, D, code)
    c.fill(rng)
    k, v, ks, vs = c.tensors(DEV)
    order, at, slots, positions = rng.permutation(pages), 0, [], []
    for r, (a, n) in enumerate(zip(lens, new)):
        row = order[at:at + need[r]]
        at += need[r]
        p = np.arange(a, a + n)
        positions.append(p)
        slots.append(np.full(n, -1) if r == refused else row[p // ps] * ps + p % ps)
        if r == 1:
            slots[-1][17:19] = pages * ps + 5, -7
    slots, positions = np.concatenate(slots).astype(np.int32), np.concatenate(positions).astype(np.int32)
    T = len(slots)
    assert T > 1024
    # a run ends where the slots do: the tokens behind the hole begin another one of the same page, which
    # no caller makes; the page is left out of both
    hole = int(slots[new[0] + 16]) // ps
    slots[slots // ps == hole] = -1
    cos, sin = _rope(1200, D)
    x = torch.from_numpy(rng.standard_normal((T, (H + 2 * KV) * D)) * (0.2 + 3 * rng.random((T, 1)))).to(dtype)
    q = P.rope_append_kv(x.to(DEV), torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV),
                         torch.from_numpy(positions).to(DEV), torch.from_numpy(slots).to(DEV), k, v, ks, vs)
    want = c.append(x.float().numpy(), cos, sin, positions, slots, H)
    assert torch.equal(q.cpu(), torch.from_numpy(want).to(dtype))
    _check_cache(c, k, v, ks, vs)


@gpu
@pytest.mark.parametrize("window", [1100, 2500])
@pytest.mark.parametrize("D,code", [(64, CODES[1]), (128, CODES[0])])
def test_windows_over_several_ranges_of_keys(D, code, window):
    """Many query rows whose window is cut into ranges that are joined."""
    lens, new = [6000, 1300, 3011], [200, 40, 17]
    c, tables, starts, q = _attention_case(code, torch.float16, 8, 2, D, 64, lens, new)
    _check_finite(_run(c, tables, lens, starts, q, window=window),
                  *_oracle(c, tables, lens, starts, q, window), torch.float16)
    alone = _run(c, tables[:1], lens[:1], starts[:2], q[:200], window=window)
    _check_finite(alone, *_oracle(c, tables[:1], lens[:1], starts[:2], q[:200], window), torch.float16)


@gpu
def test_a_cache_past_32_bits_of_bytes():
    """The last pages of a cache of 5 GiB each for keys and values: written, read, attended to
    by a prompt and by a single token."""
    H, KV, D, ps, pages = 4, 4, 128, 256, 40960
    k = torch.zeros(pages, KV, ps, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(pages, KV, ps // 16, D, 16, dtype=torch.int8, device=DEV)
    ks, vs = torch.zeros(pages, KV, device=DEV), torch.zeros(pages, KV, device=DEV)
    T, rows = 300, [pages - 1, pages - 2]
    c = S.Cache(2, KV, ps, D, torch.int8)  # the same two pages alone
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((T, (H + 2 * KV) * D))).half()
    cos, sin = _rope(T, D)
    p = np.arange(T)
    want = c.append(x.float().numpy(), cos, sin, p, p, H)
    slots = np.array(rows)[p // ps] * ps + p % ps
    q = P.rope_append_kv(x.to(DEV), torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV),
                         _ints(p.tolist()), _ints(slots.tolist()), k, v, ks, vs)
    assert torch.equal(q.cpu(), torch.from_numpy(want).half())
    at = torch.tensor(rows, device=DEV)
    _check_cache(c, k[at], v[at], ks[at], vs[at])
    rk, rv = P.read_kv_pages(_ints(rows), k, v, ks, vs, dtype=torch.float32)
    for got, i in ((rk, 0), (rv, 1)):
        assert torch.equal(got.cpu(), torch.from_numpy(S.decode(c.codes[i], c.dtype) * c.scales[i][..., None, None]))
    tables = np.array([[0, 1]], np.int32)
    for n in (1, T):
        starts = np.array([0, n], np.int32)
        got = P.paged_attention(q[-n:], k, v, ks, vs, _ints([rows]), _ints([T]), _ints([0, n]), scale=1 / 128 ** 0.5)
        _check_finite(got, *_oracle(c, tables, [T], starts, q[-n:].cpu()), torch.float16)


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("power,low", [(20, 130), (40, 130), (70, 130), (20, 10), (70, 40), (100, 10)])
def test_pages_of_much_larger_values(power, low, where, new):
    """A page whose values are 2^power times the others', with scores lower by about `low` (no
    weight at all, or some of the output, or all of it), or which only the last queries see."""
    lens, ps = [300, 64, 1000], 16
    c, tables, starts, q = _attention_case(CODES[0], torch.bfloat16, 4, 1, 128, ps, lens, [new] * 3, spread=1.0)
    q[..., 0] = 4.0
    for r, n in enumerate(lens):
        page = tables[r, {"first": 0, "middle": n // ps // 2, "last": (n - 1) // ps}[where]]
        c.scales[1][page] *= np.float32(2.0 ** power)
        if where != "last" or new == 1:
            c.codes[0][page, :, :, 0] = 0x81
            c.scales[0][page] = low * 128 ** 0.5 / (4 * 127)
            c.codes[0][page, :, :, 1:] = 0
    got = _run(c, tables, lens, starts, q)
    o, weight = _oracle(c, tables, lens, starts, q)
    # fp16 holds products of probabilities and scales as 2^8 of the largest and in steps of 2^-24: each is off
    # by up to 2^-33 of that, up to 1000 of them with codes up to 127 by 2^-16, where a page of the
    # largest products has codes of 0 (2^-15 of what half a code of it stands for)
    for r in range(3):
        big = int(np.argmax([c.scales[1][p, 0] for p in tables[r, :-(-lens[r] // ps)]]))
        ones = np.zeros_like(c.values(1))
        ones[tables[r, big]] = c.scales[1][tables[r, big], 0]
        rows = slice(int(starts[r]), int(starts[r + 1]))
        weight[rows] += S.attention(q[rows].double().numpy(), c.values(0), ones, tables[r:r + 1], lens[r:r + 1],
                                    np.array([0, new]), ps, 1 / 128 ** 0.5)[0] * 2.0 ** -5
    # (2^-16 of it is 2^-5 of what _tolerance takes from the weight, 2^-11)
    _check_finite(got, o, weight, torch.bfloat16)


@gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("window", [0, 30])
def test_keys_past_the_bound_are_left_out(window, new):
    """A request of more keys than ``max_kv_len``, or than its table's row holds: its queries
    see what they see of the first ones, from where they stand."""
    lens, ps = [100, 300, 64], 32
    c, tables, starts, q = _attention_case(CODES[0], torch.float16, 8, 2, 64, ps, lens, [new] * 3)
    for bound in (50, 64, 80, 288):
        want = S.attention(q.double().numpy(), c.values(0), c.values(1), tables, lens, starts, ps, 1 / 8, window,
                           bound)
        _check_finite(_run(c, tables, lens, starts, q, window=window, max_kv_len=bound), *want, torch.float16)
        if bound % ps == 0:  # and by rows of so many pages
            short = np.ascontiguousarray(tables[:, :bound // ps])
            _check_finite(_run(c, short, lens, starts, q, window=window), *want, torch.float16)


@gpu
def test_tokens_past_the_total_are_refused_with_their_request():
    """More new tokens than ``total`` says: the requests whose tokens have no place in the plan
    keep their lengths, so that no key is counted that was never written."""
    for R, total, ps in ((4, 25, 16), (4, 5000, 16)):
        new = [total - 5, 3, 4, 0]
        c = P.PagedKVCache(0, R, 2 * total, 1, 64, DEV, page_size=ps)
        plan = c.extend(_ints(new), total)
        assert plan.kv_lens.tolist() == [total - 5, 3, 0, 0]
        assert plan.q_starts.tolist() == [0, total - 5, total - 2, total, total]
        assert plan.slots.tolist()[total - 2:] == [-1, -1] and min(plan.slots.tolist()[:total - 2]) >= 0
        taken = -(-(total - 5) // ps) + 1
        pages = c.free_pages.numel()
        assert c.pool.tolist() == [taken, pages - taken, 1, 0] and plan.first.tolist() == [0, 0, -1, 0]
        plan = c.extend(_ints([0, 0, 4, 1]), 5)
        assert plan.kv_lens.tolist() == [total - 5, 3, 4, 1] and min(plan.slots.tolist()) >= 0


@gpu
@pytest.mark.parametrize("R,ps,longest,newest,short", [(70, 16, 200, 90, 100), (300, 64, 1000, 90, 7000), (5, 32, 10, 4, 1)])
def test_extend_with_a_total_that_is_too_small(R, ps, longest, newest, short):
    rng = random.Random(R)
    tables, lens, new, free, pool = _random_tables(rng, R, ps, longest, newest, 3)
    total = max(0, sum(new) - short)
    want = S.extend_tables(tables, lens, new, free, pool, ps, total)
    t = _ints(tables)
    plan = P.extend_block_tables(t, _ints(lens), _ints(new), _ints(free), _ints(pool), ps, total)
    got = (t, plan.q_starts, plan.kv_lens, plan.first, plan.positions, plan.slots, plan.pool)
    assert want[6][2] > pool[2]
    for name, g, w in zip(("tables", "q_starts", "kv_lens", "first", "positions", "slots", "pool"), got, want):
        assert g.tolist() == w, name


def test_the_workspace_of_a_bound_past_the_table_is_enough():
    """What the query asks for a bound is what the call takes with it, whatever the table's
    width: more keys may take fewer ranges, and so less workspace."""
    L = _lib.lib()
    sizes = dict(T=300, R=1, H=4, KV=1, D=128, max_q=300)
    need = {n: L.pmi_paged_attention_workspace_bytes(*sizes.values(), n, 0) for n in (42432, 42433, 1 << 30, (1 << 31) - 1)}
    assert need[42433] < need[42432] and need[1 << 30] == need[(1 << 31) - 1]
    for max_kv in need:
        args = dict(**sizes, ps=64, width=663, tstride=663, max_kv=max_kv)  # 42432 tokens
        rc = L.pmi_paged_attention(*_attention_args(**args, ws=None))
        assert rc == _lib.PMI_ERR_INVALID and f" {need[max_kv]} bytes" in _lib.last_error()
    many = L.pmi_paged_attention_workspace_bytes(100000, 8, 32, 8, 128, 100000, (1 << 31) - 1, 0)
    assert many == L.pmi_paged_attention_workspace_bytes(100000, 8, 32, 8, 128, 100000, 1 << 30, 0) < 1 << 30


@gpu
def test_a_cache_without_heads_is_refused():
    k, v = torch.zeros(2, 0, 16, 64, dtype=torch.int8, device=DEV), torch.zeros(2, 0, 1, 64, 16, dtype=torch.int8, device=DEV)
    s, i, angles = torch.zeros(2, 0, device=DEV), _ints([0]), torch.zeros(1, 32, device=DEV)
    qkv = torch.zeros(1, 192, dtype=torch.float16, device=DEV)
    for call in (lambda: P.rope_append_kv(qkv, angles, angles, i, i, k, v, s, s), lambda: P.read_kv_pages(i, k, v, s, s),
                 lambda: P.paged_attention(qkv.view(1, 3, 64), k, v, s, s, i[None], i, scale=1.0)):
        with pytest.raises(AssertionError, match="head"):
            call()
