"""Requests from one prompt, as a serving loop and the decoder have them: forks, steps,
releases, compactions and resizes of one cache, its attention and its logits together,
captured and on other streams; generation behind a prefix and with rules."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import pare_amd as P
from oracle import serving_oracle as S
from pare_amd import _lib
from pare_amd.decoder import DecoderConfig, QuantizedDecoder, add_rmsnorm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
CODES = [torch.int8, torch.float8_e4m3fn]
SMALL = DecoderConfig(hidden=1024, heads=8, kv_heads=2, ffn=2048, vocab=2000, layers=2)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rope(L, D):
    a = np.arange(L)[:, None] / 10000.0 ** (np.arange(0, D, 2) / D)
    return tuple(torch.from_numpy(f(a).astype(np.float32)).to(DEV) for f in (np.cos, np.sin))


def _against_64_bits(q, out, cache, layer, plan, scale):
    """Attention over the pages as they are read back, in 64 bits: half a step of fp16 in
    the output and in the probabilities, the latter twice (numerator and sum) with their
    scores' fp32 sums (2^-12), and the smallest subnormal's half."""
    pages = cache.k_scale[layer].shape[0]
    k, v = P.read_kv_pages(torch.arange(pages, dtype=torch.int32, device=DEV), cache.k[layer], cache.v[layer],
                           cache.k_scale[layer], cache.v_scale[layer], dtype=torch.float32)
    k, v = (t.double().cpu().numpy() for t in (k, v))
    o, weight = S.attention(q.double().cpu().numpy(), k, v, cache.block_tables.cpu().numpy(),
                            plan.kv_lens.cpu().numpy(), plan.q_starts.cpu().numpy(), cache.page_size, scale)
    err = np.abs(out.double().cpu().numpy() - o)
    assert (err <= 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2.0 ** -12) * 1.001 * weight + 2.0 ** -25).all(), err.max()


def _values(cache, r, n):
    """The first n tokens of request r, of every layer, by its table."""
    pages = cache.block_tables[r, :-(-n // cache.page_size)].contiguous()
    got = []
    for i in range(len(cache.k)):
        for t in P.read_kv_pages(pages, cache.k[i], cache.v[i], cache.k_scale[i], cache.v_scale[i], dtype=torch.float32):
            got.append(t.transpose(1, 2).flatten(0, 1)[:n])
    return torch.stack(got) if got else None


def _consistent(cache):
    """Every page is free, or has as many owners as shares says; the free ones have none."""
    pages, lens = cache.free_pages.numel(), cache.kv_lens.tolist()
    owners, rows = [0] * pages, cache.block_tables.tolist()
    for r, n in enumerate(lens):
        held = rows[r][:-(-n // cache.page_size)]
        assert len(set(held)) == len(held) and all(0 <= p < pages for p in held)
        for p in held:
            owners[p] += 1
    head, count = cache.pool.tolist()[:2]
    free = [cache.free_pages.tolist()[(head + i) % pages] for i in range(count)]
    assert sorted(free) == [p for p in range(pages) if owners[p] == 0]
    assert cache.shares.tolist() == [max(o - 1, 0) for o in owners]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page_size,seed", [(16, 0), (32, 1), (64, 2)])
def test_a_serving_loop_of_forks(code, page_size, seed):
    """Requests are extended by chunks and by single tokens, forked at any length, end, and the cache is made
    dense, smaller and larger; after every step each page has the owners it should, what requests
    hold is what they held before (bit for bit, but for pages that a new token has rounded again), and attention is
    that of their own tables."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    R, H, KV, D, L = 8, 4, 2, 64, 300
    cache = P.PagedKVCache(2, R, L, KV, D, DEV, page_size=page_size, dtype=code, sharing=True)
    cos, sin = _rope(L, D)
    lens = [0] * R
    for step in range(40):
        what = rng.choice(["extend", "extend", "token", "token", "token", "fork", "fork", "release", "compact", "resize"])
        before = [_values(cache, r, n) if n else None for r, n in enumerate(lens)]
        if what in ("extend", "token"):
            new = [0 if n == 0 and what == "token" else min(L - n, 1 if what == "token" else rng.randint(0, 60)) for n in lens]
            if sum(new) == 0:
                continue
            plan = cache.extend(_ints(new), sum(new))
            shared = cache.shared_prefixes(plan, least=page_size)
            qkv = torch.randn(2, sum(new), (H + 2 * KV) * D, generator=g).half().to(DEV)
            for layer in range(2):
                q = cache.append(layer, qkv[layer], cos, sin, plan)
                out = cache.attend(layer, q, plan, scale=0.125, max_q_len=max(new), shared=shared)
                _against_64_bits(q, out, cache, layer, plan, 0.125)
            old, lens = lens, [n + m for n, m in zip(lens, new)]
            for r in range(R):
                kept = old[r] // page_size * page_size if new[r] else old[r]  # whole pages stay as they were
                if kept:
                    assert torch.equal(_values(cache, r, old[r])[:, :kept], before[r][:, :kept])
            assert int(plan.pool[2]) == int(cache.pool[2])
        elif what == "fork":
            parents = [rng.randrange(-1, R) for _ in range(R)]
            at = [rng.choice([10 ** 6, rng.randint(0, L)]) for _ in range(R)]
            refused = int(cache.pool[2])
            cache.fork(_ints(parents), _ints(at))
            want = list(lens)
            for r, p in enumerate(parents):
                if 0 <= p != r and lens[r] == 0:
                    want[r] = min(lens[p], at[r])
                refused += 0 <= p != r and lens[r] > 0
            assert cache.kv_lens.tolist() == want and int(cache.pool[2]) == refused
            for r in range(R):
                if want[r] and not lens[r]:
                    assert torch.equal(_values(cache, r, want[r]), before[parents[r]][:, :want[r]])
            lens = want
        elif what == "release":
            done = [rng.random() < 0.4 for _ in range(R)]
            cache.release(torch.tensor(done, device=DEV))
            lens = [0 if d else n for n, d in zip(lens, done)]
        elif what == "compact":
            cache.compact()
            live = cache.free_pages.numel() - int(cache.pool[1])
            assert cache.free_pages.tolist()[:1] == [live % cache.free_pages.numel()]
        else:
            live = cache.free_pages.numel() - int(cache.pool[1])
            with pytest.raises(ValueError):
                cache.resize(live - 1 if live > 1 else 0)
            cache.resize(live + R * (-(-L // page_size)))
        assert cache.kv_lens.tolist() == lens
        _consistent(cache)
        if what in ("fork", "release", "compact", "resize"):
            for r, n in enumerate(lens):
                if n and before[r] is not None:
                    assert torch.equal(_values(cache, r, n), before[r])
    cache.reset()
    _consistent(cache)


@pytest.mark.parametrize("sharing", [True, False])
def test_compaction_and_sizes_of_a_cache(sharing):
    """Both kinds of cache are compacted, shrunk and grown, and serve on; a plan's slots are those of
    the places at its making."""
    cache = P.PagedKVCache(2, 4, 128, 2, 64, DEV, page_size=16, sharing=sharing)
    cos, sin = _rope(128, 64)
    g = torch.Generator(device=DEV).manual_seed(int(sharing))

    def step(lens):
        total = sum(lens)
        plan = cache.extend(_ints(lens), total)
        for i in range(2):
            cache.append(i, torch.randn(total, 8 * 64, generator=g, device=DEV).half(), cos, sin, plan)
        return plan

    step([40, 100, 16, 33])
    cache.release(torch.tensor([False, True, False, False], device=DEV))
    for change in (cache.compact, lambda: cache.resize(8), lambda: cache.resize(40), cache.compact):
        lens = cache.kv_lens.tolist()
        want = [_values(cache, r, n) for r, n in enumerate(lens) if n]
        change()
        assert cache.kv_lens.tolist() == lens
        for a, b in zip(want, [_values(cache, r, n) for r, n in enumerate(lens) if n]):
            assert torch.equal(a, b)
        live = sum(-(-n // 16) for n in lens)
        assert sorted(p for r, n in enumerate(lens) for p in cache.block_tables[r, :-(-n // 16)].tolist()) == [*range(live)]
        pages = cache.free_pages.numel()
        assert cache.pool.tolist()[:2] == [0, pages - live]
        assert cache.free_pages.tolist() == [(live + i) % pages for i in range(pages)]
    with pytest.raises(ValueError, match="hold 7 pages"):
        cache.resize(6)
    plan = step([3, 20, 1, 0])
    assert plan.kv_lens.tolist() == [43, 20, 17, 33] and cache.pool.tolist()[2] == 0
    q = torch.randn(24, 4, 64, generator=g, device=DEV).half()
    for i in range(2):
        _against_64_bits(q, cache.attend(i, q, plan, scale=0.125), cache, i, plan, 0.125)
    if sharing:
        _consistent(cache)


def test_forks_that_the_pool_cannot_hold_are_refused_whole():
    cache = P.PagedKVCache(1, 4, 64, 1, 64, DEV, page_size=16, pages=4, sharing=True)
    cache.extend(_ints([40, 0, 0, 0]), 40)
    cache.fork(_ints([-1, 0, 0, 0]), _ints([0, 40, 40, 32]))  # one page is left; whole pages need none
    assert cache.kv_lens.tolist() == [40, 40, 0, 32] and cache.pool.tolist()[1:3] == [0, 1]
    _consistent(cache)
    plain = P.PagedKVCache(1, 4, 64, 1, 64, DEV)
    for call in (lambda: plain.fork(_ints([0] * 4)),):
        with pytest.raises(RuntimeError):
            call()


def test_a_step_of_all_operators_captured_and_on_another_stream():
    """extend, runs, append, attend, greedy choice and the release of what has ended, in one graph, with
    eager work between the replays; the same steps made eagerly on another cache, bit for bit."""
    R, H, KV, D, L, V = 6, 8, 2, 128, 60000, 3001  # (long enough for shared pages to be read once)

    def make():
        g = torch.Generator(device=DEV).manual_seed(3)
        cache = P.PagedKVCache(1, R, L, KV, D, DEV, page_size=64, sharing=True)
        cos, sin = _rope(L, D)
        w = torch.randn(H * D, V, generator=g, device=DEV).half() * 0.1
        emb = torch.randn(V, (H + 2 * KV) * D, generator=g, device=DEV).half()
        prompt = torch.randn(2500, (H + 2 * KV) * D, generator=g, device=DEV).half()
        plan = cache.extend(_ints([2500] + [0] * (R - 1)), 2500)
        cache.append(0, prompt, cos, sin, plan)
        cache.fork(_ints([-1] + [0] * (R - 1)), _ints([0, 2500, 2496, 2490, 1000, 2500]))
        s = dict(tok=torch.arange(R, device=DEV)[:, None] * 7, live=_ints([1] * R), history=torch.zeros(R, 64, dtype=torch.int32,
                 device=DEV), lens=_ints([0] * R))
        rules = P.LogitRules(repetition=torch.full((R,), 1.3, device=DEV), frequency=torch.full((R,), 0.5, device=DEV),
                             allowed=torch.full((1, -(-V // 32)), -2, dtype=torch.int32, device=DEV),
                             allowed_rows=_ints([0, -1] * (R // 2)))

        def step():
            plan = cache.extend(s["live"], R)
            shared = cache.shared_prefixes(plan)
            order = torch.where(s["live"] > 0, plan.q_starts[:-1], R).long()
            rows = torch.zeros(R + 1, dtype=torch.long, device=DEV).scatter_(0, order, s["tok"][:, 0])[:R]
            q = cache.append(0, emb.index_select(0, rows), cos, sin, plan)
            o = cache.attend(0, q, plan, scale=D ** -0.5, max_q_len=1, shared=shared)
            logits = torch.matmul(o.reshape(R, -1), w)
            last = (plan.q_starts[1:] - 1).clamp(min=0)
            P.greedy_tokens(logits.index_select(0, last), history=s["history"], history_lens=s["lens"], out=s["tok"],
                            **rules._asdict())
            s["history"].scatter_(1, s["lens"][:, None].long(), s["tok"].int())
            s["lens"].add_(s["live"])
            ended = s["tok"][:, 0] % 5 == 0
            cache.release(ended & (s["live"] > 0))
            s["live"].masked_fill_(ended, 0)
        return cache, s, step

    a, sa, eager = make()
    b, sb, captured = make()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        eager(), captured()
        with torch.cuda.graph(graph, stream=stream):
            captured()
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(12):
        eager()
        torch.randn(1000, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((a.block_tables, a.kv_lens, a.pool, a.shares, *sa.values()), (b.block_tables, b.kv_lens, b.pool,
                                                                                      b.shares, *sb.values())):
            assert torch.equal(x, y)
        _consistent(a)
    assert (sa["history"][0, :int(sa["lens"][0])] != 0).all()  # token 0 is not allowed for every second request


@pytest.mark.parametrize("R,L", [(6, 300), (40, 4000)])
def test_forks_releases_and_compactions_captured(R, L):
    """The tables' small forms and the large ones, with their copies, in a graph: replays leave the cache as the same
    calls do eagerly, bit for bit, with other requests each time."""
    KV, D, ps = 2, 64, 16

    def make():
        cache = P.PagedKVCache(2, R, L, KV, D, DEV, page_size=ps, sharing=True)
        s = dict(new=_ints([0] * R), parents=_ints([-1] * R), at=_ints([0] * R),
                 done=torch.zeros(R, dtype=torch.bool, device=DEV))
        qkv = torch.randn(8 * R, (2 + 2 * KV) * D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
        cos, sin = _rope(L, D)

        def step():
            plan = cache.extend(s["new"], 8 * R)
            for layer in range(2):
                cache.append(layer, qkv, cos, sin, plan)
            cache.fork(s["parents"], s["at"])
            cache.release(s["done"])
            cache.compact()
        return cache, s, step

    (a, sa, eager), (b, sb, captured) = make(), make()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager(), captured()
        with torch.cuda.graph(graph, stream=stream):
            captured()
    torch.cuda.current_stream().wait_stream(stream)
    rng, lens, forks = random.Random(R), [0] * R, 0
    for i in range(25):
        held = [r for r, n in enumerate(lens) if n]
        new = [rng.randint(0, 8) if n or rng.random() < 0.2 else 0 for n in lens]
        parents = [rng.choice(held) if held and not lens[r] and not new[r] and rng.random() < 0.5 else -1 for r in range(R)]
        at = [rng.choice([L, rng.randint(0, L)]) for _ in range(R)]
        done = [rng.random() < 0.15 for _ in range(R)]
        for s in (sa, sb):
            for t, x in zip(s.values(), (new, parents, at, done)):
                t.copy_(torch.tensor(x, dtype=t.dtype))
        eager()
        torch.randn(1000, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((a.block_tables, a.kv_lens, a.pool, a.shares, a.free_pages, *a.k, *a.v, *a.k_scale, *a.v_scale),
                        (b.block_tables, b.kv_lens, b.pool, b.shares, b.free_pages, *b.k, *b.v, *b.k_scale, *b.v_scale)):
            assert torch.equal(x, y)
        lens = a.kv_lens.tolist()
        forks += sum(0 <= p and lens[r] > 0 for r, p in enumerate(parents))
    assert forks > 3
    _consistent(a)


def test_two_streams_at_once():
    """Calls that interleave on two streams have workspaces of their own."""
    x = [torch.randn(64, 50000, device=DEV) for _ in range(2)]
    want = [t.argmax(1) for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(P.greedy_tokens(x[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])


# --- the decoder ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def model():
    return QuantizedDecoder(SMALL, DEV, seed=3)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, SMALL.vocab, (n,), generator=g).to(DEV) for n in lens]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("before", [16, 37, 131])
def test_generation_behind_a_prefix(model, code, before, monkeypatch):
    """Every layer's attention against 64 bits over the pages, shared ones among them; the first layer's
    keys are those of prefix and prompt at their positions (twice half a code: a page that a prompt begins
    inside of may be rounded again)."""
    prefix, prompts = _prompts([before], seed=9)[0], _prompts([5, 40, 1, 17])
    caches = []
    make = model.new_paged_cache

    def recorded(*args, **kw):
        cache = make(*args, **kw)
        caches.append(cache)
        attend = cache.attend

        def check(layer, q, plan, **kw):
            out = attend(layer, q, plan, **kw)
            _against_64_bits(q, out, cache, layer, plan, kw["scale"])
            return out
        monkeypatch.setattr(cache, "attend", check)
        return cache

    monkeypatch.setattr(model, "new_paged_cache", recorded)
    got, _ = model.generate_ragged(prompts, 4, dtype=code, page_size=16, prefix=prefix, use_graph=False)
    cache = caches[0]
    assert cache.kv_lens.tolist() == [before + n + 3 for n in (5, 40, 1, 17)]
    _consistent(cache)
    whole = before // 16
    assert (cache.block_tables[1:, :whole] == cache.block_tables[:1, :whole]).all()
    layer = model.layers[0]
    cos, sin = (t.double().cpu().numpy() for t in model.rope_tables(300))
    for r, p in enumerate(prompts):
        tokens = torch.cat([prefix, p, got[r, :3]])
        x = torch.nn.functional.embedding(tokens, model.embed)
        with torch.no_grad():
            qkv = layer.qkv.fused(add_rmsnorm(x[None], None, layer.attn_norm.weight, SMALL.rms_eps)[0])[0]
        n = len(tokens)
        want = S.rotate(qkv.double().cpu().numpy().reshape(n, -1, 128)[:, 8:10], cos[:n], sin[:n])
        held = _values(cache, r, n)[0].double().cpu().numpy()
        for a in range(0, n, 16):
            x, y = held[a:a + 16], want[a:a + 16]
            top = max(np.abs(y).max(), np.abs(x).max())
            half = top / 254 if code == torch.int8 else np.maximum(np.abs(y) * 2.0 ** -4, top / 448 * 2.0 ** -10)
            # a page may be rounded once more for each of the four calls that write to it, and the row's products
            # are those of another call's kernel: fp16's step of the largest
            assert (np.abs(x - y) <= 4.2 * half + top * 2.0 ** -8).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("before,lens", [(16, [24]), (37, [5, 90, 1]), (300, [33] * 6)])
def test_generation_behind_a_prefix_graph_matches_eager(model, code, before, lens):
    prefix, prompts = _prompts([before], seed=9)[0], _prompts(lens)
    eager, _ = model.generate_ragged(prompts, 12, dtype=code, prefix=prefix, use_graph=False, page_size=16)
    graph, t = model.generate_ragged(prompts, 12, dtype=code, prefix=prefix, page_size=16)
    assert eager.shape == (len(lens), 12) and torch.equal(eager, graph)
    eos = graph[0, 5].item()
    runs = [model.generate_ragged(prompts, 12, dtype=code, prefix=prefix, page_size=16, eos=eos, use_graph=u)[0]
            for u in (False, True)]
    assert torch.equal(*runs)
    for row in runs[0].tolist():
        at = (row + [eos]).index(eos)
        assert row[at:] == [eos] * (12 - at)
    # the prompts that follow the prefix decide: others give other answers
    assert not torch.equal(model.generate_ragged(_prompts(lens, seed=4), 12, dtype=code, prefix=prefix, page_size=16)[0], graph)


@pytest.mark.parametrize("before", [0, 20])
def test_generation_with_rules(model, before):
    """The tokens of a loop over the logits and process_logits, eager and captured; masks hold."""
    V, R, n = SMALL.vocab, 3, 10
    prefix = _prompts([before], seed=9)[0] if before else None
    prompts = _prompts([5, 30, 12])
    mask = torch.randint(-2 ** 31, 2 ** 31, (1, -(-V // 32)), generator=torch.Generator().manual_seed(1)).int().to(DEV)
    rules = P.LogitRules(repetition=torch.tensor([1.0, 1.5, 2.0], device=DEV), presence=torch.tensor([0.0, 0.5, 9.0], device=DEV),
                         frequency=torch.tensor([0.0, 0.3, 0.0], device=DEV), bias_ids=_ints([[3, -1], [4, 5], [6, 6]]),
                         bias=torch.tensor([[9.0, 0.0], [0.5, 0.5], [1.0, 1.0]], device=DEV), allowed=mask,
                         allowed_rows=_ints([-1, 0, -1]))
    got = [model.generate_ragged(prompts, n, prefix=prefix, rules=rules, use_graph=u, page_size=16)[0] for u in (False, True)]
    assert torch.equal(*got)
    bits = np.unpackbits(mask.cpu().numpy().view(np.uint8), bitorder="little")
    assert bits[got[0][1].cpu().numpy()].all()
    assert len(set(got[0][2].tolist())) == n          # 9 for having been said: no token twice
    free = model.generate_ragged(prompts, n, prefix=prefix, page_size=16)[0]
    assert not torch.equal(free, got[0])
    none = model.generate_ragged(prompts, n, prefix=prefix, rules=P.LogitRules(), page_size=16)[0]
    assert torch.equal(none, free)
    # by hand
    whole = [torch.cat([prefix, p]) if before else p for p in prompts]
    lens = [len(p) for p in whole]
    L = max(lens) + n
    cache = model.new_paged_cache(R, L, page_size=16, sharing=before > 0)
    cos, sin = model.rope_tables(L)
    history = [p.tolist() for p in whole]
    with torch.no_grad():
        if before:
            plan = cache.extend(_ints([before, 0, 0]), before)
            assert model.forward_paged(prefix, cos, sin, cache, plan, max_q_len=before, max_kv_len=before, head=False) is None
            cache.fork(_ints([-1, 0, 0]))
        new, tokens = [len(p) for p in prompts], torch.cat(prompts)
        for i in range(n):
            plan = cache.extend(_ints(new), sum(new))
            logits = model.forward_paged(tokens, cos, sin, cache, plan, max_q_len=max(new), max_kv_len=L if i else max(lens))
            longest = max(map(len, history))
            h = _ints([x + [-1] * (longest - len(x)) for x in history])
            out = P.process_logits(logits, history=h, history_lens=_ints([len(x) for x in history]), prompt_lens=_ints(lens),
                                   **rules._asdict())
            tokens = torch.from_numpy(out.float().cpu().numpy().argmax(1)).to(DEV)
            assert tokens.tolist() == got[0][:, i].tolist()
            for r, t in enumerate(tokens.tolist()):
                history[r].append(t)
            new = [1] * R


@pytest.mark.parametrize("before,lens", [(16, [24, 24]), (37, [27] * 5), (300, [4] * 6), (15, [1, 9])])
def test_a_prefix_takes_its_pages_once(model, before, lens, monkeypatch):
    """The cache holds a prefix's whole pages once and everything else of every request, of whom none is refused: the
    tokens are those of a cache with room for all of them at full length."""
    prefix, prompts, n, ps = _prompts([before], seed=9)[0], _prompts(lens), 9, 16
    R, width, common = len(lens), -(-(before + max(lens) + n) // ps), before // ps
    make = model.new_paged_cache
    for use_graph in (False, True):
        got = []
        for whole in (False, True):
            caches = []

            def recorded(*args, pages=None, **kw):
                caches.append(make(*args, pages=None if whole else pages, **kw))
                return caches[-1]

            monkeypatch.setattr(model, "new_paged_cache", recorded)
            got.append(model.generate_ragged(prompts, n, prefix=prefix, page_size=ps, use_graph=use_graph)[0])
            assert caches[0].free_pages.numel() == (R * width if whole else common + R * (width - common))
            assert caches[0].kv_lens.tolist() == [before + m + n - 1 for m in lens]
            assert caches[0].pool.tolist()[2] == 0
            _consistent(caches[0])
        assert torch.equal(*got)
    # every page is needed where the requests are as long as each other
    if len(set(lens)) == 1 and (before + lens[0] + n - 2) // ps == width - 1:
        cache = caches[0]
        cache.compact()
        cache.resize(common + R * (width - common))
        assert int(cache.pool[1]) == 0


def test_refusals(model):
    prompts = _prompts([9, 2])
    for bad in (torch.zeros(0, dtype=torch.long), torch.zeros(1, 2, dtype=torch.long)):
        with pytest.raises(ValueError):
            model.generate_ragged(prompts, 4, prefix=bad)
    with pytest.raises(AssertionError):
        model.generate_ragged(prompts, 4, rules=P.LogitRules(repetition=torch.ones(3, device=DEV)))


@pytest.mark.parametrize("page_size", [0, -16, 24])
def test_page_sizes_that_no_cache_has_are_refused(model, page_size):
    for prefix in (None, *_prompts([30])):
        with pytest.raises(ValueError, match="page_size"):
            model.generate_ragged(_prompts([9, 2]), 4, prefix=prefix, page_size=page_size)


@pytest.mark.parametrize("code", CODES)
def test_a_fork_inside_a_page_has_its_parents_scale(code):
    """Tokens behind the fork's, in the page where it ends, have made the page what it is: coarse for large ones, NaN
    for an infinity. Its whole pages, and the page's other heads, are not touched by that."""
    cache = P.PagedKVCache(1, 4, 64, 2, 64, DEV, page_size=16, dtype=code, sharing=True)
    cos, sin = _rope(64, 64)
    qkv = torch.randn(60, 6 * 64, generator=torch.Generator().manual_seed(2)).half()
    qkv[28, 4 * 64:5 * 64] = 1000            # values of head 0, behind the first fork's 24 tokens
    qkv[45, 5 * 64:] = float("inf")          # of head 1, behind the second's 40
    plan = cache.extend(_ints([60, 0, 0, 0]), 60)
    cache.append(0, qkv.to(DEV), cos, sin, plan)
    cache.fork(_ints([-1, 0, 0, 0]), _ints([0, 24, 40, 32]))
    for r, n in ((1, 24), (2, 40), (3, 32)):
        mine, parent = _values(cache, r, n), _values(cache, 0, n)
        assert torch.equal(mine.isnan(), parent.isnan()) and torch.equal(mine.nan_to_num(), parent.nan_to_num())
    values = _values(cache, 2, 40)[1]
    assert values[32:, 1].isnan().all() and not values[:32].isnan().any() and not values[32:, 0].isnan().any()
    page = int(cache.block_tables[1, 1])
    top = 127 if code == torch.int8 else 448
    assert abs(float(cache.v_scale[0][page, 0]) * top / 1000 - 1) < 1e-6


def test_generation_whose_shared_pages_are_read_once(model, monkeypatch):
    """As many requests behind as long a prefix as the rule wants: every layer's attention of the prompts' step and of
    the tokens' is the one of parts, and within its tolerance; captured steps give the same tokens."""
    before, n = 7300, 3
    lens = [1 + i * 5 % 8 for i in range(36)]
    prefix, prompts = _prompts([before], seed=9)[0], _prompts(lens)
    make, seen = model.new_paged_cache, []
    L, R, H, KV, D = _lib.lib(), len(lens), SMALL.heads, SMALL.kv_heads, SMALL.head_dim

    def recorded(*args, **kw):
        cache = make(*args, **kw)
        attend = cache.attend

        def check(layer, q, plan, *, max_q_len, max_kv_len, shared, **kw):
            out = attend(layer, q, plan, max_q_len=max_q_len, max_kv_len=max_kv_len, shared=shared, **kw)
            if shared is not None:
                sizes = (q.shape[0], R, H, KV, D, max_q_len, max_kv_len, 0)
                assert L.pmi_paged_attention_shared_workspace_bytes(*sizes) > L.pmi_paged_attention_workspace_bytes(*sizes)
                assert shared.lens.tolist() == [before // 64 * 64] * R and shared.runs[0, 2] == q.shape[0]
                _against_64_bits(q, out, cache, layer, plan, kw["scale"])
                seen.append(layer)
            return out
        monkeypatch.setattr(cache, "attend", check)
        return cache

    with monkeypatch.context() as m:
        m.setattr(model, "new_paged_cache", recorded)
        eager, _ = model.generate_ragged(prompts, n, prefix=prefix, use_graph=False)
    assert seen == [0, 1] * n
    assert torch.equal(model.generate_ragged(prompts, n, prefix=prefix)[0], eager)
