"""The operators of serving many requests from one prompt, as cases to be timed and compared.

Four operators: requests that begin as forks of another one, with the pages that they cannot
share copied (``fork``); finished requests' shared pages given back and the cache's live pages
moved to its front (``compact``); attention of requests whose first pages are the same, those
pages read once for all of them (``attention``); and penalties for repeated tokens, biases and
masks on logits, with the processed logits or only their greedy tokens as the result
(``logits``, ``greedy``). With ``own`` false ``run`` computes them from elementary torch
operations, with ``own`` true it calls pare_amd.

The cache: ``k_cache`` int8 or float8_e4m3fn [pages, kv_heads, page_size, D], ``v_cache`` of
the same type [pages, kv_heads, page_size / 16, D, 16] (token 16 b + j of a page at [b, :, j]),
and one fp32 scale per page and head for each of them; a value is its code times that scale.
``shares`` int32 [pages] counts a page's owners beyond the first.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}  # the largest code


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # four answers to one chat, all layers of an 8B decoder's cache (8 heads of 128): latency
        dict(name="fork_answers", op="fork", requests=4, parents=1, longest=700, kv_heads=8, dim=128, page=64,
             codes="int8", layers=32, lens=1),
        # a scheduler's step that starts 120 requests from eight system prompts, 4 heads, odd lengths
        dict(name="fork_prompts", op="fork", requests=128, parents=8, longest=8190, kv_heads=4, dim=128, page=32,
             codes="fp8", layers=28, lens=2),
        # some of a few chats end: a small cache made dense again
        dict(name="compact_chats", op="compact", requests=12, parents=3, longest=900, kv_heads=8, dim=128, page=64,
             codes="int8", layers=2, lens=3),
        # most of a large batch ends, many small pages, heads of 64
        dict(name="compact_batch", op="compact", requests=256, parents=16, longest=3000, kv_heads=8, dim=64, page=16,
             codes="fp8", layers=32, lens=4),
        # eight answers being written to one chat: the smallest attention call
        dict(name="attn_answers", op="attention", requests=8, families=1, prefix=2000, own=300, newest=1, heads=32,
             kv_heads=8, dim=128, page=64, codes="int8", type="fp16", lens=5),
        # a serving batch behind one long system prompt, one token each
        dict(name="attn_batch", op="attention", requests=64, families=1, prefix=8192, own=700, newest=1, heads=32,
             kv_heads=8, dim=128, page=64, codes="int8", type="fp16", lens=6),
        # several documents, each with its own readers
        dict(name="attn_documents", op="attention", requests=40, families=5, prefix=32000, own=1500, newest=1,
             heads=28, kv_heads=4, dim=128, page=128, codes="fp8", type="bf16", lens=7),
        # questions read in one pass behind a shared context, heads of 64, small pages
        dict(name="attn_questions", op="attention", requests=24, families=2, prefix=6000, own=40, newest=200, heads=32,
             kv_heads=4, dim=64, page=16, codes="fp8", type="bf16", lens=8),
        # one chat's next token, with everything on: latency
        dict(name="logits_one", op="logits", requests=1, vocab=32000, history=300, biases=20, grammars=1, type="fp16",
             lens=9),
        # a serving batch, a vocabulary of odd size, constrained rows among free ones
        dict(name="logits_batch", op="logits", requests=64, vocab=128257, history=4000, biases=64, grammars=8,
             type="bf16", lens=10),
        # greedy decode of a few requests with the vocabulary of an 8B decoder
        dict(name="greedy_few", op="greedy", requests=4, vocab=128256, history=900, biases=0, grammars=0, type="fp16",
             lens=11),
        # a large greedy batch with long histories
        dict(name="greedy_batch", op="greedy", requests=96, vocab=152064, history=16000, biases=300, grammars=16,
             type="fp32", lens=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4))))))


def draw(rng):
    op = rng.choice(["fork", "compact", "attention", "attention", "logits", "greedy"])
    seed = rng.randrange(1 << 20)
    if op in ("logits", "greedy"):
        requests = _log(rng, 1, 96)
        return dict(op=op, requests=requests, vocab=_log(rng, 1000, 152064), history=_log(rng, 1, 16000),
                    biases=rng.choice([0, _log(rng, 1, 300)]), grammars=rng.choice([0, rng.randint(1, 16)]),
                    type=rng.choice(["fp16", "bf16", "fp32"]), lens=seed)
    cache = dict(dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), codes=rng.choice(["int8", "fp8"]),
                 lens=seed)
    if op != "attention":
        parents, children, longest = _log(rng, 1, 16), _log(rng, 1, 120), _log(rng, 10, 4000)
        kv = rng.choice([1, 2, 4, 8])
        page_bytes = 2 * kv * cache["page"] * cache["dim"]
        pages = parents * (longest // cache["page"] + 1) + 2 * children  # a cache of 1 GB, copies of 100 MB
        layers = min(rng.randint(1, 32), 10 ** 9 // (pages * page_bytes), 10 ** 8 // (children * page_bytes))
        return dict(op=op, requests=parents + children, parents=parents, longest=longest, kv_heads=kv,
                    layers=max(1, layers), **cache)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8] if kv <= 4 else [1, 2, 4])
    families = _log(rng, 1, 6)
    if rng.random() < 0.65:
        prefix = _log(rng, 100, 32000)
        requests = families + min(_log(rng, 1, 80), 48 * 8192 // prefix)
        return dict(op=op, requests=requests, families=families, prefix=prefix, own=_log(rng, 1, 1500), newest=1,
                    heads=heads, kv_heads=kv, type=rng.choice(["fp16", "bf16"]), **cache)
    return dict(op=op, requests=families + _log(rng, 1, 12), families=families, prefix=_log(rng, 100, 6000),
                own=_log(rng, 1, 100), newest=_log(rng, 2, 131), heads=heads, kv_heads=kv,
                type=rng.choice(["fp16", "bf16"]), **cache)


def _attention_lengths(case):
    """(family, prefix, own, new) of each request, from the case alone; families in a row."""
    r = random.Random(case["lens"])
    R, F = case["requests"], min(case["families"], case["requests"])
    family = sorted([i if i < F else r.randrange(F) for i in range(R)])
    prefixes = [case["prefix"] if f == 0 else r.randint(max(1, case["prefix"] // 2), case["prefix"]) for f in range(F)]
    behind = [case["own"] if i == 0 else r.randint(0, case["own"]) for i in range(R)]
    new = [case["newest"] if i == 0 else r.randint(max(1, case["newest"] // 8), case["newest"]) for i in range(R)]
    return family, [prefixes[f] for f in family], behind, new


def _fork_lengths(case):
    """Lengths of the parents, and of each child its parent and how many of its tokens it begins with."""
    r = random.Random(case["lens"])
    n = case["requests"] - case["parents"]
    lengths = [case["longest"] if i == 0 else r.randint(max(1, case["longest"] // 4), case["longest"])
               for i in range(case["parents"])]
    parent = [r.randrange(case["parents"]) for _ in range(n)]
    return lengths, parent, [lengths[p] if r.random() < 0.5 else r.randint(1, lengths[p]) for p in parent]


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _quantised(x, kind):
    """Codes and scales of x [pages, heads, tokens, D], one scale per page and head."""
    amax = x.abs().amax((2, 3)).float()
    y = x.float() * (TOP[kind] / amax.clamp_min(1e-20))[..., None, None]
    codes = y.round().to(torch.int8) if kind == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, amax * (1.0 / TOP[kind])


def _filled_cache(pages, case, gen):
    """Caches whose pages all hold keys and values of a model: some channels larger."""
    kv, ps, d, kind = case["kv_heads"], case["page"], case["dim"], case["codes"]
    k = torch.empty(pages, kv, ps, d, dtype=CODES[kind], device=DEV)
    v = torch.empty(pages, kv, ps // 16, d, 16, dtype=CODES[kind], device=DEV)
    ks = torch.empty(pages, kv, dtype=torch.float32, device=DEV)
    vs = torch.empty_like(ks)
    spread = 0.5 + torch.rand(kv, 1, d, generator=gen, device=DEV)
    step = max(1, (1 << 26) // (kv * ps * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        for codes, scales in ((k, ks), (v, vs)):
            x = torch.randn(b - a, kv, ps, d, generator=gen, device=DEV, dtype=torch.float16) * spread.half()
            c, scales[a:b] = _quantised(x, kind)
            if codes is v:
                c = c.view(torch.uint8).reshape(b - a, kv, ps // 16, 16, d).transpose(3, 4)
                c = c.contiguous().view(CODES[kind])
            codes.view(torch.uint8)[a:b] = c.view(torch.uint8)
    return k, v, ks, vs


def _raw_cache(pages, case, gen):
    """All layers' caches, in one buffer each, with codes of any value (none of them NaN)."""
    kv, ps, d, n = case["kv_heads"], case["page"], case["dim"], case["layers"]
    codes = [torch.randint(0, 126, shape, dtype=torch.uint8, generator=gen, device=DEV)
             for shape in ((n, pages, kv, ps, d), (n, pages, kv, ps // 16, d, 16))]
    scales = [torch.rand(n, pages, kv, generator=gen, device=DEV) for _ in range(2)]
    return [c.view(CODES[case["codes"]]) for c in codes] + scales


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _prepare_attention(case, gen, s):
    family, prefix, behind, new = _attention_lengths(case)
    ps, R = case["page"], case["requests"]
    total = [p + b + n for p, b, n in zip(prefix, behind, new)]
    width = -(-max(total) // ps) + 3
    counts = [-(-t // ps) for t in total]
    pages = sum(counts) + 1
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    at, leader = 0, {}
    for r, c in enumerate(counts):
        same = prefix[r] // ps if family[r] in leader else 0
        if same:
            tables[r, :same] = tables[leader[family[r]], :same]
        leader.setdefault(family[r], r)
        tables[r, same:c] = order[at:at + c - same]
        at += c - same
    k, v, ks, vs = _filled_cache(at, case, gen)
    # pages are numbered as they are taken: a shuffled number among those that the cache holds
    rank = torch.argsort(torch.argsort(order[:at])).to(torch.int32)
    names = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    names[order[:at].long()] = rank
    tables = torch.where(tables >= 0, names[tables.clamp_min(0).long()], -1).to(torch.int32)
    q = 2 * torch.randn(sum(new), case["heads"], case["dim"], generator=gen, device=DEV)
    s.update(tables=tables.contiguous(), kv_lens=_int32(total), k=k, v=v, ks=ks, vs=vs,
             q_starts=_int32(np.concatenate([[0], np.cumsum(new)]).tolist()), q=q.to(TYPES[case["type"]]),
             least=256,  # positions that two requests share at least to be of one run
             max_q=max(new), max_kv=max(total), scale=1.0 / math.sqrt(case["dim"]))


def _prepare_pages(case, gen, s):
    ps, P, R = case["page"], case["parents"], case["requests"]
    lengths, parent, begins = _fork_lengths(case)
    held = [-(-n // ps) for n in lengths]
    width = max(held) + 4
    spare = R - P if case["op"] == "fork" else 2 * (R - P)
    pages = sum(held) + spare + 7
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    lens = lengths + [0] * (R - P)
    shares = torch.zeros(pages, dtype=torch.int32, device=DEV)
    at = 0
    for r, c in enumerate(held):
        tables[r, :c] = order[at:at + c]
        at += c
    if case["op"] == "compact":
        # the children are there: their own pages behind what they share
        for i, (p, n) in enumerate(zip(parent, begins)):
            full, extra = n // ps, -(-n // ps) - n // ps + 1
            extra = min(extra, width - full)
            tables[P + i, :full] = tables[p, :full]
            tables[P + i, full:full + extra] = order[at:at + extra]
            shares.scatter_add_(0, tables[p, :full].long(), torch.ones(full, dtype=torch.int32, device=DEV))
            at += extra
            lens[P + i] = ps * (full + extra) - i % ps
    ring = torch.zeros(pages, dtype=torch.int32, device=DEV)
    head = int(torch.randint(0, pages, (1,), generator=gen, device=DEV))
    ring[(torch.arange(pages - at, device=DEV) + head) % pages] = order[at:]
    k, v, ks, vs = _raw_cache(pages, case, gen)
    s.update(tables=tables, kv_lens=_int32(lens), free=ring, pool=_int32([head, pages - at, 0, 0]), shares=shares,
             k=k, v=v, ks=ks, vs=vs)
    if case["op"] == "fork":
        s.update(parents_of=_int32([-1] * P + parent), begins=_int32([0] * P + begins))
    else:
        s["done"] = torch.rand(R, generator=gen, device=DEV) < 0.6


def _prepare_logits(case, gen, s):
    R, V, L = case["requests"], case["vocab"], case["history"]
    r = random.Random(case["lens"])
    # tokens of a text: a few of them often, most of them seldom
    history = (V * torch.rand(R, L, generator=gen, device=DEV) ** 6).to(torch.int32).clamp_max(V - 1)
    spread = torch.randperm(V, generator=gen, device=DEV).to(torch.int32)
    history = spread[history.long()]
    lens = [L if i == 0 else r.randint(L // 3, L) for i in range(R)]
    prompts = [r.randint(0, n) for n in lens]
    u = torch.rand(3, R, generator=gen, device=DEV)
    s.update(logits=(3 * torch.randn(R, V, generator=gen, device=DEV)).to(TYPES[case["type"]]), tokens=history,
             token_lens=_int32(lens), prompt_lens=_int32(prompts), repetition=1 + 0.3 * u[0], presence=u[1].clone(),
             frequency=0.5 * u[2], ids=None, values=None, allowed=None, rows=None)
    if case["biases"]:
        n = min(case["biases"], V)
        ids = torch.stack([torch.randperm(V, generator=gen, device=DEV)[:n] for _ in range(R)]).to(torch.int32)
        count = _int32([r.randint(0, n) for _ in range(R)])
        s["ids"] = torch.where(torch.arange(n, device=DEV) < count[:, None], ids, -1).to(torch.int32)
        s["values"] = 4 * torch.randn(R, n, generator=gen, device=DEV)
    if case["grammars"]:
        words = -(-V // 32)
        dense = torch.rand(case["grammars"], 32 * words, generator=gen, device=DEV) < \
            torch.rand(case["grammars"], 1, generator=gen, device=DEV) ** 4
        weights = (1 << torch.arange(32, device=DEV, dtype=torch.int64))
        bits = (dense.view(-1, words, 32).long() * weights).sum(-1)
        s["allowed"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        s["rows"] = _int32([r.randint(-1, case["grammars"] - 1) for _ in range(R)])


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case)
    if case["op"] == "attention":
        _prepare_attention(case, gen, s)
    elif case["op"] in ("fork", "compact"):
        _prepare_pages(case, gen, s)
    else:
        _prepare_logits(case, gen, s)
    return s


# ---- plain forms ------------------------------------------------------------

def _bytes(cache):
    return cache.view(torch.uint8)


def _copy_pages(s, src, dst):
    """Pages of all layers, from src to dst (-1: no copy)."""
    some = (src >= 0) & (dst >= 0)
    a, b = src[some].long(), dst[some].long()
    for cache in (_bytes(s["k"]), _bytes(s["v"]), s["ks"], s["vs"]):
        cache[:, b] = cache[:, a]


def _plain_fork(s):
    ps, ring = s["page"], s["free"].numel()
    tables, lens = s["tables"].clone(), s["kv_lens"].long().clamp_min(0)
    R, width = tables.shape
    p = s["parents_of"].long()
    asked = (p >= 0) & (p < R) & (p != torch.arange(R, device=p.device))
    at = torch.where(asked, p, 0)
    begins = torch.where(asked, torch.minimum(s["begins"].long().clamp_min(0), lens[at].clamp_max(width * ps)), 0)
    empty = lens == 0
    full = begins // ps
    need = torch.where(asked & empty & (begins % ps > 0), 1, 0)
    upto = need.cumsum(0)
    head, count, refused = s["pool"][0].long(), s["pool"][1].long(), s["pool"][2].long()
    granted = asked & empty & ((need == 0) | (upto <= count))
    fresh = s["free"][(head + upto - need) % ring].long()
    j = torch.arange(width, device=p.device)[None]
    shared = granted[:, None] & (j < full[:, None])
    theirs = tables[at]
    taken = granted & (need > 0)
    src = torch.where(taken, theirs.gather(1, full.clamp_max(width - 1)[:, None])[:, 0].long(), -1)
    dst = torch.where(taken, fresh, -1)
    tables = torch.where(shared, theirs, tables)
    tables = torch.where(taken[:, None] & (j == full[:, None]), dst[:, None].to(torch.int32), tables)
    some = shared & (theirs >= 0) & (theirs < ring)
    shares = s["shares"].clone().scatter_add_(0, torch.where(some, theirs, 0).long().flatten(),
                                              some.to(torch.int32).flatten())
    n = taken.sum()
    pool = torch.stack([(head + n) % ring, count - n, refused + (asked & ~granted).sum(), torch.zeros_like(head)])
    _copy_pages(s, src, dst)
    return {"tables": tables, "kv_lens": torch.where(granted, begins, lens).to(torch.int32),
            "pool": pool.to(torch.int32), "shares": shares, "src": src.to(torch.int32), "dst": dst.to(torch.int32),
            **_codes(s)}


def _codes(s):
    # a copy changes no bit: codes and scales as they lie, as whole numbers
    return {"k": _bytes(s["k"]), "v": _bytes(s["v"]), "k_scale": s["ks"].view(torch.int32),
            "v_scale": s["vs"].view(torch.int32)}


def _plain_compact(s):
    ps, ring = s["page"], s["free"].numel()
    tables, lens, done = s["tables"], s["kv_lens"].long().clamp_min(0), s["done"]
    R, width = tables.shape
    j = torch.arange(width, device=tables.device)[None]
    held = j < ((lens + ps - 1) // ps)[:, None]
    some = held & (tables >= 0) & (tables < ring)
    # the finished requests' pages: those that nobody else owns are free
    gone = (some & done[:, None]).long().flatten()
    owners = torch.zeros(ring, dtype=torch.long, device=tables.device)
    owners.scatter_add_(0, torch.where(some, tables, 0).long().flatten(), gone)
    freed = owners > s["shares"]
    shares = torch.where(freed, 0, s["shares"] - owners)
    lens = torch.where(done, 0, lens)
    # the live pages to the front: the i-th of those behind it takes the i-th free one in it
    kept = (some & ~done[:, None]).long().flatten()
    live = torch.zeros(ring, dtype=torch.long, device=tables.device)
    live.scatter_add_(0, torch.where(some, tables, 0).long().flatten(), kept)
    live = live > 0
    n = live.sum()
    page = torch.arange(ring, device=tables.device)
    hole, mover = ~live & (page < n), live & (page >= n)
    most = ring // 2
    room = torch.full((ring + 1,), -1, dtype=torch.long, device=tables.device)
    dst = room.scatter(0, torch.where(hole, hole.cumsum(0) - 1, ring), page)[:most]
    src = room.scatter(0, torch.where(mover, mover.cumsum(0) - 1, ring), page)[:most]
    to = torch.where(mover, dst[(mover.cumsum(0) - 1).clamp(0, max(most - 1, 0))], page)
    tables = torch.where(some & ~done[:, None], to[tables.clamp(0, ring - 1).long()].to(torch.int32), tables)
    moved = torch.where(live & (page < n), shares, 0)
    at = torch.where(dst >= 0, dst, ring)
    moved = torch.cat([moved, moved[:1]]).scatter(0, at, shares[src.clamp_min(0)])[:ring]
    _copy_pages(s, src, dst)
    zero = torch.zeros_like(n)
    pool = torch.stack([zero, ring - n, s["pool"][2].long(), zero]).to(torch.int32)
    return {"tables": tables, "kv_lens": lens.to(torch.int32), "free": ((n + page) % ring).to(torch.int32),
            "pool": pool, "shares": moved.to(torch.int32), "src": src.to(torch.int32), "dst": dst.to(torch.int32),
            **_codes(s)}


def _plain_runs(s):
    """Where each run of requests with the same first pages begins, and how many positions a request shares."""
    ps, R = s["page"], len(s["kv_lens"])
    tables, lens = s["tables"], s["kv_lens"].long()
    new = (s["q_starts"][1:] - s["q_starts"][:-1]).long()
    whole = ((lens - new).clamp_min(0) // ps).clamp_max(tables.shape[1])
    j = torch.arange(tables.shape[1], device=tables.device)[None]
    same = (tables[1:] == tables[:-1]) & (tables[1:] >= 0) & (j < torch.minimum(whole[1:], whole[:-1])[:, None])
    common = torch.cat([whole.new_zeros(1), same.long().cumprod(1).sum(1)])  # with the request before
    begins = common < -(-s["least"] // ps)
    run = begins.long().cumsum(0) - 1
    least = torch.full((R,), 1 << 30, dtype=torch.long, device=tables.device)
    least = least.scatter_reduce(0, run, torch.where(begins, 1 << 30, common), "amin")
    shared = torch.where(least[run] < 1 << 30, least[run] * ps, 0)
    index = torch.arange(R, device=tables.device)
    starts = torch.full((R + 1,), R, dtype=torch.long, device=tables.device)
    starts = starts.scatter(0, torch.where(begins, run, R), torch.where(begins, index, R))
    return starts.to(torch.int32), shared.to(torch.int32)


def _plain_attention(s):
    h, kv, d, ps = s["heads"], s["kv_heads"], s["dim"], s["page"]
    q, lens, starts = s["q"], s["kv_lens"].long(), s["q_starts"].long()
    width = -(-s["max_kv"] // ps)
    bt = s["tables"][:, :width].long().clamp_min(0)
    R, L, n = len(lens), width * ps, s["max_q"]
    g = h // kv
    k = (_bytes(s["k"])[bt].view(s["k"].dtype).float() * s["ks"][bt][..., None, None]).transpose(1, 2)
    k = k.reshape(R, kv, L, d)
    v = _bytes(s["v"])[bt].view(s["v"].dtype).float() * s["vs"][bt][..., None, None, None]
    v = v.transpose(4, 5).transpose(1, 2).reshape(R, kv, L, d)
    t = torch.arange(n, device=q.device)
    count = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + t).clamp_max(len(q) - 1)
    rows = q[at].float().view(R, n, kv, g, d).transpose(1, 2).reshape(R, kv, n * g, d)
    scores = torch.matmul(rows, k.transpose(2, 3)) * s["scale"]
    limit = (lens - count)[:, None] + t  # the last position that a query sees
    seen = torch.arange(L, device=q.device) <= limit[..., None]
    scores.masked_fill_(~seen[:, None].repeat_interleave(g, 2), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = (scores - torch.where(top.isinf(), 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    o = o.view(R, kv, n, g, d).transpose(1, 2).reshape(R, n, h, d).to(q.dtype)
    token = torch.arange(len(q), device=q.device)
    r = torch.searchsorted(starts[1:], token, right=True)
    runs, shared = _plain_runs(s)
    return {"out": o[r, token - starts[r]], "starts": runs, "shared": shared}


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    j = torch.arange(s["tokens"].shape[1], device=x.device)[None]
    there = (j < s["token_lens"][:, None]) & (s["tokens"] >= 0) & (s["tokens"] < V)
    at = torch.where(there, s["tokens"], 0).long()
    seen = torch.zeros(R, V, device=x.device).scatter_add_(1, at, there.float())
    count = torch.zeros(R, V, device=x.device).scatter_add_(1, at, (there & (j >= s["prompt_lens"][:, None])).float())
    rho = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rho, x * rho), x)
    x = torch.where(count > 0, x - s["frequency"][:, None] * count - s["presence"][:, None], x)
    if s["ids"] is not None:
        some = (s["ids"] >= 0) & (s["ids"] < V)
        x = x.scatter_add(1, torch.where(some, s["ids"], 0).long(), torch.where(some, s["values"], 0.0))
    if s["allowed"] is not None:
        token = torch.arange(V, device=x.device)
        words = s["allowed"][s["rows"].clamp_min(0).long()][:, token // 32]
        ok = ((words >> (token % 32)) & 1 > 0) | (s["rows"] < 0)[:, None]
        x = x.masked_fill(~ok, float("-inf"))
    return x.to(s["logits"].dtype)


def _plain_greedy(s):
    # the lowest of the tokens with the largest logit
    x = _plain_logits(s)
    index = torch.arange(x.shape[1], device=x.device)
    return torch.where(x == x.amax(1, keepdim=True), index, x.shape[1]).amin(1)


def run(s):
    if own:
        import pare_amd as P

        if s["op"] in ("fork", "compact"):
            tables, lens, pool, shares = (s[name].clone() for name in ("tables", "kv_lens", "pool", "shares"))
            free = s["free"]
            if s["op"] == "fork":
                moves = P.fork_block_tables(tables, lens, s["parents_of"], free, pool, shares, s["page"],
                                            lengths=s["begins"])
            else:
                free = free.clone()
                P.release_block_tables(tables, lens, s["done"], free, pool, s["page"], shares=shares)
                moves = P.compact_block_tables(tables, lens, free, pool, shares, s["page"])
            P.copy_kv_pages(moves, s["k"], s["v"], s["ks"], s["vs"])
            out = {"tables": tables, "kv_lens": lens, "pool": pool, "shares": shares, "src": moves.src,
                   "dst": moves.dst, **_codes(s)}
            return out if s["op"] == "fork" else {**out, "free": free}
        if s["op"] == "attention":
            shared = P.shared_prefixes(s["tables"], s["kv_lens"], s["q_starts"], s["page"], least=s["least"])
            out = P.paged_attention(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["kv_lens"],
                                    s["q_starts"], scale=s["scale"], max_q_len=s["max_q"], max_kv_len=s["max_kv"],
                                    shared=shared)
            return {"out": out, "starts": shared.starts, "shared": shared.lens}
        call = P.process_logits if s["op"] == "logits" else P.greedy_tokens
        return call(s["logits"], history=s["tokens"], history_lens=s["token_lens"], prompt_lens=s["prompt_lens"],
                    repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                    bias_ids=s["ids"], bias=s["values"], allowed=s["allowed"], allowed_rows=s["rows"])
    return {"fork": _plain_fork, "compact": _plain_compact, "attention": _plain_attention, "logits": _plain_logits,
            "greedy": _plain_greedy}[s["op"]](s)


# ---- work -------------------------------------------------------------------

def _page_bytes(case):
    return case["layers"] * case["kv_heads"] * (2 * case["page"] * case["dim"] + 8)


def work(case):
    op, ps = case["op"], case.get("page")
    if op in ("logits", "greedy"):
        R, V = case["requests"], case["vocab"]
        r = random.Random(case["lens"])
        held = sum(case["history"] if i == 0 else r.randint(case["history"] // 3, case["history"]) for i in range(R))
        size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
        return {"bytes": R * V * size * (2 if op == "logits" else 1) + 4 * held + 8 * R * case["biases"]
                + case["grammars"] * (V + 7) // 8, "flops": 2 * R * V}
    if op in ("fork", "compact"):
        lengths, parent, begins = _fork_lengths(case)
        entries = sum(-(-n // ps) for n in begins)
        if op == "fork":
            partial = sum(n % ps > 0 for n in begins)
            return {"bytes": 2 * partial * _page_bytes(case) + 12 * entries, "flops": entries}
        # with six tenths of the requests gone about so many pages are live, spread evenly over all
        pages = sum(-(-n // ps) for n in lengths) + 2 * len(begins) + 7
        live = pages * 0.6
        return {"bytes": 2 * live * (1 - live / pages) * _page_bytes(case) + 8 * entries + 16 * pages, "flops": pages}
    family, prefix, behind, new = _attention_lengths(case)
    h, kv, d, tokens = case["heads"], case["kv_heads"], case["dim"], sum(new)
    pairs = sum(n * (p + b) + n * (n + 1) // 2 for p, b, n in zip(prefix, behind, new))
    first = {f: p // ps * ps for f, p in zip(family, prefix)}
    held = sum(first.values()) + sum(p + b + n - p // ps * ps for p, b, n in zip(prefix, behind, new))
    return {"bytes": 2 * kv * d * held + 8 * kv * (held // ps) + 4 * tokens * h * d, "flops": 4 * h * d * pairs}


# ---- the definitions in 64 bits ---------------------------------------------

def _exact_attention(s):
    h, kv, d, g = s["heads"], s["kv_heads"], s["dim"], s["heads"] // s["kv_heads"]
    out = torch.zeros(len(s["q"]), h, d, dtype=torch.float64, device=DEV)
    starts = s["q_starts"].tolist()
    for r, length in enumerate(s["kv_lens"].tolist()):
        a, b = starts[r], starts[r + 1]
        pages = s["tables"][r, :math.ceil(length / s["page"])].long()
        last = torch.arange(length - (b - a), length, device=DEV)[:, None]
        hidden = torch.arange(length, device=DEV)[None] > last
        k = _bytes(s["k"])[pages].view(s["k"].dtype).double() * s["ks"][pages].double()[..., None, None]
        v = _bytes(s["v"])[pages].view(s["v"].dtype).double().movedim(-1, -2).flatten(2, 3)
        v = v * s["vs"][pages].double()[..., None, None]
        k, v = (x.movedim(1, 0).flatten(1, 2)[:, :length].repeat_interleave(g, 0) for x in (k, v))
        e = torch.matmul(s["q"][a:b].double().movedim(1, 0), k.transpose(1, 2).contiguous()) * s["scale"]
        out[a:b] = torch.matmul(torch.softmax(e.masked_fill(hidden, -math.inf), 2), v).movedim(1, 0)
    return {"out": out, "starts": None, "shared": None}


def _exact_logits(s):
    """Row by row on the host, from the counts of the tokens."""
    rows = []
    for r, x in enumerate(s["logits"].double().cpu().numpy()):
        held = s["tokens"][r, :int(s["token_lens"][r])].cpu().numpy()
        said = held[int(s["prompt_lens"][r]):]
        seen, count = np.bincount(held, minlength=len(x)), np.bincount(said, minlength=len(x))
        rho, alpha, beta = (float(s[name][r]) for name in ("repetition", "presence", "frequency"))
        x = np.where(seen > 0, np.where(x > 0, x / rho, x * rho), x) - beta * count - alpha * (count > 0)
        if s["ids"] is not None:
            ids, values = s["ids"][r].cpu().numpy(), s["values"][r].double().cpu().numpy()
            np.add.at(x, ids[ids >= 0], values[ids >= 0])
        if s["allowed"] is not None and int(s["rows"][r]) >= 0:
            bits = np.unpackbits(s["allowed"][int(s["rows"][r])].cpu().numpy().view(np.uint8), bitorder="little")
            x = np.where(bits[:len(x)] > 0, x, -np.inf)
        rows.append(x)
    return torch.from_numpy(np.stack(rows))


def exact(case, seed):
    # (what a fork, a compaction and a greedy choice return has no rounding)
    if case["op"] in ("fork", "compact", "greedy"):
        return None
    return {"attention": _exact_attention, "logits": _exact_logits}[case["op"]](prepare(case, seed))
