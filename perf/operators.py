"""The operators of serving in 8 bits, as cases to be timed and compared.

Four operators: block tables and slot maps from request lengths (``tables``), RoPE and the
write into a paged cache of 8-bit keys and values (``append``), attention over that cache
(``attention``), and a linear layer in 8-bit integers (``w8a8``). With ``own`` false
``run`` computes them from elementary torch operations, with ``own`` true it calls pare_amd.

The cache: ``k_cache`` int8 or float8_e4m3fn [pages, kv_heads, page_size, D], ``v_cache`` of
the same type [pages, kv_heads, page_size / 16, D, 16] (token 16 b + j of a page at [b, :, j]),
and one fp32 scale per page and head for each of them; a value is its code times that scale.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}  # the largest code


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # the bookkeeping of one decode step: latency alone
        dict(name="tables_decode", op="tables", requests=48, longest=4096, newest=1, page=64, lens=1),
        # a scheduler's step that admits many prompts at once, small pages
        dict(name="tables_admit", op="tables", requests=700, longest=900, newest=700, page=16, lens=2),
        # one new token for each of 64 sequences of an 8B decoder (32 / 8 heads of 128)
        dict(name="append_decode", op="append", requests=64, past=4000, newest=1, heads=32, kv_heads=8, dim=128,
             page=64, codes="int8", type="fp16", lens=3),
        # ragged prompts of a 7B decoder with 28 / 4 heads, odd lengths, bf16 and fp8
        dict(name="append_prompts", op="append", requests=7, past=0, newest=1777, heads=28, kv_heads=4, dim=128,
             page=32, codes="fp8", type="bf16", lens=4),
        # one short chat: the smallest attention call
        dict(name="attn_decode_one", op="attention", requests=1, past=700, newest=1, heads=32, kv_heads=8, dim=128,
             page=64, codes="int8", type="fp16", window=0, lens=5),
        # a serving batch of ragged sequences, one token each
        dict(name="attn_decode_batch", op="attention", requests=64, past=8191, newest=1, heads=32, kv_heads=8,
             dim=128, page=64, codes="int8", type="fp16", window=0, lens=6),
        # two very long documents
        dict(name="attn_decode_long", op="attention", requests=2, past=131000, newest=1, heads=28, kv_heads=4,
             dim=128, page=128, codes="fp8", type="bf16", window=0, lens=7),
        # ragged prompts read in one pass
        dict(name="attn_prompts", op="attention", requests=5, past=0, newest=2048, heads=32, kv_heads=8, dim=128,
             page=64, codes="int8", type="fp16", window=0, lens=8),
        # chunks of prompts behind long contexts, heads of 64, a sliding window
        dict(name="attn_chunks", op="attention", requests=3, past=15000, newest=500, heads=16, kv_heads=2, dim=64,
             page=16, codes="fp8", type="bf16", window=4096, lens=9),
        # the output head of an 8B decoder for one token: the weights' bytes
        dict(name="w8a8_head_one", op="w8a8", m=1, n=128256, k=4096, type="fp16", bias=False),
        # a decode batch of odd size through an output of odd size
        dict(name="w8a8_batch", op="w8a8", m=37, n=14335, k=4096, type="bf16", bias=True),
        # prompts through the gate and up projections of an 8B decoder: the largest product
        dict(name="w8a8_prompts", op="w8a8", m=4099, n=28672, k=4096, type="fp16", bias=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "w8a8", "w8a8"])
    seed = rng.randrange(1 << 20)
    if op == "tables":
        newest = _log(rng, 1, 700)
        return dict(op=op, requests=_log(rng, 1, 700), longest=newest + _log(rng, 1, 4000), newest=newest,
                    page=rng.choice([16, 32, 64, 128]), lens=seed)
    if op == "w8a8":
        m, k = _log(rng, 1, 4099), 16 * _log(rng, 4, 512)
        n = _log(rng, 8, 128256)
        n = max(8, min(n, 4099 * 28672 * 4096 // (m * k), 128256 * 4096 // k))
        return dict(op=op, m=m, n=n, k=k, type=rng.choice(["fp16", "bf16"]), bias=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8] if kv <= 4 else [1, 2, 4])
    common = dict(heads=heads, kv_heads=kv, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                  codes=rng.choice(["int8", "fp8"]), type=rng.choice(["fp16", "bf16"]), lens=seed)
    if op == "append":
        if rng.random() < 0.5:
            return dict(op=op, requests=_log(rng, 1, 128), past=_log(rng, 1, 4000), newest=1, **common)
        return dict(op=op, requests=rng.randint(1, 7), past=rng.choice([0, _log(rng, 1, 500)]),
                    newest=_log(rng, 2, 1777), **common)
    window = rng.choice([0, 0, _log(rng, 64, 4096)])
    if rng.random() < 0.6:
        past = _log(rng, 1, 131000)
        return dict(op=op, requests=min(_log(rng, 1, 64), max(1, 64 * 8191 // past)), past=past, newest=1,
                    window=window, **common)
    newest = _log(rng, 2, 2048)
    return dict(op=op, requests=rng.randint(1, 5), past=rng.choice([0, _log(rng, 1, 2048)]), newest=newest,
                window=window, **common)


def _lengths(case):
    """(past, new) of each request, from the case alone; the first has the longest."""
    r, n = random.Random(case["lens"]), case["requests"]
    longest = case["longest"] - case["newest"] if case["op"] == "tables" else case["past"]
    past = [longest if i == 0 else r.randint(longest // 4, longest) for i in range(n)]
    new = [case["newest"] if i == 0 else r.randint(max(1, case["newest"] // 8), case["newest"]) for i in range(n)]
    return past, new


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


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _paged(case, gen):
    """Block tables over shuffled pages, and the lengths after the new tokens."""
    past, new = _lengths(case)
    ps = case["page"]
    total = [p + n for p, n in zip(past, new)]
    width = -(-max(total) // ps)
    counts = [-(-t // ps) for t in total]
    pages = sum(counts) + 1
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    rows = torch.zeros(len(total), width, dtype=torch.int32, device=DEV)
    at = 0
    for r, c in enumerate(counts):
        rows[r, :c] = order[at:at + c]
        at += c
    return past, new, pages, rows, _int32(total), _int32(np.concatenate([[0], np.cumsum(new)]).tolist())


def prepare(case, seed):
    gen = _generator(seed)
    op, s = case["op"], dict(case)
    if op == "tables":
        past, new = _lengths(case)
        ps = case["page"]
        held = [-(-p // ps) for p in past]
        width = -(-(max(past) + max(new)) // ps) + 2
        pages = sum(-(-(p + n) // ps) for p, n in zip(past, new)) + 16
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        tables = torch.full((len(past), width), -1, dtype=torch.int32, device=DEV)
        at = 0
        for r, c in enumerate(held):
            tables[r, :c] = order[at:at + c]
            at += c
        free = torch.zeros(pages, dtype=torch.int32, device=DEV)  # a ring: head, count in `pool`
        head = int(torch.randint(0, pages, (1,), generator=gen, device=DEV))
        free[(torch.arange(pages - at, device=DEV) + head) % pages] = order[at:]
        s.update(tables=tables, kv_lens=_int32(past), new_lens=_int32(new), free=free,
                 pool=_int32([head, pages - at, 0, 0]), total=sum(new))
        return s
    if op == "w8a8":
        w = torch.empty(case["n"], case["k"], dtype=torch.int8, device=DEV)
        ws = torch.empty(case["n"], dtype=torch.float32, device=DEV)
        for a in range(0, case["n"], 16384):
            x = torch.randn(min(16384, case["n"] - a), case["k"], generator=gen, device=DEV) * 0.02
            amax = x.abs().amax(1)
            ws[a:a + 16384] = amax * (1.0 / 127.0)
            w[a:a + 16384] = (x * (127.0 / amax)[:, None]).round().to(torch.int8)
        t = TYPES[case["type"]]
        x = torch.randn(case["m"], case["k"], generator=gen, device=DEV)
        x *= 0.3 + 3 * torch.rand(case["k"], generator=gen, device=DEV) ** 8  # a few large channels
        bias = (torch.randn(case["n"], generator=gen, device=DEV)).to(t) if case["bias"] else None
        s.update(x=x.to(t), w=w, ws=ws, bias_values=bias)
        return s
    past, new, pages, tables, kv_lens, q_starts = _paged(case, gen)
    t = TYPES[case["type"]]
    k, v, ks, vs = _filled_cache(pages, case, gen)
    s.update(tables=tables, kv_lens=kv_lens, q_starts=q_starts, k=k, v=v, ks=ks, vs=vs,
             max_q=max(new), max_kv=max(p + n for p, n in zip(past, new)))
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "append":
        positions = torch.cat([torch.arange(p, p + n, device=DEV) for p, n in zip(past, new)])
        request = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
        page = tables[request, positions // case["page"]]
        s["slots"] = (page * case["page"] + positions % case["page"]).to(torch.int32)
        s["positions"] = positions.to(torch.int32)
        s["pages"] = torch.unique(page).to(torch.int32)  # what the tokens go to
        # keys grow with some channels; the last tokens are a little larger than a page's first
        x = torch.randn(len(positions), h + 2 * kv, d, generator=gen, device=DEV)
        s["qkv"] = (x * (0.5 + torch.rand(1, h + 2 * kv, d, generator=gen, device=DEV))).to(t).flatten(1)
        inv = 1.0 / 500000.0 ** (torch.arange(0, d, 2, device=DEV).double() / d)
        angle = torch.arange(max(p + n for p, n in zip(past, new)), device=DEV).double()[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["q"] = (2 * torch.randn(sum(new), h, d, generator=gen, device=DEV)).to(t)
    s["scale"] = 1.0 / math.sqrt(d)
    return s


# ---- plain forms ------------------------------------------------------------

def _plain_tables(s):
    ps, ring = s["page"], s["free"].numel()
    tables = s["tables"]
    width = tables.shape[1]
    old, new = s["kv_lens"].long().clamp_min(0), s["new_lens"].long().clamp_min(0)
    head, count, refused = s["pool"][0].long(), s["pool"][1].long(), s["pool"][2].long()
    held, wanted = (old + ps - 1) // ps, (old + new + ps - 1) // ps
    fits = wanted <= width
    need = torch.where(fits, wanted - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= count))
    j = torch.arange(width, device=tables.device)[None]
    fresh = granted[:, None] & (j >= held[:, None]) & (j < wanted[:, None])
    at = (head + (upto - need)[:, None] + j - held[:, None]) % ring
    tables.copy_(torch.where(fresh, s["free"][at], tables))
    taken = torch.where(granted, need, 0).sum()
    pool = torch.stack([(head + taken) % ring, count - taken, refused + (~granted).sum(),
                        torch.zeros_like(head)]).to(torch.int32)
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    t = torch.arange(s["total"], device=tables.device)
    r = torch.searchsorted(starts[1:], t, right=True).clamp_max(len(new) - 1)
    live = (t < starts[-1]) & granted[r]
    pos = torch.where(live, old[r] + t - starts[r], 0)
    slots = torch.where(live, tables[r, pos // ps].long() * ps + pos % ps, -1)
    return {"tables": tables, "q_starts": starts.to(torch.int32),
            "kv_lens": torch.where(granted, old + new, old).to(torch.int32),
            "positions": pos.to(torch.int32), "slots": slots.to(torch.int32), "pool": pool}


def _floats(codes):
    return codes.float()


def _pick(cache, pages):
    """Pages of a cache, by their bytes: 8-bit floats cannot be indexed everywhere."""
    return cache.view(torch.uint8)[pages].view(cache.dtype)


def _put(cache, pages, values):
    cache.view(torch.uint8)[pages] = values.view(torch.uint8)


def _coded(x, kind):
    return x.round().clamp(-127, 127).to(torch.int8) if kind == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(s):
    h, kv, d, ps, kind = s["heads"], s["kv_heads"], s["dim"], s["page"], s["codes"]
    x = s["qkv"].view(-1, h + 2 * kv, d).float()
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    # the touched pages, each with its old tokens and its new ones
    pages = s["pages"].long()
    where = torch.searchsorted(pages, s["slots"].long() // ps)
    off = s["slots"].long() % ps
    fresh = torch.zeros(len(pages), ps, dtype=torch.bool, device=x.device)
    fresh[where, off] = True
    first = torch.where(fresh, torch.arange(ps, device=x.device), ps).amin(1)
    old = torch.arange(ps, device=x.device)[None] < first[:, None]
    out = [turned[:, :h].to(s["qkv"].dtype)]
    for cache, scales, values in ((s["k"], s["ks"], turned[:, h:]), (s["v"], s["vs"], x[:, h + kv:])):
        held = _floats(_pick(cache, pages))
        if cache.dim() == 5:
            held = held.transpose(3, 4).reshape(len(pages), kv, ps, d)
        new = torch.zeros_like(held).transpose(1, 2).contiguous()
        new[where, off] = values
        new = new.transpose(1, 2)
        amax = new.abs().amax((2, 3))
        before = torch.where((first > 0)[:, None], scales[pages], 0.0)
        scale = torch.maximum(before, amax * (1.0 / TOP[kind]))
        grown = scale > before
        factor = torch.where(grown, before / scale, 1.0)
        inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
        codes = torch.where(fresh[:, None, :, None], new * inverse[..., None, None], held)
        again = old[:, None, :, None] & grown[..., None, None]
        codes = _coded(torch.where(again, held * factor[..., None, None], codes), kind)
        stored = codes
        if cache.dim() == 5:
            stored = codes.view(torch.uint8).reshape(len(pages), kv, ps // 16, 16, d).transpose(3, 4).contiguous().view(cache.dtype)
        _put(cache, pages, stored)
        scales[pages] = scale
        out.append((_floats(codes) * scale[..., None, None]).to(s["qkv"].dtype))
    return out


def _plain_attention(s):
    h, kv, d, ps = s["heads"], s["kv_heads"], s["dim"], s["page"]
    q, lens, starts = s["q"], s["kv_lens"].long(), s["q_starts"].long()
    width = -(-s["max_kv"] // ps)
    bt = s["tables"][:, :width].long()
    R, L, n = len(lens), width * ps, s["max_q"]
    g = h // kv
    k = (_floats(_pick(s["k"], bt)) * s["ks"][bt][..., None, None]).transpose(1, 2).reshape(R, kv, L, d)
    v = _floats(_pick(s["v"], bt)) * s["vs"][bt][..., None, None, None]
    v = v.transpose(4, 5).transpose(1, 2).reshape(R, kv, L, d)
    t = torch.arange(n, device=q.device)
    count = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + t).clamp_max(len(q) - 1)
    rows = q[at].float().view(R, n, kv, g, d).transpose(1, 2).reshape(R, kv, n * g, d)
    scores = torch.matmul(rows, k.transpose(2, 3)) * s["scale"]
    limit = (lens - count)[:, None] + t  # the last position that a query sees
    p = torch.arange(L, device=q.device)
    seen = p <= limit[..., None]
    if s["window"]:
        seen &= p > limit[..., None] - s["window"]
    seen = seen[:, None].repeat_interleave(g, 2)
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = (scores - torch.where(top.isinf(), 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    o = o.view(R, kv, n, g, d).transpose(1, 2).reshape(R, n, h, d).to(q.dtype)
    if n == 1:
        return o[:, 0]
    token = torch.arange(len(q), device=q.device)
    r = torch.searchsorted(starts[1:], token, right=True)
    return o[r, token - starts[r]]


def _plain_w8a8(s):
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    codes = (x * torch.where(amax > 0, 127.0 / amax, 0.0)).round()
    y = torch.matmul(codes, s["w"].float().t()) * (amax * (1.0 / 127.0)) * s["ws"]
    if s["bias_values"] is not None:
        y = y + s["bias_values"].float()
    return y.to(s["x"].dtype)


def run(s):
    if own:
        import pare_amd as P

        if s["op"] == "tables":
            plan = P.extend_block_tables(s["tables"], s["kv_lens"], s["new_lens"], s["free"], s["pool"], s["page"],
                                         s["total"])
            return {"tables": s["tables"], "q_starts": plan.q_starts, "kv_lens": plan.kv_lens,
                    "positions": plan.positions, "slots": plan.slots, "pool": plan.pool}
        if s["op"] == "append":
            q = P.rope_append_kv(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["k"], s["v"],
                                 s["ks"], s["vs"])
            k, v = P.read_kv_pages(s["pages"], s["k"], s["v"], s["ks"], s["vs"], dtype=s["qkv"].dtype)
            return [q, k, v]
        if s["op"] == "attention":
            return P.paged_attention(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["kv_lens"],
                                     s["q_starts"], scale=s["scale"], window=s["window"], max_q_len=s["max_q"],
                                     max_kv_len=s["max_kv"])
        return P.matmul_w8a8(s["x"], s["w"], s["ws"], bias=s["bias_values"])
    if s["op"] == "tables":
        return _plain_tables(s)
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attention":
        return _plain_attention(s)
    return _plain_w8a8(s)


# ---- work -------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "w8a8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + 4 * n + 2 * m * (n + k) + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    past, new = _lengths(case)
    ps, tokens = case["page"], sum(new)
    if op == "tables":
        fresh = sum(-(-(p + n) // ps) + -p // ps for p, n in zip(past, new))
        return {"bytes": 16 * len(past) + 8 * tokens + 8 * fresh, "flops": 8 * tokens}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "append":
        # the new rows in, the turned queries out, codes in and out of the touched pages, and their values
        touched = sum(-(-(p + n) // ps) - p // ps for p, n in zip(past, new))
        codes = 2 * kv * d * (tokens + touched * ps)
        return {"bytes": 2 * tokens * (2 * h + 2 * kv) * d + codes + 4 * kv * d * touched * ps, "flops": 8 * tokens * (h + 2 * kv) * d}
    w, pairs, held = case["window"], 0, 0
    for p, n in zip(past, new):
        if w:
            pairs += sum(min(w, p + i + 1) for i in range(n))
            held += min(p + n, w + n - 1)
        else:
            pairs += n * p + n * (n + 1) // 2
            held += p + n
    return {"bytes": 2 * kv * d * held + 8 * kv * (held // ps) + 4 * tokens * h * d, "flops": 4 * h * d * pairs}


# ---- the definitions in 64 bits ---------------------------------------------

def _exact_tables(s):
    """By the definition, one request after another, on the host."""
    ps, ring = s["page"], s["free"].numel()
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
    head, count, refused = (int(v) for v in s["pool"].cpu()[:3])
    asked, lens, starts, positions, slots = 0, [], [0], [], []
    taken = 0
    for r, (old, new) in enumerate(zip(s["kv_lens"].tolist(), s["new_lens"].tolist())):
        held, wanted = math.ceil(old / ps), math.ceil((old + new) / ps)
        starts.append(starts[-1] + new)
        ok = wanted <= tables.shape[1]
        need = wanted - held if ok else 0
        asked += need
        ok = ok and (need == 0 or asked <= count)
        if ok:
            for i in range(need):
                tables[r, held + i] = free[(head + asked - need + i) % ring]
            taken += need
        refused += not ok
        lens.append(old + new if ok else old)
        for i in range(new):
            positions.append(old + i if ok else 0)
            slots.append(int(tables[r, (old + i) // ps]) * ps + (old + i) % ps if ok else -1)
    values = {"tables": tables, "q_starts": starts, "kv_lens": lens, "positions": positions, "slots": slots,
              "pool": [(head + taken) % ring, count - taken, refused, 0]}
    return {name: torch.tensor(np.asarray(v), dtype=torch.int32) for name, v in values.items()}


def _page64(s, cache, scales, page):
    """Values of one or several pages in 64 bits, [.., heads, tokens, D]."""
    c = _pick(cache, page).double()
    if cache.dim() == 5:
        c = c.movedim(-1, -2).flatten(-3, -2)
    return c * scales[page].double()[..., None, None]


def _exact_append(s):
    h, kv, d, ps, kind = s["heads"], s["kv_heads"], s["dim"], s["page"], s["codes"]
    x = s["qkv"].double().unflatten(1, (h + 2 * kv, d))
    c, sn = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    z = torch.complex(x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:]) * torch.complex(c, sn)[:, None]
    turned = torch.cat([z.real, z.imag], 2)
    slots, out = s["slots"].tolist(), [turned[:, :h]]
    tokens = {}
    for t, slot in enumerate(slots):
        tokens.setdefault(slot // ps, []).append(t)
    pages = s["pages"].tolist()
    for cache, scales, new in ((s["k"], s["ks"], turned[:, h:]), (s["v"], s["vs"], x[:, h + kv:])):
        codes = _pick(cache, s["pages"].long()).double()
        if cache.dim() == 5:
            codes = codes.movedim(-1, -2).flatten(-3, -2)
        scale = scales[s["pages"].long()].double()
        values = torch.empty_like(codes)
        for i, page in enumerate(pages):
            t = tokens[page]
            first = slots[t[0]] % ps
            mine = new[t[0]:t[-1] + 1].transpose(0, 1)
            before = scale[i] if first else torch.zeros_like(scale[i])
            after = torch.maximum(before, mine.abs().amax((1, 2)) / TOP[kind])
            full = codes[i].clone()
            if first:
                again = _coded(full[:, :first] * (before / after)[:, None, None], kind).double()
                full[:, :first] = torch.where((after > before)[:, None, None], again, full[:, :first])
            full[:, first:first + len(t)] = _coded(mine / after[:, None, None], kind).double()
            values[i] = full * after[:, None, None]
        out.append(values)
    return out


def _exact_attention(s):
    h, kv, d, g = s["heads"], s["kv_heads"], s["dim"], s["heads"] // s["kv_heads"]
    out = torch.zeros(len(s["q"]), h, d, dtype=torch.float64, device=DEV)
    starts = s["q_starts"].tolist()
    for r, length in enumerate(s["kv_lens"].tolist()):
        a, b = starts[r], starts[r + 1]
        pages = s["tables"][r, :math.ceil(length / s["page"])].long()
        last = torch.arange(length - (b - a), length, device=DEV)[:, None]
        p = torch.arange(length, device=DEV)[None]
        hidden = (p > last) | ((p <= last - s["window"]) if s["window"] else False)
        for j in range(kv):
            k = _page64(s, s["k"][:, j:j + 1], s["ks"][:, j:j + 1], pages).flatten(0, 2)[:length]
            v = _page64(s, s["v"][:, j:j + 1], s["vs"][:, j:j + 1], pages).flatten(0, 2)[:length]
            for i in range(j * g, (j + 1) * g):
                e = s["q"][a:b, i].double() @ k.t() * s["scale"]
                out[a:b, i] = torch.softmax(e.masked_fill(hidden, -math.inf), 1) @ v
    return out


def _exact_w8a8(s):
    x = s["x"].double()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.round(x / torch.where(top > 0, top, 1.0) * 127)
    y = torch.empty(len(x), len(s["w"]), dtype=torch.float64, device=DEV)
    for a in range(0, len(s["w"]), 16384):
        y[:, a:a + 16384] = codes @ s["w"][a:a + 16384].double().t() * s["ws"][a:a + 16384].double()
    y *= top / 127
    return y if s["bias_values"] is None else y + s["bias_values"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "attention": _exact_attention,
            "w8a8": _exact_w8a8}[case["op"]](s)
