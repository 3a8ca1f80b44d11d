"""Plain implementations of what requests from one prompt need, on the CPU: pages with
several owners, runs of requests with the same first pages, and processed logits. One request,
one page, one token after another, in Python integers and 64 bits. Test-only.
"""

from __future__ import annotations

import numpy as np


def fork(tables, kv_lens, parents, lengths, free_pages, pool, shares, ps):
    """(tables, kv_lens, pool, shares, src, dst), all new."""
    before, R, ring = [list(row) for row in tables], len(kv_lens), len(free_pages)
    tables, lens, shares = [list(row) for row in tables], list(kv_lens), list(shares)
    width = len(tables[0]) if R else 0
    head, count, refused = pool[0], pool[1], pool[2]
    if not 0 <= head < ring:
        head = 0
    count = min(max(count, 0), ring)
    asked = taken = 0
    src, dst = [-1] * R, [-1] * R
    for r, p in enumerate(parents):
        if not 0 <= p < R or p == r:
            continue
        n = min(max(kv_lens[p], 0), width * ps)
        if lengths is not None:
            n = min(n, max(lengths[r], 0))
        if kv_lens[r] > 0:
            refused += 1
            continue
        if n % ps:
            asked += 1
            if asked > count:
                refused += 1
                continue
            taken += 1
            src[r] = before[p][n // ps]
            dst[r] = tables[r][n // ps] = free_pages[(head + asked - 1) % ring]
        for j in range(n // ps):
            tables[r][j] = before[p][j]
            if 0 <= before[p][j] < ring:
                shares[before[p][j]] += 1
        lens[r] = n
    return tables, lens, [(head + taken) % ring if ring else 0, count - taken, refused, 0], shares, src, dst


def release(tables, kv_lens, done, free_pages, pool, shares, ps):
    """(kv_lens, free_pages, pool, shares), all new."""
    lens, free, shares, ring = list(kv_lens), list(free_pages), list(shares), len(free_pages)
    left = set()
    for r, d in enumerate(done):
        if not d:
            continue
        for page in tables[r][:-(-max(lens[r], 0) // ps)]:
            if 0 <= page < ring:
                shares[page] -= 1
                if shares[page] < 0:
                    left.add(page)
        lens[r] = 0
    for i, page in enumerate(sorted(left)):
        free[(pool[0] + pool[1] + i) % ring] = page
        shares[page] = 0
    return lens, free, [pool[0], pool[1] + len(left), *pool[2:]], shares


def compact(tables, kv_lens, pool, shares, ps):
    """(tables, free_pages, pool, shares, src, dst) of len(shares) pages, all new."""
    pages = len(shares)
    held = [min(-(-max(n, 0) // ps), len(row)) for row, n in zip(tables, kv_lens)]
    live = sorted({p for row, h in zip(tables, held) for p in row[:h] if 0 <= p < pages})
    n = len(live)
    moved = dict(zip([p for p in live if p >= n], [p for p in range(n) if p not in set(live)]))
    tables = [[moved.get(p, p) if j < h else p for j, p in enumerate(row)] for row, h in zip(tables, held)]
    owners = [0] * pages
    for p in live:
        owners[moved.get(p, p)] = shares[p]
    pad = [-1] * (pages // 2 - len(moved))
    return (tables, [(n + i) % pages for i in range(pages)], [0, pages - n, pool[2], 0], owners,
            list(moved) + pad, list(moved.values()) + pad)


def runs(tables, kv_lens, q_starts, ps, least):
    """(starts [R + 1], lens [R], runs [R][4])."""
    R = len(kv_lens)
    groups, last = [], None
    for r in range(R):
        n = 1 if q_starts is None else max(q_starts[r + 1] - q_starts[r], 0)
        if kv_lens[r] <= 0 or n == 0:
            continue
        whole = min(max(kv_lens[r] - n, 0) // ps, len(tables[r]))
        common = 0
        if last is not None:
            while common < min(whole, last[1]) and tables[r][common] == tables[last[0]][common] >= 0:
                common += 1
        if common * ps < least:
            groups.append([r, []])
        else:
            groups[-1][1].append((r, common))
        last = (r, whole)
    lens = [0] * R
    for first, members in groups:
        for r in [first] + [m for m, _ in members] if members else []:
            lens[r] = ps * min(c for _, c in members)
    starts = [g[0] for g in groups] + [R] * (R + 1 - len(groups))
    rows = [[0] * 4 for _ in range(R)]
    for i, (first, members) in enumerate(groups):
        if members:
            a, b = (first, starts[i + 1]) if q_starts is None else (q_starts[first], q_starts[starts[i + 1]])
            rows[i] = [first, a, b - a, lens[first]]
    return starts, lens, rows


def logits(x, history, history_lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, rows):
    """(processed, magnitude) in 64 bits of x [R, V]: magnitude is the sum of what a logit is made
    of, on which fp32's roundings on the way are counted. Arguments as numpy arrays or None."""
    x = np.asarray(x, np.float64)
    R, V = x.shape
    out, size = x.copy(), np.abs(x)
    for r in range(R):
        if history is not None:
            n = history.shape[1] if history_lens is None else min(max(int(history_lens[r]), 0), history.shape[1])
            prompt = 0 if prompt_lens is None else int(prompt_lens[r])
            count = {}
            for i, t in enumerate(history[r, :n].tolist()):
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + (i >= prompt)
            for t, c in count.items():
                rho = 1.0 if repetition is None else float(repetition[r])
                with np.errstate(invalid="ignore"):
                    v = x[r, t] / rho if x[r, t] > 0 else x[r, t] * rho
                a = 0.0 if presence is None else float(presence[r])
                b = 0.0 if frequency is None else float(frequency[r])
                out[r, t] = v - (b * c + a if c else 0)
                size[r, t] = abs(v) + (abs(b) * c + abs(a) if c else 0)
        if bias_ids is not None:
            for t, b in zip(bias_ids[r].tolist(), bias[r].tolist()):
                if 0 <= t < V:
                    out[r, t] += b
                    size[r, t] += abs(b)
        if allowed is not None:
            m = r if rows is None else int(rows[r])
            if 0 <= m < len(allowed):
                bits = np.unpackbits(np.ascontiguousarray(allowed[m]).view(np.uint8), bitorder="little")[:V]
                out[r, bits == 0] = -np.inf
    return out, size
