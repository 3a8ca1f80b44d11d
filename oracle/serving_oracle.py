"""Plain implementations of serving in 8 bits, on the CPU: block tables, the paged
cache's write and read, attention over it, integer products.

Bookkeeping in Python integers. What is rounded to codes is computed twice: in fp32
with the kernels' definition (scale = max(old, amax * (1/top)), code = round(x * (1/scale))),
whose every step is one IEEE operation, so codes and scales can be held to its bits, and
attention and products in 64 bits from those codes. Test-only.
"""

from __future__ import annotations

import numpy as np
import torch

TOP = {torch.int8: np.float32(127.0), torch.float8_e4m3fn: np.float32(448.0)}
LARGEST = np.finfo(np.float32).max


def extend_tables(tables, kv_lens, new_lens, free_pages, pool, ps, total):
    """One request after another; tables (a copy) with its fresh entries, and the plan."""
    tables = [list(row) for row in tables]
    ring, width = len(free_pages), len(tables[0]) if tables else 0
    head, count, refused = pool[0], pool[1], pool[2]
    starts, lens, first, positions, slots, asked, taken, tokens = [0], [], [], [], [], 0, 0, 0
    for r, (length, new) in enumerate(zip(kv_lens, new_lens)):
        length, new = max(length, 0), max(new, 0)
        held, want = -(-length // ps), -(-(length + new) // ps)
        ok = want <= width
        need = want - held if ok else 0
        asked += need
        tokens += new
        ok = ok and (need == 0 or asked <= count) and (new == 0 or tokens <= total)
        if ok:
            for i in range(need):
                tables[r][held + i] = free_pages[(head + taken + i) % ring]
            taken += need
        else:
            refused += 1
        starts.append(min(starts[-1] + new, total))
        lens.append(length + new if ok else length)
        first.append(length if ok else -1)
        for i in range(new):
            if len(slots) < total:
                page = tables[r][(length + i) // ps] if ok else -1
                positions.append(length + i if ok else 0)
                slots.append(page * ps + (length + i) % ps if 0 <= page < ring else -1)
    rest = total - len(slots)
    pool = [(head + taken) % ring if ring else 0, count - taken, refused, 0]
    return tables, starts, lens, first, positions + [0] * rest, slots + [-1] * rest, pool


def encode(x: np.ndarray, dtype) -> np.ndarray:
    """fp32 x, already divided by its scale, as the bytes of the nearest codes."""
    if dtype == torch.int8:
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    return torch.from_numpy(np.clip(x, -448, 448).astype(np.float32)).to(dtype).view(torch.uint8).numpy()


def decode(codes: np.ndarray, dtype) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(codes)).view(dtype).to(torch.float32).numpy()


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """rotate_half of x [T, heads, D], each operation rounded to x's type."""
    d = x.shape[-1] // 2
    a, b, c, s = x[..., :d], x[..., d:], cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


class Cache:
    """Token-major codes uint8 [pages, KV, ps, D] and fp32 scales [pages, KV] of k and v."""

    def __init__(self, pages: int, KV: int, ps: int, D: int, dtype):
        self.ps, self.dtype = ps, dtype
        self.codes = [np.zeros((pages, KV, ps, D), np.uint8) for _ in range(2)]
        self.scales = [np.zeros((pages, KV), np.float32) for _ in range(2)]

    def append(self, qkv: np.ndarray, cos, sin, positions, slots, H: int) -> np.ndarray:
        """fp32 q rotated [T, H, D]; k and v of qkv (fp32 [T, (H + 2 KV) * D]) into the cache."""
        pages, KV, ps, D = self.codes[0].shape
        x = qkv.astype(np.float32).reshape(len(qkv), H + 2 * KV, D)
        turned = rotate(x[:, :H + KV], cos[positions], sin[positions])
        t = 0
        while t < len(slots):
            n = 1
            if not 0 <= slots[t] < pages * ps:
                t += 1
                continue
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % ps:
                n += 1
            page, at = slots[t] // ps, slots[t] % ps
            for i, new in enumerate((turned[t:t + n, H:], x[t:t + n, H + KV:])):
                for h in range(KV):
                    top = TOP[self.dtype]
                    old = self.scales[i][page, h] if at else np.float32(0)
                    want = np.abs(new[:, h]).max() * np.float32(np.float32(1) / top)
                    scale = np.maximum(old, want)
                    with np.errstate(over="ignore"):
                        inv = np.minimum(np.float32(1) / scale, LARGEST) if scale > 0 else np.float32(0)
                    cells = self.codes[i][page, h]
                    if at and scale > old:
                        cells[:at] = encode(decode(cells[:at], self.dtype) * np.float32(old / scale), self.dtype)
                    cells[at:at + n] = encode(new[:, h] * inv, self.dtype)
                    self.scales[i][page, h] = scale
            t += n
        return turned[:, :H]

    def fill(self, rng: np.random.Generator) -> None:
        """Every page full of keys and values of a model."""
        for i in range(2):
            x = rng.standard_normal(self.codes[i].shape, np.float32)
            x *= rng.uniform(0.25, 2.0, (x.shape[0], x.shape[1], 1, x.shape[3])).astype(np.float32)
            self.scales[i] = np.abs(x).max((2, 3)) * np.float32(np.float32(1) / TOP[self.dtype])
            self.codes[i] = encode(x / self.scales[i][..., None, None], self.dtype)

    def values(self, i: int) -> np.ndarray:
        return decode(self.codes[i], self.dtype).astype(np.float64) * self.scales[i][..., None, None]

    def tensors(self, device):
        """k_cache, v_cache, k_scale, v_scale as the operators take them."""
        k = torch.from_numpy(self.codes[0].copy()).to(device).view(self.dtype)
        p, kv, ps, d = self.codes[1].shape
        v = np.ascontiguousarray(self.codes[1].reshape(p, kv, ps // 16, 16, d).swapaxes(3, 4))
        return (k, torch.from_numpy(v).to(device).view(self.dtype),
                torch.from_numpy(self.scales[0].copy()).to(device), torch.from_numpy(self.scales[1].copy()).to(device))


def token_major(v_cache: torch.Tensor) -> np.ndarray:
    """The bytes of a v_cache tensor as [pages, KV, ps, D]."""
    v = v_cache.cpu().view(torch.uint8).numpy()
    p, kv, b, d, _ = v.shape
    return np.ascontiguousarray(v.swapaxes(3, 4)).reshape(p, kv, 16 * b, d)


def attention(q, k, v, tables, kv_lens, q_starts, ps, scale, window=0, max_kv=None):
    """(o, weight) in 64 bits: q [T, H, D] and the values k, v [pages, KV, ps, D]; weight =
    sum p |v|, what a relative error of the probabilities moves o by. Of a request of
    more keys than max_kv, or than its row of tables holds, the first ones. Rows behind
    the last request are NaN."""
    T, H, D = q.shape
    pages, KV = k.shape[:2]
    out, weight = np.full((T, H, D), np.nan), np.full((T, H, D), np.nan)
    for r, length in enumerate(kv_lens):
        a, b = q_starts[r], q_starts[r + 1]
        length, n = max(length, 0), b - a
        bound = tables.shape[1] * ps if max_kv is None else min(max_kv, tables.shape[1] * ps)
        for i in range(n):
            last = length - n + i
            p = np.arange(max(0, last - window + 1) if window else 0, min(last + 1, bound))
            page = tables[r, p // ps] if len(p) else np.zeros(0, int)
            p, page = p[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
            for h in range(H):
                if not len(p):
                    out[a + i, h] = weight[a + i, h] = 0
                    continue
                kk, vv = k[page, h // (H // KV), p % ps], v[page, h // (H // KV), p % ps]
                s = kk @ q[a + i, h].astype(np.float64) * scale
                e = np.exp(s - s.max())
                out[a + i, h] = e @ vv / e.sum()
                weight[a + i, h] = e @ np.abs(vv) / e.sum()
    return out, weight


def quantize_rows(x: np.ndarray):
    """codes int8 [M, K], scales fp32 [M] of fp32 rows, one IEEE operation at a time."""
    amax = np.abs(x).max(1).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(amax > 0, np.minimum(np.float32(127) / amax, LARGEST), np.float32(0)).astype(np.float32)
    return np.clip(np.rint(x * inv[:, None]), -127, 127).astype(np.int8), amax * np.float32(np.float32(1) / np.float32(127))


def matmul_w8a8(cx, sx, cw, sw, bias=None):
    y = (cx.astype(np.float64) @ cw.astype(np.float64).T) * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    return y if bias is None else y + bias.astype(np.float64)
