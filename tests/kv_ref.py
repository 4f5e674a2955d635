"""Plain 64-bit forms of the cached-attention operators (CPU), written from the definitions in include/pgt_hip.h."""
import math

import torch

E_MIN, E_MAX = -32, 32


def rope(x, heads, pos, freqs, gain, eps, inter):
    """x (rows, heads * hd) float64 -> normed and turned, float64 (differentiable)"""
    rows = x.shape[0]
    x = x.reshape(rows, heads, -1)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if gain is not None:
        y = y * gain
    if freqs is not None and freqs.numel():
        rot = 2 * freqs.numel()
        a = 2 * math.pi * torch.remainder(pos.double()[:, None] * freqs, 1.0)
        c, s = a.cos()[:, None], a.sin()[:, None]
        i = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
        j = i + 1 if inter else i + rot // 2
        z = y.clone()
        z[..., i] = y[..., i] * c - y[..., j] * s
        z[..., j] = y[..., j] * c + y[..., i] * s
        y = z
    return y.reshape(rows, -1)


def exponent(amax):
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def e4m3(x):
    """float64 -> nearest e4m3 value, ties to even, saturating; NaN stays"""
    x = x.clamp(-448.0, 448.0)      # clamp keeps NaN
    mag = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(mag)) - 3)
    return torch.round(x / step) * step


class Cache:
    """values[w] (pages, page, kv, hd) float64 (of the codes, scale taken out) and exponents[w] (pages, kv)"""

    def __init__(self, pages, kv, page, hd):
        self.page, self.pages = page, pages
        self.code = [torch.zeros((pages, page, kv, hd), dtype=torch.float64) for _ in range(2)]
        self.e = [torch.zeros((pages, kv), dtype=torch.int64) for _ in range(2)]
        self.written = [torch.zeros((pages, kv), dtype=torch.bool) for _ in range(2)]

    def append(self, k, v, table, lens, cu):
        kv, hd = self.code[0].shape[2:]
        for w, x in enumerate((k, v)):
            x = x.double().reshape(-1, kv, hd)
            for b in range(table.shape[0]):
                rows, p = range(cu[b], cu[b + 1]), max(int(lens[b]), 0)
                todo = {}
                for i, r in enumerate(rows):
                    todo.setdefault((p + i) // self.page, []).append(((p + i) % self.page, r))
                for idx, items in todo.items():
                    if idx >= table.shape[1] or not 0 <= int(table[b, idx]) < self.pages:
                        continue
                    pid, first = int(table[b, idx]), items[0][0]
                    for h in range(kv):
                        new = x[[r for _, r in items], h]
                        fin = new[torch.isfinite(new)]
                        e = exponent(float(fin.abs().max()) if fin.numel() else 0.0)
                        if first > 0:
                            old = int(self.e[w][pid, h])
                            e = max(e, old)
                            if e > old:
                                self.code[w][pid, :first, h] = e4m3(self.code[w][pid, :first, h] * 2.0 ** (old - e))
                        else:
                            self.code[w][pid, :, h] = 0
                        self.code[w][pid, [t for t, _ in items], h] = e4m3(new * 2.0 ** -e)
                        self.e[w][pid, h] = e
                        self.written[w][pid, h] = True

    def value(self, w, pid):
        return self.code[w][pid] * torch.exp2(self.e[w][pid].double())[None, :, None]

    def tokens(self, w, table, b, first, end):
        """(end - first, kv, hd), and which of them the cache holds"""
        kv, hd = self.code[0].shape[2:]
        out = torch.zeros((max(end - first, 0), kv, hd), dtype=torch.float64)
        have = torch.zeros(max(end - first, 0), dtype=torch.bool)
        for t in range(first, end):
            idx = t // self.page
            if 0 <= idx < table.shape[1] and 0 <= int(table[b, idx]) < self.pages:
                out[t - first] = self.value(w, int(table[b, idx]))[t % self.page]
                have[t - first] = True
        return out, have


def attention(q, cache, table, lens, cu, heads, causal, window, scale):
    """(out, bound pieces) float64 (rows, heads * hd): out; sum of weights * |v|; largest sum |q k| scale; NaN rows excluded from none"""
    kv, hd = cache.code[0].shape[2:]
    rows = q.shape[0]
    q = q.double().reshape(rows, heads, hd)
    out, wv = torch.zeros((rows, heads, hd), dtype=torch.float64), torch.zeros((rows, heads, hd), dtype=torch.float64)
    amax = torch.zeros((rows, heads, 1), dtype=torch.float64)
    cap = table.shape[1] * cache.page
    for b in range(table.shape[0]):
        n, length = cu[b + 1] - cu[b], min(max(int(lens[b]), 0), cap)
        if n <= 0 or length == 0:
            continue
        k, have = cache.tokens(0, table, b, 0, length)
        v, _ = cache.tokens(1, table, b, 0, length)
        j = torch.arange(length)
        for i in range(n):
            p = length - n + i
            if p < 0:
                continue
            end = (p // causal + 1) * causal if causal else length
            see = have & (j < end) & (j >= (end - window if window else 0))
            if not bool(see.any()):
                continue
            for h in range(heads):
                kk, vv = k[see, h * kv // heads], v[see, h * kv // heads]
                qq = q[cu[b] + i, h]
                w = torch.softmax((kk @ qq) * scale, 0)
                out[cu[b] + i, h] = w @ vv
                wv[cu[b] + i, h] = w @ vv.abs()
                amax[cu[b] + i, h] = ((kk.abs() @ qq.abs()) * abs(scale)).max()
    return out.reshape(rows, -1), wv.reshape(rows, -1), amax.expand(rows, heads, hd).reshape(rows, -1)
