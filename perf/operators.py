"""Measured cases of the cached-attention operators: the per-head norm with rotation (and its gradient), the 8-bit key / value
cache (append and read back) and the attention that reads it.

The code transformer works on 32 x 32 = 1024 tokens per frame, 8 heads of 64; a stream of frames attends to the frames before it through
the cache.  The other head layouts (grouped heads of 128) and lengths are those such operators meet in general.

`own = False`: plain torch forms, fp32 (angles in 64 bits).  `own = True`: the framework's operators.  `exact`: 64 bits, from the
definitions.

The cache: pages of `page` tokens; per page and kv head one power-of-two scale for K and one for V, codes e4m3.
    k_pages (pages, kv, hd / 16, page, 16)     16 bytes = 16 dims of one token
    v_pages (pages, kv, page / 16, hd, 16)     16 bytes = 16 tokens of one dim
    k_scale, v_scale (pages, kv) fp32
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
LAYOUTS = ((8, 8), (16, 4), (32, 8), (12, 2), (40, 8), (6, 6))      # (heads, kv heads)
E_MIN, E_MAX = -32, 32                                              # range of a block's scale exponent


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a serving step: a few streams, one new token each (latency)
        dict(name="norm+rope, 4 tokens", op="rope", rows=4, heads=32, kv=8, hd=128, rot=128, inter=False, type="bf16"),
        # one frame of the code transformer in its parity type, half of each head rotated, neighbouring pairs
        dict(name="norm+rope, a frame fp32", op="rope", rows=1024, heads=8, kv=8, hd=64, rot=32, inter=True, type="f32"),
        # a long prompt / many frames at once
        dict(name="norm+rope, 16411 tokens", op="rope", rows=16411, heads=32, kv=8, hd=128, rot=128, inter=False, type="bf16"),
        # training: the gradient for one frame's tokens, parity type
        dict(name="norm+rope grad, 999 fp32", op="rope_bwd", rows=999, heads=8, kv=8, hd=64, rot=64, inter=True, type="f32"),
        # training: a packed batch
        dict(name="norm+rope grad, 8190", op="rope_bwd", rows=8190, heads=32, kv=8, hd=128, rot=128, inter=False, type="bf16"),
        # a serving step: one token appended to every stream, the pages it lands in read back
        dict(name="append, 48 x 1 token", op="append", B=48, new=1, old=4100, kv=8, hd=128, page=32, type="bf16"),
        # prompts of ragged lengths written into caches that hold some tokens, and read back
        dict(name="append, 7 prompts", op="append", B=7, new=4099, old=777, kv=8, hd=64, page=64, type="f16"),
        # a few drafted tokens per stream, short caches, fp32, sliding window
        dict(name="attention, 3 x 5 fp32", op="attn", B=3, new=5, len=701, heads=8, kv=8, hd=64, page=16, causal=1, window=300, type="f32"),
        # serving: 48 streams of ragged lengths, one token each
        dict(name="attention, 48 x 1", op="attn", B=48, new=1, len=8191, heads=32, kv=8, hd=128, page=32, causal=1, window=0, type="bf16"),
        # one stream with a long past
        dict(name="attention, 1 x 1 of 131071", op="attn", B=1, new=1, len=131071, heads=40, kv=8, hd=128, page=64, causal=1, window=0, type="f16"),
        # the code transformer's streams: two new frames each, frame-causal, a window of eight frames
        dict(name="attention, 4 x 2 frames", op="attn", B=4, new=2048, len=10240, heads=8, kv=8, hd=64, page=64, causal=1024, window=8192, type="f16"),
        # prompt chunks over a cache
        dict(name="attention, 2 chunks", op="attn", B=2, new=2047, len=8190, heads=32, kv=8, hd=128, page=32, causal=1, window=0, type="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("rope", "rope", "rope_bwd", "append", "append", "attn", "attn", "attn"))
    heads, kv = rng.choice(LAYOUTS)
    hd, typ = rng.choice((64, 128)), rng.choice(("bf16", "f16", "f32"))
    if op in ("rope", "rope_bwd"):
        hd = rng.choice((32, 64, 128, 256))
        rows = min(_log(rng, 1, 16411), 40 * 128 * 16411 // ((heads + kv) * hd))
        return dict(op=op, rows=rows, heads=heads, kv=kv, hd=hd, rot=rng.choice((hd, hd, hd // 2, 0)), inter=rng.random() < 0.5, type=typ)
    page = rng.choice((16, 32, 64, 128))
    if op == "append":
        B = _log(rng, 1, 64)
        new = rng.choice((1, rng.randint(2, 9), _log(rng, 10, max(11, 30000 // B))))
        return dict(op=op, B=B, new=new, old=rng.choice((0, rng.randint(1, 500), _log(rng, 500, 8000))), kv=kv, hd=hd, page=page, type=typ)
    new = rng.choice((1, 1, rng.randint(2, 9), _log(rng, 10, 2047)))
    B = _log(rng, 1, 48) if new < 10 else _log(rng, 1, 4)
    most = min(131071 if B == 1 else 1 << 18, int(1.0e9 / (B * heads * new)), int(2.2e9 / (B * kv * hd)) // 8)
    length = max(new, min(_log(rng, 1, 131071), most))
    causal = rng.choice((1, 1, 1, 0, 16, 100))
    window = rng.choice((0, 0, 0, max(causal, _log(rng, 1, max(2, length))))) if causal else 0
    return dict(op=op, B=B, new=new, len=length, heads=heads, kv=kv, hd=hd, page=page, causal=causal, window=window, type=typ)


def _ragged(n, B, least):
    """lengths of B sequences, the longest n: fixed fractions, so that the work is the same for every seed"""
    return [max(least, int(n * (1 - 0.75 * (b * 0.6180339887 % 1.0)))) for b in range(B)]


def _sizes(c):
    """(old, new): tokens of every sequence in the cache before, and new ones (query rows)"""
    if c["op"] == "append":
        return [c["old"] * (b + 1) // c["B"] for b in range(c["B"])], _ragged(c["new"], c["B"], 1)
    new = _ragged(c["new"], c["B"], 1)
    length = [max(a, b) for a, b in zip(_ragged(c["len"], c["B"], 1), new)]
    return [a - b for a, b in zip(length, new)], new


# --------------------------------------------------------------------------------------------------------------------- inputs
def _scale(amax):
    """power-of-two scale of a block: 2^e, e the least exponent with amax <= 448 * 2^e"""
    m, e = torch.frexp(amax / 448.0)      # amax / 448 = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX))


def _codes(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _cache(g, pages, kv, hd, page):
    k = torch.randn((pages, kv, hd // 16, page, 16), generator=g, device="cuda")
    k *= torch.exp(0.5 * torch.randn((1, kv, hd // 16, 1, 16), generator=g, device="cuda"))      # channels of different strength
    v = torch.randn((pages, kv, page // 16, hd, 16), generator=g, device="cuda")
    v *= torch.exp(0.7 * torch.randn((pages, kv, 1, 1, 1), generator=g, device="cuda"))
    ks, vs = (_scale(t.abs().amax((2, 3, 4))) for t in (k, v))
    return (_codes(k, ks[:, :, None, None, None]).view(torch.uint8), _codes(v, vs[:, :, None, None, None]).view(torch.uint8), ks, vs)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["type"]]
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")      # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    s = {"case": c}
    if c["op"] in ("rope", "rope_bwd"):
        n, h, kv, hd = c["rows"], c["heads"], c["kv"], c["hd"]
        qkv = (rn(n, (h + 2 * kv) * hd) * 1.3).to(t)      # the fused projection's rows
        s["q"], s["k"] = qkv[:, :h * hd], qkv[:, h * hd:(h + kv) * hd]
        s["q_gain"], s["k_gain"] = 1 + 0.2 * rn(hd), 1 + 0.2 * rn(hd)
        first = torch.randint(0, 1 << 20, (1,), generator=g, device="cuda")
        s["pos"] = ((first + torch.arange(n, device="cuda")) % 1000003).to(torch.int32)
        i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
        s["freqs"] = 10000.0 ** (-2.0 * i / max(1, c["rot"])) / (2 * math.pi)      # revolutions per position
        if c["op"] == "rope_bwd":
            s["dq"], s["dk"] = rn(n, h * hd).to(t), rn(n, kv * hd).to(t)
        return s
    old, new = _sizes(c)
    B, kv, hd, page = c["B"], c["kv"], c["hd"], c["page"]
    width = max(-(-(a + b) // page) for a, b in zip(old, new))
    perm = torch.randperm(B * width, generator=g, device="cuda")
    s["table"] = perm.reshape(B, width).to(torch.int32)
    s["cache"] = _cache(g, B * width, kv, hd, page)
    at = [0]
    for b in new:
        at.append(at[-1] + b)
    s["cu"], s["rows"], s["new"] = ints(at), at[-1], max(new)
    if c["op"] == "append":
        s["lens"] = ints(old)
        kvrows = rn(at[-1], 2 * kv * hd)
        kvrows = (kvrows * torch.exp(rn(at[-1], 1).clamp(-2, 2))).to(t)
        s["k"], s["v"] = kvrows[:, :kv * hd], kvrows[:, kv * hd:]
        start = [a // page * page for a in old]      # from the beginning of the first page that is written to
        back = [0]
        for a, b, st in zip(old, new, start):
            back.append(back[-1] + a + b - st)
        s["start"], s["back"], s["back_rows"] = ints(start), ints(back), back[-1]
        s["back_new"] = max(y - x for x, y in zip(back, back[1:]))
        return s
    s["lens"] = ints([a + b for a, b in zip(old, new)])
    s["q"] = (rn(at[-1], c["heads"] * hd) * 1.5).to(t)
    s["scale"] = hd ** -0.5
    return s


# ------------------------------------------------------------------------------------------------------------------------ run
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s)
    if op == "rope":
        return _plain_rope(s)
    if op == "rope_bwd":
        return _plain_rope_bwd(s)
    return _plain_append(s) if op == "append" else _plain_attention(s)


def _own(s):
    from pgtformer_amd import ops
    c = s["case"]
    if c["op"] == "rope":
        return ops.qk_norm_rope(s["q"], s["k"], s["pos"], s["freqs"], s["q_gain"], s["k_gain"], heads=c["heads"], kv_heads=c["kv"],
                                interleaved=c["inter"])
    if c["op"] == "rope_bwd":
        return ops.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["pos"], s["freqs"], s["q_gain"], s["k_gain"], heads=c["heads"],
                                         kv_heads=c["kv"], interleaved=c["inter"])
    cache = ops.KvCache(*s["cache"])
    if c["op"] == "append":
        ops.kv_append(cache, s["k"], s["v"], s["table"], s["lens"], s["cu"], max_new=s["new"])
        return ops.kv_read(cache, s["table"], s["start"], s["back_rows"], TYPES[c["type"]], s["back"], max_rows=s["back_new"])
    return ops.kv_attention(s["q"], cache, s["table"], s["lens"], s["cu"], heads=c["heads"], max_new=s["new"], causal=c["causal"],
                            window=c["window"], scale=s["scale"])


def _turns(s):
    """cos, sin (rows, 1, rot / 2) of the rotation, the angle in 64 bits"""
    turn = s["pos"].double()[:, None] * s["freqs"]
    a = 2 * math.pi * (turn - turn.round())
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _rotate(x, cos, sin, rot, inter):
    if not rot:
        return x
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _turns(s)

    def one(x, gain):
        f = x.float().reshape(c["rows"], -1, c["hd"])
        f = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * gain
        return _rotate(f, cos, sin, c["rot"], c["inter"]).reshape(c["rows"], -1).to(x.dtype)
    return one(s["q"], s["q_gain"]), one(s["k"], s["k_gain"])


def _plain_rope_bwd(s):
    c = s["case"]
    cos, sin = _turns(s)

    def one(dy, x, gain):
        f, z = (t.float().reshape(c["rows"], -1, c["hd"]) for t in (x, dy))
        z = _rotate(z, cos, -sin, c["rot"], c["inter"])
        r = torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)
        f = f * r
        u = z * gain
        dx = r * (u - f * (f * u).mean(-1, keepdim=True))
        return dx.reshape(c["rows"], -1).to(x.dtype), (z * f).double().sum((0, 1)).float()
    dq, gq = one(s["dq"], s["q"], s["q_gain"])
    dk, gk = one(s["dk"], s["k"], s["k_gain"])
    return dq, dk, gq, gk


def _row_index(cu, rows):
    """(sequence, index in it) of every packed row"""
    r = torch.arange(rows, device=cu.device, dtype=torch.int32)
    b = (torch.searchsorted(cu, r, right=True) - 1).clamp(0, cu.numel() - 2)
    return b, r - cu[b]


def _plain_append(s):
    c = s["case"]
    page, kv, hd, B = c["page"], c["kv"], c["hd"], c["B"]
    width = (s["new"] + page - 1 + page - 1) // page      # pages that a sequence's new tokens can touch
    count = s["cu"][1:] - s["cu"][:-1]
    first = s["start"] // page
    pages = (first[:, None] + torch.arange(width, device="cuda")).clamp(max=s["table"].shape[1] - 1)
    pages = torch.gather(s["table"].long(), 1, pages.long())
    pos = s["start"][:, None] + torch.arange(width * page, device="cuda")
    is_old = (pos < s["lens"][:, None])
    is_new = ~is_old & (pos < (s["lens"] + count)[:, None])
    row = (s["cu"][:-1, None] + pos - s["lens"][:, None]).clamp(0, s["rows"] - 1).long()
    any_old = is_old.reshape(B, width, page).any(2)[:, :, None]

    def one(x, codes, scale, axes):
        before = codes[pages].view(torch.float8_e4m3fn).float().permute(axes).reshape(B, width, page, kv, hd)
        was = scale[pages]
        x = (x.float()[row] * is_new[:, :, None]).reshape(B, width, page, kv, hd)
        need = _scale(x.abs().amax((2, 4)))
        now = torch.where(any_old, torch.maximum(was, need), need)
        now, was = now[:, :, None, :, None], was[:, :, None, :, None]
        held = torch.where(is_old.reshape(B, width, page, 1, 1), before * (was / now), x / now)
        held = held.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * now
        b, i = _row_index(s["back"], s["back_rows"])
        return held.reshape(B, width * page, kv * hd)[b, i.long()].to(TYPES[c["type"]])
    kp, vp, ks, vs = s["cache"]
    return one(s["k"], kp, ks, (0, 1, 4, 2, 3, 5)), one(s["v"], vp, vs, (0, 1, 3, 5, 2, 4))


def _plain_attention(s):
    c = s["case"]
    B, kv, hd, h = c["B"], c["kv"], c["hd"], c["heads"]
    kp, vp, ks, vs = s["cache"]
    table = s["table"].long()
    k = kp[table].view(torch.float8_e4m3fn).float() * ks[table][..., None, None, None]
    k = k.permute(0, 2, 1, 4, 3, 5).reshape(B, kv, -1, hd)
    v = vp[table].view(torch.float8_e4m3fn).float() * vs[table][..., None, None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B, kv, -1, hd)
    n, L = s["new"], k.shape[2]
    count = (s["cu"][1:] - s["cu"][:-1])[:, None]
    i = torch.arange(n, device="cuda", dtype=torch.int32)
    q = s["q"].float()[(s["cu"][:-1, None] + i).clamp(max=s["rows"] - 1).long()]
    q = q.reshape(B, n, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, hd)
    x = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).reshape(B, kv, h // kv, n, L)
    lens = s["lens"][:, None]
    pos = lens - count + i
    end = (pos // c["causal"] + 1) * c["causal"] if c["causal"] else lens.expand(B, n)
    j = torch.arange(L, device="cuda", dtype=torch.int32)
    seen = (j < end[..., None]) & (j < lens[..., None])
    if c["window"]:
        seen &= j >= end[..., None] - c["window"]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    d = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, kv, -1, L), v) / torch.where(d == 0, 1.0, d).reshape(B, kv, -1, 1)
    o = o.reshape(B, kv, h // kv, n, hd).permute(0, 3, 1, 2, 4).reshape(B, n, h * hd)
    b, i = _row_index(s["cu"], s["rows"])
    return o[b, i.long()].to(TYPES[c["type"]])


# ----------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c, e = case, BYTES[case["type"]]
    if c["op"] in ("rope", "rope_bwd"):
        n = c["rows"] * (c["heads"] + c["kv"]) * c["hd"]
        fwd = c["op"] == "rope"
        return {"bytes": n * e * (2 if fwd else 3) + 4 * c["rows"] + 8 * c["hd"] * (1 if fwd else 2), "flops": n * (9 if fwd else 17)}
    old, new = _sizes(c)
    kv, hd, page = c["kv"], c["hd"], c["page"]
    if c["op"] == "append":
        held = [a % page for a in old]
        pages = sum(-(-(a + b) // page) for a, b in zip(held, new))
        n = sum(new)
        # new rows read; codes and scales written and read back; what the first pages held read; the values written
        back = n + sum(held)
        return {"bytes": 2 * kv * (hd * (n * (e + 1) + back * (1 + e) + sum(held)) + 8 * pages), "flops": 2 * kv * hd * (4 * n + back)}
    flops = byts = 0
    for a, b in zip(old, new):
        ends = [min(a + b, (p // c["causal"] + 1) * c["causal"]) if c["causal"] else a + b for p in range(a, a + b)]
        wide = [(p // c["causal"] + 1) * c["causal"] if c["causal"] else a + b for p in range(a, a + b)]
        lows = [max(0, w - c["window"]) if c["window"] else 0 for w in wide]
        flops += 4 * hd * c["heads"] * sum(max(0, y - x) for x, y in zip(lows, ends))
        span = max(0, max(ends) - min(lows))
        byts += 2 * b * c["heads"] * hd * e + 2 * kv * span * hd + (8 * kv + 4) * -(-span // page)
    return {"bytes": byts, "flops": max(1, flops)}


# ---------------------------------------------------------------------------------------------------------------------- exact
def _exact_turn(x, s, c):
    """(rows, heads, hd) 64-bit: pairs of each head as complex numbers, times exp(i angle)"""
    rot = c["rot"]
    if not rot:
        return x
    angle = 2 * math.pi * (s["pos"].double().unsqueeze(1) * s["freqs"]).remainder(1.0)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
    head, tail = x[..., :rot], x[..., rot:]
    if c["inter"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(head.shape)
    else:
        z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
        head = torch.cat((z.real, z.imag), -1)
    return torch.cat((head, tail), -1)


def _exact_rope(s, c, x, gain):
    x = x.reshape(c["rows"], -1, c["hd"])
    return _exact_turn(gain * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6), s, c).reshape(c["rows"], -1)


def _exact_code(x):
    """nearest e4m3 value (ties to even) of |x| <= 448 in 64 bits"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_values():
    """the 256 numbers an e4m3 byte stands for"""
    v = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v.append(-x if code & 128 else x)
    v[0x7f] = v[0xff] = math.nan
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _exact_rows(s, c, b, first, end):
    """K, V (tokens, kv, hd) of tokens first .. end - 1 of sequence b, in 64 bits"""
    kp, vp, ks, vs = s["cache"]
    page = c["page"]
    ids = s["table"][b, first // page:-(-end // page)].long()
    val = _exact_values()
    k = val[kp[ids].int()] * ks[ids].double()[:, :, None, None, None]
    v = val[vp[ids].int()] * vs[ids].double()[:, :, None, None, None]
    k = k.permute(0, 3, 1, 2, 4).reshape(-1, c["kv"], c["hd"])
    v = v.permute(0, 2, 4, 1, 3).reshape(-1, c["kv"], c["hd"])
    off = first // page * page
    return k[first - off:end - off], v[first - off:end - off]


def _exact_exponent(amax):
    """least e in the range with amax <= 448 * 2^e"""
    e = torch.full_like(amax, float(E_MIN))
    for step in range(E_MIN, E_MAX):
        e = torch.where(amax > 448.0 * 2.0 ** step, float(step + 1), e)
    return e


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        return tuple(_exact_rope(s, c, s[n].double(), s[n + "_gain"].double()) for n in "qk")
    if c["op"] == "rope_bwd":
        got = []
        for n in "qk":
            x, gain = s[n].double().requires_grad_(), s[n + "_gain"].double().requires_grad_()
            got.append(torch.autograd.grad(_exact_rope(s, c, x, gain), (x, gain), s["d" + n].double()))
        return got[0][0], got[1][0], got[0][1], got[1][1]
    old, new = _sizes(c)
    page = c["page"]
    if c["op"] == "append":
        outs, at = ([], []), 0
        for b in range(c["B"]):
            first = old[b] // page * page
            held = _exact_rows(s, c, b, first, old[b]) if old[b] > first else (None, None)
            for w, name in enumerate("kv"):
                x = s[name][at:at + new[b]].double().reshape(new[b], c["kv"], c["hd"])
                n_old = old[b] - first
                total = n_old + new[b]
                blocks = -(-total // page)
                pad = torch.zeros((blocks * page, c["kv"], c["hd"]), dtype=torch.float64, device="cuda")
                pad[n_old:total] = x
                e = _exact_exponent(pad.reshape(blocks, page, c["kv"], c["hd"]).abs().amax((1, 3)))
                if n_old:
                    was = torch.log2(s["cache"][2 + w][s["table"][b, old[b] // page].long()].double())
                    e[0] = torch.maximum(e[0], was)
                    pad[:n_old] = held[w]
                u = torch.exp2(e).repeat_interleave(page, 0)[:, :, None]
                outs[w].append((_exact_code(pad / u) * u)[:total].reshape(total, -1))
            at += new[b]
        return tuple(torch.cat(o) for o in outs)
    out, h, group = [], c["heads"], c["heads"] // c["kv"]
    at = 0
    for b in range(c["B"]):
        n, length = new[b], old[b] + new[b]
        pos = torch.arange(old[b], length, device="cuda")
        end = (pos // c["causal"] + 1) * c["causal"] if c["causal"] else torch.full_like(pos, length)
        low = end - c["window"] if c["window"] else torch.zeros_like(end)
        first = max(0, int(low.min()))
        o = torch.zeros((n, h, c["hd"]), dtype=torch.float64, device="cuda")
        if first < length:
            k, v = _exact_rows(s, c, b, first, length)
            q = s["q"][at:at + n].double().reshape(n, h, c["hd"])
            j = torch.arange(first, length, device="cuda")
            seen = (j[None] < end[:, None]) & (j[None] >= low[:, None])
            some = seen.any(1)
            for a in range(h):
                x = (q[:, a] @ k[:, a // group].T) * s["scale"]
                p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                o[:, a] = torch.where(some[:, None], p, 0.0) @ v[:, a // group]
        out.append(o.reshape(n, -1))
        at += n
    return torch.cat(out)
