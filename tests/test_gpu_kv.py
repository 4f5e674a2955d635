"""Cached-attention operators on the GPU against plain 64-bit forms (tests/kv_ref.py): per-head norm + rotation and its gradient,
append / read of the 8-bit cache, attention over it.  Tolerances: half a step of the output type plus the fp32 (and, for the attention
weights, half) roundings inside, derived beside each check."""
import pytest
import torch

from pgtformer_amd import hip, ops
from tests import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step (e.g. bf16: eps / 2 = 2^-8)
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}     # half a step of a subnormal


def close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()), float(((got - want).abs() / tol).max()))


# ------------------------------------------------------------------------------------------------------- norm + rotation
ROPE = [  # rows, heads, kv, hd, rot, interleaved, type
    (1, 8, 8, 64, 64, False, "bf16"), (1, 40, 8, 128, 128, True, "f16"), (3, 5, 1, 32, 8, True, "f32"), (37, 8, 2, 64, 32, True, "bf16"),
    (129, 32, 8, 128, 128, False, "bf16"), (7, 3, 3, 256, 256, False, "f32"), (65, 2, 2, 256, 24, False, "f16"), (4097, 4, 2, 64, 64, False, "f16"),
    (4099, 3, 1, 32, 32, True, "f32"), (5, 8, 8, 64, 0, False, "bf16"), (2, 6, 2, 128, 40, True, "f32"), (4096, 3, 1, 32, 16, True, "bf16"),
    (4100, 2, 1, 256, 48, False, "f16"), (4101, 4, 2, 128, 0, False, "bf16"), (4097, 2, 2, 128, 24, False, "bf16"), (4098, 5, 1, 128, 128, True, "f16"),
    (601, 8, 2, 64, 64, False, "bf16"), (2499, 3, 1, 64, 32, True, "f32"), (777, 3, 1, 32, 8, True, "f16"), (2501, 2, 2, 128, 64, True, "bf16"), (512, 1, 1, 256, 256, False, "f32"),
]


def rope_inputs(rows, heads, kv, hd, rot, typ, seed=0, pad=8):
    g = torch.Generator().manual_seed(seed)
    wide = (torch.randn((rows, (heads + 2 * kv) * hd + pad), generator=g) * 2).to(DT[typ])
    q, k = wide[:, :heads * hd], wide[:, heads * hd:(heads + kv) * hd]
    pos = torch.randint(-(1 << 30), 1 << 30, (rows,), generator=g, dtype=torch.int32)
    pos[: rows // 2] = torch.arange(rows // 2, dtype=torch.int32)
    qg, kg = 1 + 0.3 * torch.randn(hd, generator=g), 1 + 0.3 * torch.randn(hd, generator=g)
    freqs = ops.rope_freqs(rot, device="cpu") if rot else None
    return wide, q, k, pos, qg, kg, freqs


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def pair_norm(y, rot, inter, heads):
    """hypot of the pair that an element is turned with"""
    y = y.abs().reshape(y.shape[0], heads, -1)
    if rot:
        i = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
        j = i + 1 if inter else i + rot // 2
        n = torch.hypot(y[..., i], y[..., j])
        y = y.clone()
        y[..., i] = n
        y[..., j] = n
    return y.reshape(y.shape[0], -1)


@pytest.mark.parametrize("rows,heads,kv,hd,rot,inter,typ", ROPE)
def test_qk_norm_rope(rows, heads, kv, hd, rot, inter, typ):
    wide, q, k, pos, qg, kg, freqs = rope_inputs(rows, heads, kv, hd, rot, typ)
    w, p, f, a, b = dev(wide, pos, freqs, qg, kg)
    qd, kd = w[:, :heads * hd], w[:, heads * hd:(heads + kv) * hd]
    got = ops.qk_norm_rope(qd, kd, p, f, a, b, heads=heads, kv_heads=kv, eps=1e-5, interleaved=inter)
    again = ops.qk_norm_rope(qd, kd, p, f, a, b, heads=heads, kv_heads=kv, eps=1e-5, interleaved=inter)
    for x, g_, y, y2, n in ((q, qg, got[0], again[0], heads), (k, kg, got[1], again[1], kv)):
        want = kv_ref.rope(x.double(), n, pos, freqs, g_.double(), 1e-5, inter)
        # fp32: mean of squares (tree of <= 13 additions), root, reciprocal, two products: < 24 roundings of 2^-24; the angle's fraction is
        # rounded to 2^-24 of a turn (2 pi 2^-24 / 2 < 2^-22), sin / cos 2 ulp, two products and a sum: < 2^-20 of the pair's norm in all
        tol = HALF[typ] * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -20 * pair_norm(want, rot, inter, n) + TINY[typ]
        close(y, want, tol)
        assert torch.equal(y, y2)


def test_qk_norm_rope_in_place_and_strided_outputs():
    rows, heads, kv, hd = 33, 8, 2, 64
    wide, q, k, pos, qg, kg, freqs = rope_inputs(rows, heads, kv, hd, hd, "bf16")
    w, p, f, a, b = dev(wide, pos, freqs, qg, kg)
    qd, kd = w[:, :heads * hd], w[:, heads * hd:(heads + kv) * hd]
    want = ops.qk_norm_rope(qd, kd, p, f, a, b, heads=heads, kv_heads=kv)
    rest = w[:, (heads + kv) * hd:].clone()
    got = ops.qk_norm_rope(qd, kd, p, f, a, b, heads=heads, kv_heads=kv, out=(qd, kd))
    assert got[0].data_ptr() == qd.data_ptr() and torch.equal(qd, want[0]) and torch.equal(kd, want[1])
    assert torch.equal(w[:, (heads + kv) * hd:], rest)


def test_qk_norm_rope_without_gain_zero_rows_and_special_values():
    heads, kv, hd = 4, 1, 64
    _, q, k, pos, _, _, freqs = rope_inputs(9, heads, kv, hd, hd, "f32", pad=0)
    q, k = q.contiguous(), k.contiguous()
    q[2] = 0
    q[3, 5] = float("nan")
    q[4, 70] = float("inf")
    qd, kd, p, f = dev(q, k, pos, freqs)
    y, _ = ops.qk_norm_rope(qd, kd, p, f, heads=heads, kv_heads=kv)
    want = kv_ref.rope(q.double(), heads, pos, freqs, None, 1e-6, False)
    ok = torch.ones(9, dtype=torch.bool)
    ok[3:5] = False
    close(y.cpu()[ok], want[ok], 2.0 ** -20 * (pair_norm(want, hd, False, heads)[ok] + 2.0 ** -20))
    assert bool((y[2] == 0).all())
    y = y.cpu()
    assert bool(y[3, :64].isnan().all()) and not bool(y[3, 64:].isnan().any())      # a head with NaN, its neighbours untouched
    assert not bool(y[4, :64].isnan().any()) and bool(y[4, 64:128].isnan().any())
    e = ops.qk_norm_rope(qd[:0], kd[:0], p[:0], f, heads=heads, kv_heads=kv)
    assert e[0].shape == (0, heads * hd) and e[1].shape == (0, kv * hd)
    g = ops.qk_norm_rope_backward(e[0], e[1], qd[:0], kd[:0], p[:0], f, heads=heads, kv_heads=kv)
    assert g[0].shape == (0, heads * hd) and bool((g[2] == 0).all()) and bool((g[3] == 0).all())


@pytest.mark.parametrize("rows,heads,kv,hd,rot,inter,typ", ROPE)
def test_qk_norm_rope_backward(rows, heads, kv, hd, rot, inter, typ):
    wide, q, k, pos, qg, kg, freqs = rope_inputs(rows, heads, kv, hd, rot, typ, seed=1)
    g = torch.Generator().manual_seed(2)
    dq, dk = (torch.randn((rows, n * hd), generator=g).to(DT[typ]) for n in (heads, kv))
    w, p, f, a, b, dqd, dkd = dev(wide, pos, freqs, qg, kg, dq, dk)
    args = (w[:, :heads * hd], w[:, heads * hd:(heads + kv) * hd], p, f, a, b)
    kw = dict(heads=heads, kv_heads=kv, eps=1e-5, interleaved=inter)
    got = ops.qk_norm_rope_backward(dqd, dkd, *args, **kw)
    again = ops.qk_norm_rope_backward(dqd, dkd, *args, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    for x, dy, gain, n, dx, dg in ((q, dq, qg, heads, got[0], got[2]), (k, dk, kg, kv, got[1], got[3])):
        xd, gd = x.double().requires_grad_(), gain.double().requires_grad_()
        y = kv_ref.rope(xd, n, pos, freqs, gd, 1e-5, inter)
        wx, wg = torch.autograd.grad(y, (xd, gd), dy.double())
        xh = x.double().reshape(rows, n, hd)
        r = 1 / torch.sqrt((xh * xh).mean(-1, keepdim=True) + 1e-5)
        xh = (xh * r).abs()
        z = pair_norm(dy.double(), rot, inter, n).reshape(rows, n, hd)
        u = z * gain.double().abs()
        # the same roundings as forward on u, on xh and on the mean of their product, times r
        tol = HALF[typ] * (1 + 2.0 ** -8) * wx.abs() + (2.0 ** -19 * r * (u + xh * (xh * u).mean(-1, keepdim=True))).reshape(rows, -1) + TINY[typ]
        close(dx, wx, tol)
        # each of the rows * n products to 2^-20; a lane adds at most ceil(4 (heads + kv) / head rows in flight) * ceil(rows / 4 / groups) <= 200
        # of them, 16-64 lanes in order, then fp64: < 300 additions of 2^-24 each
        close(dg, wg, (2.0 ** -20 + 300 * 2.0 ** -24) * (z * xh).sum((0, 1)) + 2.0 ** -24 * wg.abs())


def test_qk_norm_rope_backward_against_differences():
    rows, heads, kv, hd = 3, 2, 1, 64
    _, q, k, pos, qg, kg, freqs = rope_inputs(rows, heads, kv, hd, 32, "f32", seed=3)
    pos = pos.abs() % 1000
    g = torch.Generator().manual_seed(4)
    dq, dk = torch.randn((rows, heads * hd), generator=g), torch.randn((rows, kv * hd), generator=g)
    got = ops.qk_norm_rope_backward(*dev(dq, dk, q.contiguous(), k.contiguous(), pos, freqs, qg, kg), heads=heads, kv_heads=kv)

    def loss(x, n, gain, dy):
        return float((kv_ref.rope(x, n, pos, freqs, gain, 1e-6, False) * dy.double()).sum())
    h = 1e-5      # central differences in 64 bits: error h^2 |f'''| + 2^-52 |f| / h < 1e-8
    for x, n, gain, dy, dx, dg in ((q, heads, qg, dq, got[0], got[2]), (k, kv, kg, dk, got[1], got[3])):
        x, gain = x.double(), gain.double()
        for i, j in ((0, 0), (1, 17), (2, hd - 1), (rows - 1, n * hd - 5)):
            d = torch.zeros_like(x)
            d[i, j] = h
            num = (loss(x + d, n, gain, dy) - loss(x - d, n, gain, dy)) / (2 * h)
            assert abs(float(dx[i, j]) - num) < 1e-5 * (1 + abs(num))
        for j in (0, 31, 32, hd - 1):
            d = torch.zeros_like(gain)
            d[j] = h
            num = (loss(x, n, gain + d, dy) - loss(x, n, gain - d, dy)) / (2 * h)
            assert abs(float(dg[j]) - num) < 1e-5 * (1 + abs(num)) * rows


# ----------------------------------------------------------------------------------------------------- append and read
def scatter_table(B, width, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[: B * width].reshape(B, width).to(torch.int32)


def gpu_codes(cache):
    """(K, V) code values (pages, page, kv, hd) float64 and scales of a KvCache, on the CPU"""
    k = cache.k_pages.view(torch.float8_e4m3fn).float().permute(0, 3, 1, 2, 4).reshape(cache.pages, cache.page, cache.kv_heads, cache.hd)
    v = cache.v_pages.view(torch.float8_e4m3fn).float().permute(0, 2, 4, 1, 3).reshape(cache.pages, cache.page, cache.kv_heads, cache.hd)
    return [t.double().cpu() for t in (k, v)], [t.double().cpu() for t in (cache.k_scale, cache.v_scale)]


def same_cache(cache, ref, used):
    """the cache equals the reference on its `used` (page, token) pairs"""
    codes, scales = gpu_codes(cache)
    for w in range(2):
        for pid in range(ref.pages):
            n = used.get(pid, 0)
            if n:
                assert torch.equal(scales[w][pid], torch.exp2(ref.e[w][pid].double())), (w, pid)
                x, y = codes[w][pid, :n], ref.code[w][pid, :n]
                assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num()), (w, pid)


def used_of(table, lens, page):
    used = {}
    for b in range(table.shape[0]):
        for t in range(min(int(lens[b]), table.shape[1] * page)):
            pid = int(table[b, t // page])
            used[pid] = max(used.get(pid, 0), t % page + 1)
    return used


@pytest.mark.parametrize("page,hd,kv,typ", [(16, 64, 1, "f32"), (16, 128, 2, "bf16"), (32, 64, 3, "f16"), (64, 128, 1, "f32"), (128, 64, 2, "bf16"),
                                            (128, 128, 1, "f16")])
def test_kv_append_and_read_over_several_calls(page, hd, kv, typ):
    """ragged appends from empty: codes, scales and values equal the definition bit for bit, whatever growth the pages saw"""
    B, width = 4, 5
    pages = B * width + 3
    cache, ref = ops.KvCache.alloc(pages, kv, page, hd, DEV), kv_ref.Cache(pages, kv, page, hd)
    table = scatter_table(B, width, pages, 5)
    tab = table.to(DEV)
    lens = [0] * B
    g = torch.Generator().manual_seed(6)
    for step, counts in enumerate(([1, 0, page, page + 3], [1, 2, 1, 1], [1, page - 2, 2, 0], [3, 1, page, 5], [1, 1, 1, 1])):
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        wide = torch.randn((cu[-1], 2 * kv * hd + 16), generator=g) * torch.exp(3 * torch.randn((cu[-1], 1), generator=g))
        if step == 1:
            wide *= 2.0 ** -12       # a page's scale stays, small values go under its smallest step
        wide = wide.to(DT[typ])
        k, v = wide[:, :kv * hd], wide[:, kv * hd:2 * kv * hd]
        ref.append(k, v, table, lens, cu)
        wd = wide.to(DEV)
        ops.kv_append(cache, wd[:, :kv * hd], wd[:, kv * hd:2 * kv * hd], tab, torch.tensor(lens, dtype=torch.int32, device=DEV),
                      torch.tensor(cu, dtype=torch.int32, device=DEV), max_new=max(counts))
        lens = [a + c for a, c in zip(lens, counts)]
        same_cache(cache, ref, used_of(table, lens, page))
    for out in ("f32", "bf16", "f16"):
        start = [0, 1, min(page, lens[2]), lens[3] - 1]
        cu = [0]
        for b in range(B):
            cu.append(cu[-1] + lens[b] - start[b])
        back = ops.kv_read(cache, tab, torch.tensor(start, dtype=torch.int32, device=DEV), cu[-1], DT[out],
                           torch.tensor(cu, dtype=torch.int32, device=DEV))
        for w in range(2):
            want = torch.cat([ref.tokens(w, table, b, start[b], lens[b])[0] for b in range(B)]).reshape(cu[-1], -1)
            lim = torch.finfo(DT[out]).max
            assert torch.equal(back[w].cpu(), want.clamp(-lim, lim).to(DT[out])), (out, w)


def test_kv_append_special_values_and_scale_range():
    """zeros, infinities (saturate), NaN (stays, does not count), values at the border of an exponent, beyond the scale's range"""
    page, hd, kv = 16, 64, 1
    rows = []
    one = torch.zeros(hd)
    rows.append(one.clone())                                                     # all zeros
    for top in (448.0, 448.0 * (1 + 2.0 ** -22), 447.99997, 1.75, 1.7500001, 3.4e38, 1e-38, 2.0 ** -41, 1e13):
        r = torch.linspace(-1, 1, hd) * top * 0.3
        r[7] = top
        rows.append(r)
    r = torch.linspace(-3, 3, hd)
    r[0], r[1], r[2] = float("inf"), -float("inf"), float("nan")
    rows.append(r)
    rows.append(torch.full((hd,), float("nan")))
    x = torch.stack(rows)
    n = x.shape[0]
    cache, ref = ops.KvCache.alloc(n, kv, page, hd, DEV), kv_ref.Cache(n, kv, page, hd)      # one row per sequence and page
    table = torch.arange(n, dtype=torch.int32).reshape(n, 1)
    ref.append(x, x.flip(1), table, [0] * n, list(range(n + 1)))
    zero = torch.zeros(n, dtype=torch.int32, device=DEV)
    ops.kv_append(cache, x.to(DEV), x.flip(1).contiguous().to(DEV), table.to(DEV), zero)
    same_cache(cache, ref, {i: page for i in range(n)})      # (a fresh page is zero behind its last token)


def test_kv_append_leaves_everything_else_alone():
    """pages of nobody, tokens behind the table, tables with ids outside the cache, negative lengths, rows that no sequence owns"""
    page, hd, kv, pages = 16, 64, 2, 6
    g = torch.Generator().manual_seed(8)
    cache = ops.KvCache.alloc(pages, kv, page, hd, DEV)
    for t in (cache.k_pages, cache.v_pages):
        t.random_(0, 120)
    cache.k_scale.fill_(0.5)
    cache.v_scale.fill_(0.25)
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)]
    k = torch.randn((40, kv * hd), generator=g).to(DEV)
    table = torch.tensor([[2, -1, 1 << 30], [pages, -5, 4]], dtype=torch.int32, device=DEV)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)      # noqa: E731
    # sequence 0: tokens -7 (= 0) .. 19: page 2, then a page that is not there; sequence 1: 40 .. 59: page 4 (from token 8), then off the table
    ops.kv_append(cache, k, k, table, ints(-7, 40), ints(0, 20, 40))
    after = [cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale]
    for i in range(4):
        for pid in range(pages):
            same = torch.equal(after[i][pid], before[i][pid])
            assert same == (pid not in (2, 4)) or (i >= 2 and pid == 4), (i, pid)
    kk = gpu_codes(cache)[0][0]
    old = before[0].view(torch.float8_e4m3fn).float().permute(0, 3, 1, 2, 4).reshape(pages, page, kv, hd).double().cpu()
    assert torch.equal(kk[4, :8], old[4, :8])      # the scale was large enough: tokens before stay as they are
    # nothing to do: no rows, no table, no tokens
    for args in ((k[:0], k[:0], table, ints(0, 0), ints(0, 0, 0)), (k, k, table[:, :0], ints(0, 0), ints(0, 20, 40))):
        keep = [t.clone() for t in after]
        ops.kv_append(cache, *args)
        assert all(torch.equal(x, y) for x, y in zip(keep, after))
    # broken offsets are bounded: descending, negative, past the end
    ops.kv_append(cache, k, k, table, ints(0, 0), ints(30, -4, 1000))
    out = torch.full((2, 50, kv * hd), 7.0, device=DEV)
    got = ops.kv_read(cache, table, ints(0, 0), 50, torch.float32, ints(3, 23, 30), max_rows=20, out=(out[0], out[1]))
    assert bool((got[0][:3] == 7).all()) and bool((got[0][30:] == 7).all()) and bool((got[1][30:] == 7).all())
    assert bool((got[0][19:23] == 0).all()) and bool((got[0][23:30] == 0).all())      # page -1, page `pages`: read as zeros


# --------------------------------------------------------------------------------------------------------------- attention
def filled(B, width, pages, kv, page, hd, lens, seed, vspread=1.0):
    """a cache holding lens[b] tokens of every sequence, and its reference"""
    cache, ref = ops.KvCache.alloc(pages, kv, page, hd, DEV), kv_ref.Cache(pages, kv, page, hd)
    for t in (cache.k_pages, cache.v_pages):
        t.fill_(0x7f)      # NaN wherever nothing is written
    table = scatter_table(B, width, pages, seed)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + max(n, 0))
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn((cu[-1], kv * hd), generator=g), torch.randn((cu[-1], kv * hd), generator=g)
    v *= torch.exp(vspread * torch.randn((cu[-1], 1), generator=g))
    ref.append(k, v, table, [0] * B, cu)
    if cu[-1]:
        ops.kv_append(cache, k.to(DEV), v.to(DEV), table.to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV),
                      torch.tensor(cu, dtype=torch.int32, device=DEV))
    return cache, ref, table, g


def attn_tol(typ, want, wv, amax, length):
    # scores: hd products and sums in fp32, the scale: delta <= 2^-17 relative to the largest sum of |q k| (hd <= 128 terms of 2^-24), in units of the
    # natural logarithm; exp2 and its argument: 2^-20.  weights rounded to half (fp32: two halves): 2^-11 (2^-22).  sums over `length`
    # weights in fp32: a random walk of 2^-24 steps, taken 8 times its spread.  each enters numerator and denominator.
    p = 2.0 ** -22 if typ == "f32" else 2.0 ** -11
    inner = p + 2 * (2.0 ** -17 * amax + 2.0 ** -20) + 16 * max(length, 1) ** 0.5 * 2.0 ** -24
    return HALF[typ] * (1 + 2.0 ** -7) * want.abs() + inner * wv + TINY[typ]


ATTN = [  # lens, new tokens, heads, kv, hd, page, causal, window, type
    ([1], [1], 8, 8, 64, 16, 1, 0, "bf16"),
    ([0, 5, 33], [0, 5, 1], 8, 2, 64, 16, 1, 0, "f16"),
    ([64, 65, 63, 128], [1, 1, 1, 1], 32, 8, 128, 32, 1, 0, "bf16"),
    ([200, 17, 130], [1, 1, 1], 40, 8, 128, 64, 1, 0, "f32"),
    ([700, 1, 300], [5, 1, 3], 6, 6, 64, 128, 1, 0, "f32"),
    ([150, 90], [37, 90], 12, 2, 64, 32, 1, 0, "bf16"),
    ([150, 90], [37, 64], 8, 8, 128, 16, 0, 0, "f16"),
    ([260, 100], [70, 100], 4, 1, 64, 64, 16, 0, "f32"),
    ([260, 100, 40], [70, 100, 40], 8, 2, 128, 32, 1, 50, "bf16"),
    ([260, 100, 40], [70, 100, 40], 4, 4, 64, 16, 100, 30, "f16"),      # a window shorter than the block: rows that see nothing
    ([1030], [3], 20, 4, 128, 128, 1, 1, "f16"),
    ([513, 257], [129, 256], 16, 2, 128, 16, 1, 0, "bf16"),
    ([300], [300], 3, 3, 64, 64, 7, 64, "bf16"),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_kv_attention(case):
    lens, new, heads, kv, hd, page, causal, window, typ = ATTN[case]
    B, width = len(lens), -(-max(lens) // page) + (case % 3)
    cache, ref, table, g = filled(B, max(width, 1), B * max(width, 1) + 2, kv, page, hd, lens, 11 + case)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    wide = (torch.randn((cu[-1], heads * hd + 8 * (case % 2)), generator=g) * 1.5).to(DT[typ])
    q = wide[:, :heads * hd]
    want, wv, amax = kv_ref.attention(q, ref, table, lens, cu, heads, causal, window, hd ** -0.5)
    qd = wide.to(DEV)[:, :heads * hd]
    ln, c = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (lens, cu))
    out = torch.full((cu[-1] + 5, heads * hd), 3.0, dtype=DT[typ], device=DEV)
    kw = dict(heads=heads, causal=causal, window=window)
    got = ops.kv_attention(qd, cache, table.to(DEV), ln, c, max_new=max(new), **kw)
    close(got, want, attn_tol(typ, want, wv, amax, max(lens)), "case %d" % case)
    assert torch.equal(got, ops.kv_attention(qd, cache, table.to(DEV), ln, c, max_new=max(new), **kw))
    # rows behind the last sequence stay as they were; without max_new the split of the work may differ, the values not beyond rounding
    qpad = torch.cat([qd, qd[:1].expand(5, -1)])
    got = ops.kv_attention(qpad, cache, table.to(DEV), ln, c, out=out, **kw)
    close(got[:cu[-1]], want, attn_tol(typ, want, wv, amax, max(lens)), "padded %d" % case)
    assert bool((out[cu[-1]:] == 3).all())


def test_kv_attention_one_token_each_without_offsets_and_in_place():
    B, heads, kv, hd, page = 5, 8, 2, 64, 16
    lens = [40, 1, 16, 77, 33]
    cache, ref, table, g = filled(B, 5, 30, kv, page, hd, lens, 3)
    q = torch.randn((B, heads * hd), generator=g).to(torch.bfloat16)
    want, wv, amax = kv_ref.attention(q, ref, table, lens, list(range(B + 1)), heads, 1, 0, 0.2)
    qd = q.to(DEV)
    got = ops.kv_attention(qd, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), heads=heads, scale=0.2, out=qd)
    assert got.data_ptr() == qd.data_ptr()
    close(got, want, attn_tol("bf16", want, wv, amax, 77))


@pytest.mark.parametrize("n,typ", [(1, "bf16"), (40, "f16"), (3, "f32")])
def test_kv_attention_nan_and_infinity_in_masked_places(n, typ):
    """NaN keys / values reach exactly the queries that see their token; unwritten parts of pages hold NaN codes throughout (filled)"""
    B, heads, kv, hd, page, length = 2, 4, 2, 64, 32, 90
    cache, ref, table, g = filled(B, 4, 9, kv, page, hd, [length, length], 21)
    clean = [t.clone() for t in (cache.k_pages, cache.v_pages)]
    q = torch.randn((B * n, heads * hd), generator=g).to(DT[typ]).to(DEV)
    ln = torch.tensor([length, length], dtype=torch.int32, device=DEV)
    base = ops.kv_attention(q, cache, table.to(DEV), ln, heads=heads, window=41)
    assert bool(torch.isfinite(base).all())

    def poison(t, which, d):      # token t of sequence 0, kv head 1
        pid = int(table[0, t // page])
        s = t % page
        if which == 0:
            cache.k_pages[pid, 1, d // 16, s, d % 16] = 0xff
        else:
            cache.v_pages[pid, 1, s // 16, d, s % 16] = 0x7f
    for which in (0, 1):
        for t in (length - n, length - 1, max(length - n - 41, 0), max(length - n - 40, 0)):
            cache.k_pages.copy_(clean[0])
            cache.v_pages.copy_(clean[1])
            poison(t, which, 19)
            got = ops.kv_attention(q, cache, table.to(DEV), ln, heads=heads, window=41)
            want = base.clone()
            for i in range(n):
                p = length - n + i
                if p - 41 < t <= p:
                    for h in (2, 3):      # the heads of kv head 1
                        if which == 0:
                            want[i, h * hd:(h + 1) * hd] = float("nan")
                        else:
                            want[i, h * hd + 19] = float("nan")
            assert torch.equal(got.isnan(), want.isnan()), (which, t, int(got.isnan().sum()), int(want.isnan().sum()))
            assert torch.equal(got.nan_to_num(), want.nan_to_num())
    cache.k_pages.copy_(clean[0])
    cache.v_pages.copy_(clean[1])
    q2 = q.clone()
    q2[0, 3] = float("inf")
    q2[0, hd + 3] = float("nan")
    got = ops.kv_attention(q2, cache, table.to(DEV), ln, heads=heads, window=41)
    assert bool(got[0, :2 * hd].isnan().all()) and torch.equal(got[0, 2 * hd:], base[0, 2 * hd:]) and torch.equal(got[1:], base[1:])


def test_kv_attention_missing_pages_and_broken_index_values():
    """table entries outside the cache, lengths past the table, negative lengths, more rows than tokens: bounded, and what is not there is
    not seen"""
    heads, kv, hd, page, pages = 4, 2, 64, 16, 12
    cache, ref, table, g = filled(3, 4, pages, kv, page, hd, [64, 64, 64], 31)
    table = table.clone()
    table[0, 1], table[1, 0], table[1, 3] = -1, pages, 1 << 30
    table[2] = -7
    lens, cu = [60, 5000, 40], [0, 2, 12, 13]
    q = torch.randn((13, heads * hd), generator=g)
    eff = [60, 64, 40]
    want, wv, amax = kv_ref.attention(q, ref, table, eff, cu, heads, 1, 0, 0.125)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)      # noqa: E731
    got = ops.kv_attention(q.to(DEV), cache, table.to(DEV), ints(lens), ints(cu), heads=heads)
    close(got, want, attn_tol("f32", want, wv, amax, 64))
    assert bool((got[12] == 0).all())
    got = ops.kv_attention(q.to(DEV), cache, table.to(DEV), ints([-3, 4, 0]), ints(cu), heads=heads)
    assert bool((got[:2] == 0).all()) and bool((got[2:8] == 0).all()) and bool((got[12] == 0).all())
    out = torch.full((13, heads * hd), 2.0, device=DEV)
    ops.kv_attention(q.to(DEV), cache, table.to(DEV), ints([60, 60, 60]), ints([9, 3, -1, 500]), heads=heads, out=out)
    e = ops.kv_attention(q[:0].to(DEV), cache, table.to(DEV), ints([60, 60, 60]), ints([0, 0, 0, 0]), heads=heads)
    assert e.shape == (0, heads * hd)
    e = ops.kv_attention(q.to(DEV), cache, table.to(DEV)[:, :0], ints([60, 60, 60]), ints(cu), heads=heads)
    assert bool((e == 0).all())


def test_kv_attention_values_of_very_different_scale():
    """V pages 2^40 apart, and weights that favour the small ones: the softmax sum and the product keep both"""
    heads, kv, hd, page = 2, 1, 64, 16
    g = torch.Generator().manual_seed(41)
    for typ in ("f32", "bf16"):
        cache, ref = ops.KvCache.alloc(8, kv, page, hd, DEV), kv_ref.Cache(8, kv, page, hd)
        table = torch.arange(8, dtype=torch.int32).reshape(1, 8)
        k = torch.randn((100, hd), generator=g)
        v = torch.randn((100, hd), generator=g) * torch.exp2(20.0 * torch.randn((100, 1), generator=g).clamp(-1, 1)).roll(0)
        v[:16], v[16:32], v[32:48] = v[:16] * 2.0 ** -30, v[16:32] * 2.0 ** 30, v[32:48] * 2.0 ** -20
        ref.append(k, v, table, [0], [0, 100])
        zero = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.kv_append(cache, k.to(DEV), v.to(DEV), table.to(DEV), zero)
        q = (3 * torch.randn((20, heads * hd), generator=g)).to(DT[typ])
        for length in (16, 48, 100):
            n = 16
            want, wv, amax = kv_ref.attention(q[:n], ref, table, [length], [0, n], heads, 1, 0, 0.125)
            got = ops.kv_attention(q[:n].to(DEV), cache, table.to(DEV), torch.tensor([length], dtype=torch.int32, device=DEV), heads=heads)
            close(got, want, attn_tol(typ, want, wv, amax, length), (typ, length))


def test_offsets_past_32_bits():
    """a cache of more than 4 GiB per tensor: pages at its end"""
    kv, hd, page, heads = 8, 128, 128, 8
    pages = 33000      # x 128 KiB = 4.03 GiB
    mk = lambda *s, dt=torch.uint8: torch.empty(s, dtype=dt, device=DEV)      # noqa: E731
    cache = ops.KvCache(mk(pages, kv, hd // 16, page, 16), mk(pages, kv, page // 16, hd, 16), mk(pages, kv, dt=torch.float32), mk(pages, kv, dt=torch.float32))
    small, ref = ops.KvCache.alloc(4, kv, page, hd, DEV), kv_ref.Cache(4, kv, page, hd)
    g = torch.Generator().manual_seed(51)
    k, v = (torch.randn((200, kv * hd), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    ta = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    tb = torch.tensor([[1, 3]], dtype=torch.int32, device=DEV)
    q = torch.randn((2, heads * hd), generator=g).to(torch.bfloat16).to(DEV)
    got = []
    for c, t in ((cache, ta), (small, tb)):
        ops.kv_append(c, k, v, t, zero)
        got.append((*ops.kv_read(c, t, zero, 200, torch.bfloat16), ops.kv_attention(q, c, t, zero + 200, heads=heads)))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    del cache
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------- the operators together
def decode_steps(run, steps, state):
    outs = []
    for i in range(steps):
        outs.append(run(state, i))
    return outs


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
def test_prompt_then_single_tokens(typ):
    """a ragged prompt, then token by token: norm + rotation -> append -> attention, against the 64-bit forms of each on the same inputs"""
    B, heads, kv, hd, page, width, eps = 3, 8, 2, 64, 16, 6, 1e-6
    pages = B * width
    cache, ref = ops.KvCache.alloc(pages, kv, page, hd, DEV), kv_ref.Cache(pages, kv, page, hd)
    table = scatter_table(B, width, pages, 61)
    tab = table.to(DEV)
    g = torch.Generator().manual_seed(62)
    freqs = ops.rope_freqs(hd, 1e6, DEV)
    qg, kg = (1 + 0.2 * torch.randn(hd, generator=g) for _ in range(2))
    lens = [0] * B
    for step, counts in enumerate([[17, 40, 1]] + [[1, 1, 1]] * 5 + [[3, 0, 2]]):
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        qkv = torch.randn((cu[-1], (heads + 2 * kv) * hd), generator=g).to(DT[typ])
        pos = torch.cat([torch.arange(lens[b], lens[b] + counts[b]) for b in range(B)]).to(torch.int32)
        d, p, cud, ln = qkv.to(DEV), pos.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        q, k, v = d[:, :heads * hd], d[:, heads * hd:(heads + kv) * hd], d[:, (heads + kv) * hd:]
        q, k = ops.qk_norm_rope(q, k, p, freqs, qg.to(DEV), kg.to(DEV), heads=heads, kv_heads=kv, eps=eps)
        ops.kv_append(cache, k, v, tab, ln, cud, max_new=max(counts))
        lens = [a + c for a, c in zip(lens, counts)]
        got = ops.kv_attention(q, cache, tab, torch.tensor(lens, dtype=torch.int32, device=DEV), cud, heads=heads, max_new=max(counts))
        ref.append(k.cpu(), v.cpu(), table, [a - c for a, c in zip(lens, counts)], cu)
        same_cache(cache, ref, used_of(table, lens, page))
        want, wv, amax = kv_ref.attention(q.cpu(), ref, table, lens, cu, heads, 1, 0, hd ** -0.5)
        close(got, want, attn_tol(typ, want, wv, amax, max(lens)), "step %d" % step)


def test_captured_steps_replay_with_growing_lengths():
    """one serving step captured; replays with the lengths counted on the device equal eager steps bit for bit, eager work between them"""
    B, heads, kv, hd, page, width = 4, 8, 2, 128, 32, 4
    g = torch.Generator().manual_seed(71)
    steps, start = 6, [30, 0, 63, 5]
    qkv = torch.randn((steps, B, (heads + 2 * kv) * hd), generator=g).to(torch.bfloat16).to(DEV)
    table = scatter_table(B, width, B * width, 72).to(DEV)
    freqs = ops.rope_freqs(hd, device=DEV)

    def fresh():
        cache = ops.KvCache.alloc(B * width, kv, page, hd, DEV)
        pre = torch.randn((sum(start), 2 * kv * hd), generator=torch.Generator().manual_seed(73)).to(torch.bfloat16).to(DEV)
        cu = [0]
        for n in start:
            cu.append(cu[-1] + n)
        ops.kv_append(cache, pre[:, :kv * hd], pre[:, kv * hd:], table, torch.zeros(B, dtype=torch.int32, device=DEV),
                      torch.tensor(cu, dtype=torch.int32, device=DEV))
        return cache, torch.tensor(start, dtype=torch.int32, device=DEV)

    def step(cache, lens, x):
        q, k = ops.qk_norm_rope(x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], lens, freqs, heads=heads, kv_heads=kv)
        ops.kv_append(cache, k, x[:, (heads + kv) * hd:], table, lens)
        lens.add_(1)
        return ops.kv_attention(q, cache, table, lens, heads=heads)

    cache, lens = fresh()
    want = [step(cache, lens, qkv[i]).clone() for i in range(steps)]
    want_cache = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)]
    cache, lens = fresh()
    x = torch.empty_like(qkv[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    keep = lens.clone()
    with torch.cuda.stream(side):
        warm, wl = fresh()
        step(warm, wl, qkv[0])
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = step(cache, lens, x)
    lens.copy_(keep)
    for i in range(steps):
        x.copy_(qkv[i])
        graph.replay()
        junk = ops.kv_attention(qkv[0][:, :heads * hd], warm, table, wl, heads=heads)      # eager work in between
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        del junk
    for a, b in zip(want_cache, (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)):
        assert torch.equal(a, b)


def test_on_another_stream_and_two_at_once():
    B, heads, kv, hd, page, width = 2, 8, 8, 64, 16, 64
    cache, _, table, g = filled(B, width, B * width, kv, page, hd, [1000, 700], 81)
    tab, ln = table.to(DEV), torch.tensor([1000, 700], dtype=torch.int32, device=DEV)
    q = [torch.randn((B, heads * hd), generator=g).to(DEV) for _ in range(2)]
    want = [ops.kv_attention(x, cache, tab, ln, heads=heads) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.kv_attention(q[i], cache, tab, ln, heads=heads))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def every_operator(typ, ragged):
    """one call of each operator on inputs made anew: all outputs, the cache included"""
    B, heads, kv, hd, page, width = 3, 8, 2, 64, 16, 6
    g = torch.Generator().manual_seed(91)
    new = [5, 0, 7] if ragged else [4, 4, 4]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rows = cu[-1]
    cache = ops.KvCache.alloc(B * width, kv, page, hd, DEV)
    table = scatter_table(B, width, B * width, 92).to(DEV)
    wide = torch.randn((rows, (heads + 2 * kv) * hd + 8), generator=g).to(DT[typ]).to(DEV)
    q, k, v = wide[:, :heads * hd], wide[:, heads * hd:(heads + kv) * hd], wide[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    gain = (1 + 0.1 * torch.randn(hd, generator=g)).to(DEV)
    before = torch.tensor([0, 20, 9], dtype=torch.int32, device=DEV)
    cud = torch.tensor(cu, dtype=torch.int32, device=DEV) if ragged else None
    most = dict(max_new=max(new)) if ragged else {}
    freqs = ops.rope_freqs(32, device=DEV)
    outs = list(ops.qk_norm_rope(q, k, pos, freqs, gain, None, heads=heads, kv_heads=kv, interleaved=ragged))
    outs += ops.qk_norm_rope(q, k, None, None, heads=heads, kv_heads=kv, eps=1e-3)
    outs += ops.qk_norm_rope_backward(outs[0], outs[1], q, k, pos, freqs, gain, gain, heads=heads, kv_heads=kv)
    ops.kv_append(cache, k, v, table, before, cud, **most)
    outs += [cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale]
    outs += ops.kv_read(cache, table, before, rows, torch.float16, cud)
    lens = before + torch.tensor(new, dtype=torch.int32, device=DEV)
    outs.append(ops.kv_attention(q, cache, table, lens, cud, heads=heads, window=9, **most))
    outs.append(ops.kv_attention(q, cache, table, lens, cud, heads=heads, causal=0, scale=0.3))
    return outs


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ragged", [False, True])
def test_native_launchers_and_the_python_ones_do_the_same(typ, ragged, monkeypatch):
    taken = []

    class Counted:
        def __init__(self, ext):
            self.ext = ext

        def __getattr__(self, name):
            def call(*a):
                r = getattr(self.ext, name)(*a)
                taken.append((name, r is not None))
                return r
            return call
    real = ops._native
    monkeypatch.setattr(ops, "_native", lambda t: (lambda n: n and (Counted(n[0]), *n[1:]))(real(t)))
    a = every_operator(typ, ragged)
    assert [n for n, ok in taken if ok] == ["qk_norm_rope", "qk_norm_rope", "qk_norm_rope_backward", "kv_append", "kv_read", "kv_attention", "kv_attention"], taken
    monkeypatch.setattr(ops, "_native", lambda t: None)
    b = every_operator(typ, ragged)
    assert len(a) == len(b)
    for i, (x, y) in enumerate(zip(a, b)):
        assert x.dtype is y.dtype and x.shape == y.shape and x.is_contiguous() and not x.requires_grad, i
        assert torch.equal(x, y), i


def test_refusals_on_the_device():
    cache = ops.KvCache.alloc(4, 2, 16, 64, DEV)
    q, lens, table = torch.zeros((2, 8 * 64), device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros((2, 2), dtype=torch.int32, device=DEV)
    odd = torch.zeros((2, 8 * 64 + 1), device=DEV)
    bad = [
        lambda: ops.kv_attention(odd[:, 1:], cache, table, lens, heads=8),                      # misaligned rows
        lambda: ops.kv_attention(q, cache, table, lens, heads=3),                               # heads that kv heads do not divide
        lambda: ops.kv_attention(q, cache, table, lens, heads=8, causal=0, window=4),           # a window needs an order
        lambda: ops.kv_attention(q, cache, table, lens, heads=8, causal=-1),
        lambda: ops.kv_attention(q, cache, table, lens, heads=8, scale=float("nan")),
        lambda: ops.kv_attention(q.double(), cache, table, lens, heads=8),
        lambda: ops.kv_attention(q.cpu(), cache, table, lens, heads=8),
        lambda: ops.kv_append(cache, q[:, :128], q[:, :128], table, lens.long()),
        lambda: ops.kv_append(cache, q[:, :64], q[:, :64], table, lens),
        lambda: ops.qk_norm_rope(q, q, lens, ops.rope_freqs(64, device=DEV).float(), heads=8, kv_heads=8),
        lambda: ops.qk_norm_rope(q, q, lens, ops.rope_freqs(128, device=DEV), heads=8, kv_heads=8),      # more rotated than there is
        lambda: ops.qk_norm_rope(q[:, :480], q[:, :480], lens, None, heads=10, kv_heads=10),            # head_dim 48
        lambda: ops.qk_norm_rope(q, q, lens, None, heads=8, kv_heads=8, eps=-1.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((hip.PgtError, TypeError)):
            f()
            print("not refused:", i)
