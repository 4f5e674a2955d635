"""Attention over the 8-bit cache at the sizes where many query rows share a workgroup, and with its work cut into pieces over all
sequences, against a plain 64-bit form (batched on the device; tests/test_gpu_kv.py has the derivation of the tolerances)."""
import pytest
import torch

from pgtformer_amd import hip, ops
from tests.test_gpu_kv import DEV, DT, attn_tol, close

pytestmark = pytest.mark.gpu


def make_cache(B, width, kv, page, hd, seed):
    """a cache of random values (per page and head another scale), its values float64 (pages, kv, page, hd), a scattered table"""
    g = torch.Generator(DEV).manual_seed(seed)
    pages = B * width + 1
    cache = ops.KvCache.alloc(pages, kv, page, hd, DEV)
    vals = []
    for w, (p, s) in enumerate(((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale))):
        e = torch.randint(5, 9, (pages, kv), generator=g, device=DEV).float()
        x = torch.randn((pages, kv, page, hd), generator=g, device=DEV)
        if w:
            x *= torch.exp(torch.randn((pages, kv, page, 1), generator=g, device=DEV))
        code = (x * torch.exp2(e)[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        s.copy_(torch.exp2(-e))
        b = code.view(torch.uint8)
        if w:
            p.copy_(b.reshape(pages, kv, page // 16, 16, hd).transpose(3, 4))
        else:
            p.copy_(b.reshape(pages, kv, page, hd // 16, 16).transpose(2, 3))
        vals.append(code.double() * torch.exp2(-e.double())[..., None, None])
    table = torch.randperm(pages, generator=g, device=DEV)[: B * width].reshape(B, width).to(torch.int32)
    return cache, vals, table, g


def attention64(q, vals, table, lens, cu, heads, causal, window, scale):
    """(out, sum of weights * |v|, largest sum |q k| scale) float64 of (rows, heads, hd); NaN in V reaches the queries that see it"""
    kv, page, hd = vals[0].shape[1:]
    rows, group, pages = q.shape[0], heads // kv, vals[0].shape[0]
    q = q.double().reshape(rows, heads, hd)
    out, wv, amax = (torch.zeros((rows, heads, hd), dtype=torch.float64, device=DEV) for _ in range(3))
    for b in range(table.shape[0]):
        n, length = cu[b + 1] - cu[b], min(max(lens[b], 0), table.shape[1] * page)
        if n <= 0 or length == 0:
            continue
        ids = table[b].long()
        good = (ids >= 0) & (ids < pages)
        pick = ids.clamp(0, pages - 1)
        k, v = (t[pick].transpose(1, 2).reshape(-1, kv, hd)[:length] for t in vals)
        have = good.repeat_interleave(page)[:length]
        i, j = torch.arange(n, device=DEV)[:, None], torch.arange(length, device=DEV)[None]
        p = length - n + i
        end = (p // causal + 1) * causal if causal else torch.full_like(p, length)
        see = have & (j < end) & (j >= (end - window if window else 0)) & (p >= 0)
        for h in range(kv):
            qq = q[cu[b]:cu[b + 1], h * group:(h + 1) * group].transpose(0, 1)      # (group, n, hd)
            kt = k[:, h].t().contiguous()
            x = torch.matmul(qq, kt) * scale
            m = see[None].expand_as(x)
            kn = (see & kt.isnan().any(0)[None]).any(1)
            w = torch.where(m, x, torch.full_like(x, -float("inf")))
            w = torch.softmax(w, -1).nan_to_num(0.0)      # (a row that sees nothing)
            vn = v[:, h].isnan().double()
            vv = v[:, h].nan_to_num(0.0)
            o = torch.matmul(w, vv)
            o = torch.where((torch.matmul(see.double(), vn) > 0)[None], torch.full_like(o, float("nan")), o)
            o[:, kn] = float("nan")
            sl = (slice(cu[b], cu[b + 1]), slice(h * group, (h + 1) * group))
            out[sl] = o.transpose(0, 1)
            wv[sl] = torch.matmul(w, vv.abs()).transpose(0, 1)
            a = torch.where(m, torch.matmul(qq.abs(), kt.abs().nan_to_num(0.0)) * abs(scale), torch.zeros_like(x))
            amax[sl] = a.amax(-1, keepdim=True).transpose(0, 1)
    return [t.reshape(rows, -1) for t in (out, wv, amax)]


def ragged(B, most, seed, least=0):
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(least, most + 1, (B,), generator=g).tolist()
    v[B // 2] = most
    return v


def offsets(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# B, kv, heads, hd, page, pages of a sequence, most new tokens, causal, window, scale, type
MANY = [
    (64, 8, 32, 64, 32, 13, 41, 1, 0, 0.125, "bf16"),        # a workgroup per column tile
    (64, 4, 20, 128, 128, 4, 37, 0, 0, -0.09, "f16"),        # every token, a negative scale, 5 heads to a kv head
    (64, 8, 24, 64, 16, 26, 50, 50, 0, 0.2, "f16"),          # whole blocks of 50
    (33, 8, 32, 128, 16, 44, 64, 1, 0, 0.088, "bf16"),       # pieces of the line
    (33, 8, 32, 64, 64, 16, 63, 16, 600, 0.125, "f16"),      # a window over blocks
    (33, 8, 32, 64, 64, 16, 63, 1, 130, 0.125, "bf16"),      # a short window: 4 tiles at most
    (33, 8, 32, 128, 32, 30, 64, 1, 701, 0.0, "f16"),        # scale 0: the mean of what is seen
    (1, 8, 32, 64, 64, 313, 100, 1, 0, 0.125, "f16"),        # one long sequence, its segments cut many times
    (2, 8, 64, 128, 32, 70, 300, 1, 0, 0.09, "bf16"),
    (5, 1, 8, 64, 128, 9, 1100, 7, 90, 0.3, "bf16"),         # 35 column tiles, a window in which most rows see two tiles
    (64, 8, 32, 64, 32, 13, 41, 1, 0, 0.125, "f32"),
    (33, 8, 32, 64, 64, 16, 63, 16, 600, -0.125, "f32"),
    (64, 4, 20, 128, 128, 4, 37, 0, 0, 0.09, "f32"),         # (fp32 of 128 dims: 16 columns)
]


@pytest.mark.parametrize("case", range(len(MANY)))
@pytest.mark.parametrize("nan", [False, True])
def test_many_rows(case, nan):
    B, kv, heads, hd, page, width, most, causal, window, scale, typ = MANY[case]
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 100 + case)
    lens, new = ragged(B, width * page - 3, 200 + case), ragged(B, most, 300 + case)
    if B > 4:
        lens[0], new[1], lens[2], new[2] = 0, 0, 1, most            # no token, no row, more rows than tokens
        lens[3], new[3] = min(65, width * page), min(2, most)
    cu = offsets(new)
    if B > 8:
        table[4, 1], table[5, 0], table[6, width - 1] = -1, cache.pages, 1 << 30      # pages that are not there
        table[7] = -3
    q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
    if nan:      # keys of one token and values of some, in tiles that all, some and no columns of a workgroup see
        for b in range(0, B, 3):
            for t, which in ((0, 1), (max(lens[b] - 1, 0), 1), (max(lens[b] - most, 0), 1), (max(lens[b] // 2, 0), 1), (max(lens[b] - 2, 0), 0)):
                pid = int(table[b, min(t // page, width - 1)])
                if not 0 <= pid < cache.pages:
                    continue
                s, h, d = t % page, b % kv, (7 * b + t) % hd
                if which:
                    cache.v_pages[pid, h, s // 16, d, s % 16] = 0x7f if b % 2 else 0xff
                else:
                    cache.k_pages[pid, h, d // 16, s, d % 16] = 0x7f
                vals[which][pid, h, s, d] = float("nan")
    want, wv, amax = attention64(q, vals, table, lens, cu, heads, causal, window, scale)
    args = (cache, table, ints(lens), ints(cu))
    kw = dict(heads=heads, causal=causal, window=window, scale=scale, max_new=most)
    got = ops.kv_attention(q, *args, **kw)
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    assert nan or not bool(got.isnan().any())
    ok = ~want.isnan()
    tol = attn_tol(typ, want, wv, amax, max(lens))
    close(got[ok], want[ok].cpu(), tol[ok].cpu(), "case %d" % case)
    assert torch.equal(got.nan_to_num(), ops.kv_attention(q, *args, **kw).nan_to_num())
    # in place, and rows behind the last sequence stay as they were
    pad = torch.cat([q, torch.full((9, heads * hd), 5.0, device=DEV).to(DT[typ])])
    same = ops.kv_attention(pad, *args, **kw, out=pad)
    assert same is pad and torch.equal(same[:cu[-1]].nan_to_num(), got.nan_to_num()) and bool((pad[cu[-1]:] == 5).all())


def test_the_cases_reach_both_ways_of_sharing():
    """workspaces tell: some of the cases above run a workgroup per column tile (none), some in pieces (one)"""
    f = hip.lib().pgt_kv_attention_workspace_bytes
    size = [f(ops._dt(torch.empty(0, dtype=DT[c[10]])), c[0], c[6], c[2], c[1], c[3], c[5], c[4], c[7], c[8]) for c in MANY]
    assert [s > 0 for s in size] == [False, False, False, True, True, False, True, True, True, False, False, True, False], size


@pytest.mark.parametrize("case", [0, 1, 2, 3, 4, 6, 7, 10])
@pytest.mark.parametrize("low", [None, -32, -18])
def test_values_whose_pages_differ_in_scale(case, low):
    """V pages of nothing but zeros (the least scale, 2^-32) or 2^11 .. 2^26 smaller than the others: their tokens still count in the softmax sum,
    whatever their weight times their scale is to the largest's"""
    B, kv, heads, hd, page, width, most, causal, window, scale, typ = MANY[case]
    causal, window = 0, 0      # every row sees many pages
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 400 + case)
    small = torch.rand((cache.pages, kv), generator=g, device=DEV) < 0.5
    if low is None:
        cache.v_pages[small] = 0
        vals[1][small] = 0
    e = -32 if low is None else low
    was = cache.v_scale.double()
    cache.v_scale[small] = 2.0 ** e
    vals[1] *= torch.where(small, 2.0 ** e / was, torch.ones_like(was))[..., None, None]
    lens, new = [width * page - b % 7 for b in range(B)], ragged(B, most, 500 + case, 1)
    cu = offsets(new)
    q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
    want, wv, amax = attention64(q, vals, table, lens, cu, heads, causal, window, scale)
    got = ops.kv_attention(q, cache, table, ints(lens), ints(cu), heads=heads, causal=causal, window=window, scale=scale, max_new=most)
    close(got, want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu(), "case %d" % case)


def test_many_segments_of_few_rows():
    """more (sequence, column tile) pairs than a workgroup looks up at once, most of them empty; single tokens in pieces"""
    kv, heads, hd, page, width, B, most = 2, 8, 64, 16, 70, 300, 9
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 1)
    lens, new = ragged(B, width * page, 2), ragged(B, most, 3)
    for b in range(40, 290):
        new[b] = 0
    for b in range(0, 30):
        lens[b] = b % 3
    cu = offsets(new)
    for typ in ("bf16", "f32"):
        q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
        want, wv, amax = attention64(q, vals, table, lens, cu, heads, 1, 0, 0.125)
        got = ops.kv_attention(q, cache, table, ints(lens), ints(cu), heads=heads, max_new=most)
        close(got, want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu(), typ)


@pytest.mark.parametrize("typ,hd,group,width", [("bf16", 128, 4, 300), ("f16", 64, 5, 260), ("f32", 64, 1, 300), ("f32", 128, 8, 130), ("bf16", 64, 16, 64)])
@pytest.mark.parametrize("B", [1, 3, 17])
def test_single_tokens_of_long_sequences(typ, hd, group, width, B):
    page, kv = 32, 4
    heads = kv * group
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 17)
    lens = ragged(B, width * page - 5, 18 + B, 1)
    q = torch.randn((B, heads * hd), generator=g, device=DEV).to(DT[typ])
    for window in (0, 1500):
        want, wv, amax = attention64(q, vals, table, lens, list(range(B + 1)), heads, 1, window, hd ** -0.5)
        got = ops.kv_attention(q, cache, table, ints(lens), heads=heads, window=window)
        close(got, want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu(), "window %d" % window)


def test_captured_calls_share_nothing():
    """two captured graphs of calls that need a workspace, replayed in turn with eager calls between them and with other lengths"""
    kv, heads, hd, page, width = 8, 32, 64, 64, 160
    shapes = ((1, 100, "f16"), (2, 1, "bf16"))
    graphs = []
    for i, (B, n, typ) in enumerate(shapes):
        cache, vals, table, g = make_cache(B, width, kv, page, hd, 30 + i)
        q = torch.randn((B * n, heads * hd), generator=g, device=DEV).to(DT[typ])
        lens = ints([width * page] * B)
        call = (lambda q=q, cache=cache, table=table, lens=lens: ops.kv_attention(q, cache, table, lens, heads=heads))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, call, lens))
    for step, lengths in enumerate((9000, 200, 10240, 1, 0, 5000)):
        for graph, out, call, lens in graphs:
            lens.fill_(lengths)
        want = [call().clone() for _, _, call, _ in graphs]
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out, _, _), w in zip(graphs, want):
            assert torch.equal(out, w), step
