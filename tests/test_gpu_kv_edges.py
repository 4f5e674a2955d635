"""Cached-attention operators at the edges of their definitions (include/pgt_hip.h): pages that are not there in front of a page of NaN, sequences with
more rows than the call processes, pages that nobody wrote, scores of any size, broken offsets, caches past 4 GiB at many rows, recorded calls."""
import pytest
import torch

from pgtformer_amd import ops
from tests import kv_ref
from tests.test_gpu_kv import DEV, DT, HALF, TINY, attn_tol, close, filled, gpu_codes
from tests.test_gpu_kv_rows import MANY, attention64, ints, make_cache, offsets, ragged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [0, 1, 3, 4, 7, 10, 12])
@pytest.mark.parametrize("most", [0, 2])
def test_missing_pages_while_page_0_holds_nan(case, most):
    """a token without a page is not seen, whatever the page holds that is read in its place (the first one, another sequence's): here NaN, K and V"""
    B, kv, heads, hd, page, width, n, causal, window, scale, typ = MANY[case]
    n = most or n
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 700 + case)
    table[table == 0] = (set(range(cache.pages)) - set(table.flatten().tolist())).pop() if 0 in table else 0
    assert 0 not in table
    cache.k_pages[0], cache.v_pages[0] = 0xff, 0x7f
    for t in vals:
        t[0] = float("nan")
    for b in range(B):      # in the middle, at the beginning and at the end of what is seen
        for i in {(width // 2 + b) % width, 0 if b % 3 == 0 else width // 2, width - 1 if b % 5 == 0 else width // 3}:
            table[b, i] = (-1, cache.pages, 1 << 30)[(b + i) % 3]
    lens, new = [width * page - b % 5 for b in range(B)], ragged(B, n, 710 + case, 1)
    cu = offsets(new)
    q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
    for order in ((causal, window), (0, 0)):
        want, wv, amax = attention64(q, vals, table, lens, cu, heads, *order, scale)
        got = ops.kv_attention(q, cache, table, ints(lens), ints(cu), heads=heads, causal=order[0], window=order[1], scale=scale, max_new=n)
        assert not bool(want.isnan().any()) and not bool(got.isnan().any()), (order, int(got.isnan().sum()))
        close(got, want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu(), order)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,n,most,heads", [(3, 9, 4, 4), (3, 9, 1, 8), (40, 90, 60, 16)])
def test_more_rows_than_the_call_processes(typ, B, n, most, heads):
    """max_new below a sequence's rows: its first max_new rows, each at the position it has among all of them; the others stay as they were"""
    kv, hd, page, width = 4, 64, 16, 40
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 720)
    lens, new = ragged(B, width * page, 721, n), ragged(B, n, 722, 1)
    cu = offsets(new)
    q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
    done = torch.cat([torch.arange(c) < most for c in new])
    for causal, window in ((1, 0), (1, 40), (16, 0), (0, 0)):
        want, wv, amax = attention64(q, vals, table, lens, cu, heads, causal, window, 0.125)
        out = torch.full((cu[-1], heads * hd), 3.0, dtype=DT[typ], device=DEV)
        got = ops.kv_attention(q, cache, table, ints(lens), ints(cu), heads=heads, causal=causal, window=window, max_new=most, out=out)
        close(got[done.to(DEV)], want.cpu()[done], attn_tol(typ, want, wv, amax, max(lens)).cpu()[done], (causal, window))
        assert bool((got[~done.to(DEV)] == 3).all())


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 64])
def test_pages_that_nobody_wrote_hold_zeros(typ, n):
    """tokens of a fresh cache's pages count in the softmax sum as tokens of zeros do"""
    B, kv, heads, hd, page, width = 40, 2, 16, 64, 32, 12
    g = torch.Generator().manual_seed(730)
    table = torch.arange(B * width, dtype=torch.int32, device=DEV).reshape(B, width)
    fresh, zeros = (ops.KvCache.alloc(B * width, kv, page, hd, DEV) for _ in range(2))
    rows = torch.zeros((B * width * page, kv * hd), device=DEV)
    ops.kv_append(zeros, rows, rows, table, ints([0] * B))
    some = torch.randn((B * page, kv * hd), generator=g).to(DEV)
    for c in (fresh, zeros):      # the second page of every sequence
        ops.kv_append(c, some, some, table, ints([page] * B))
    lens = [width * page - b for b in range(B)]
    q = torch.randn((B * n, heads * hd), generator=g).to(DT[typ]).to(DEV)
    k, v = (t.double().reshape(B, -1, kv, hd) for t in ops.kv_read(fresh, table, ints([0] * B), B * width * page, torch.float32))
    vals = [t.reshape(B * width, page, kv, hd).transpose(1, 2) for t in (k, v)]
    assert bool((vals[1][0] == 0).all()) and bool((vals[1][1] != 0).any())
    cu = [n * b for b in range(B + 1)]
    want, wv, amax = attention64(q, vals, table, lens, cu, heads, 1, 0, 0.3)
    got = [ops.kv_attention(q, c, table, ints(lens), heads=heads, scale=0.3) for c in (fresh, zeros)]
    assert torch.equal(*got)
    close(got[0], want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu())
    # memory that was only cleared: scales of 0
    raw = ops.KvCache(*(torch.zeros_like(t) for t in (fresh.k_pages, fresh.v_pages, fresh.k_scale, fresh.v_scale)))
    ops.kv_append(raw, some, some, table, ints([page] * B))
    assert torch.equal(got[0], ops.kv_attention(q, raw, table, ints(lens), heads=heads, scale=0.3))


@pytest.mark.parametrize("scale", [3e6, 5e7, 2e8, 7e9, 1e14, 3e31])
@pytest.mark.parametrize("case,n", [(0, 0), (1, 0), (3, 0), (4, 0), (10, 0), (12, 0), (3, 1), (11, 2)])
def test_scores_of_any_size(case, n, scale):
    """finite scores, far apart: the row of the largest, whatever their size and sign.  Differences of distinct scores are beyond the exponential's range,
    so the weights are 1 and 0: what is left is the rounding of the one weight in the product (half: 2^-11; fp32: two halves 2^-22, and the quotient's
    two roundings) and of the output."""
    B, kv, heads, hd, page, width, most, causal, window, _, typ = MANY[case]
    most = n or most
    causal, window = 0, 0
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 740 + case)
    lens, new = [width * page - b % 7 for b in range(B)], ragged(B, most, 741, 1)
    cu = offsets(new)
    for sign in (1, -1):      # the second time: all products of one sign, so that every score is far below zero
        q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
        if sign < 0:
            q = q.abs()
            cache.k_pages.bitwise_and_(0x7f)
            vals[0].abs_()
        # the largest and the second largest score of every row and head, in 64 bits
        want, best = torch.zeros((cu[-1], heads, hd), dtype=torch.float64, device=DEV), torch.zeros((cu[-1], heads), dtype=torch.bool, device=DEV)
        for b in range(B):
            k, v = (t[table[b].long()].transpose(1, 2).reshape(-1, kv, hd)[:lens[b]] for t in vals)
            for h in range(heads):
                hk = h * kv // heads
                qq = q[cu[b]:cu[b + 1], h * hd:(h + 1) * hd].double()
                kt = k[:, hk].t().contiguous()
                x = torch.matmul(qq, kt) * (sign * scale)
                top, at = x.topk(2, -1)
                bound = 2.0 ** -15 * torch.matmul(qq.abs(), kt.abs()).amax(-1) * scale      # far above the fp32 sums' rounding
                best[cu[b]:cu[b + 1], h] = top[:, 0] - top[:, 1] > bound + 1000
                want[cu[b]:cu[b + 1], h] = v[at[:, 0], hk]
        got = ops.kv_attention(q, cache, table, ints(lens), ints(cu), heads=heads, causal=causal, window=window, scale=sign * scale, max_new=most)
        assert bool(torch.isfinite(got).all()), (sign, int((~torch.isfinite(got)).sum()))
        pick = best[..., None].expand_as(want).reshape(cu[-1], -1)
        assert bool(best.any())
        want = want.reshape(cu[-1], -1)
        tol = (HALF[typ] + 2.0 ** (-21 if typ == "f32" else -11)) * (1 + 2.0 ** -7) * want.abs() + TINY[typ]
        close(got[pick], want[pick].cpu(), tol[pick].cpu(), sign)


def test_broken_offsets_are_bounded_and_what_they_leave_is_processed():
    """descending, negative, past the end: a sequence owns what is left of its range inside the rows"""
    heads, kv, hd, page, pages = 4, 2, 64, 16, 12
    cache, ref, table, g = filled(3, 4, pages, kv, page, hd, [64, 64, 64], 31)
    tab = table.clone()
    tab[2] = -7
    q = torch.randn((13, heads * hd), generator=g)
    out = torch.full((13, heads * hd), 2.0, device=DEV)
    ops.kv_attention(q.to(DEV), cache, tab.to(DEV), ints([60, 60, 60]), ints([9, 3, -1, 500]), heads=heads, out=out)
    assert bool((out == 0).all())      # all 13 rows are the last sequence's, which has no page
    out.fill_(2.0)
    ops.kv_attention(q.to(DEV), cache, table.to(DEV), ints([60, 60, 60]), ints([9, 3, -1, 500]), heads=heads, out=out)
    want, wv, amax = kv_ref.attention(q, ref, table, [60, 60, 60], [0, 0, 0, 13], heads, 1, 0, 0.125)
    close(out, want, attn_tol("f32", want, wv, amax, 60))
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)]
    k = torch.randn((40, kv * hd), generator=g)
    tab = torch.tensor([[2, -1, 1 << 30], [pages, -5, 4]], dtype=torch.int32)
    ops.kv_append(cache, k.to(DEV), k.to(DEV), tab.to(DEV), ints([0, 0]), ints([30, -4, 1000]))
    # the first sequence owns nothing, the second all 40 rows: its tokens 32 .. 39 are on page 4
    for old, now in zip(before, (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)):
        assert [i for i in range(pages) if not torch.equal(old[i], now[i])] == [4]
    part = kv_ref.Cache(pages, kv, page, hd)
    part.append(k[32:], k[32:], torch.tensor([[4]]), [0], [0, 8])
    codes, scales = gpu_codes(cache)
    for w in range(2):
        assert torch.equal(codes[w][4], part.code[w][4]) and torch.equal(scales[w][4], torch.exp2(part.e[w][4].double()))


@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_many_rows_past_32_bits(typ):
    """the 256-column kernel on pages behind 4 GiB, NaN values among them, against the same tokens in a small cache"""
    kv, hd, page, heads, rows, length = 8, 128, 128, 256, 200, 300
    pages = 33000      # x 128 KiB = 4.03 GiB
    mk = lambda *s, dt=torch.uint8: torch.empty(s, dtype=dt, device=DEV)      # noqa: E731
    cache = ops.KvCache(mk(pages, kv, hd // 16, page, 16), mk(pages, kv, page // 16, hd, 16), mk(pages, kv, dt=torch.float32), mk(pages, kv, dt=torch.float32))
    small = ops.KvCache.alloc(4, kv, page, hd, DEV)
    cache.v_pages[0], cache.k_pages[0] = 0x7f, 0x7f
    g = torch.Generator().manual_seed(751)
    k, v = (torch.randn((length, kv * hd), generator=g).to(DT[typ]).to(DEV) for _ in range(2))
    zero = ints([0])
    ta, tb = ints([[pages - 1, pages - 2, pages - 3]]), ints([[1, 3, 2]])
    q = torch.randn((rows, heads * hd), generator=g).to(DT[typ]).to(DEV)
    for nan in (False, True):
        got = []
        for c, t in ((cache, ta), (small, tb)):
            ops.kv_append(c, k, v, t, zero)
            if nan:
                pid = int(t[0, 1])
                c.v_pages[pid, 3, 5, 77, 9] = 0x7f      # token 128 + 5 * 16 + 9 = 217 of kv head 3
            got.append(ops.kv_attention(q, c, t, zero + length, heads=heads))
        assert torch.equal(got[0].isnan(), got[1].isnan()) and torch.equal(got[0].nan_to_num(), got[1].nan_to_num())
        hit = torch.zeros_like(got[0], dtype=torch.bool).reshape(rows, heads, hd)
        if nan:
            hit[217 - (length - rows):, 3 * 32:4 * 32, 77] = True
        assert torch.equal(got[0].isnan(), hit.reshape(rows, -1))
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("case", range(len(MANY)))
def test_which_kernel_the_cases_of_many_rows_reach(case):
    """the 256-column kernel runs in all of them but fp32 at 128 dims"""
    B, kv, heads, hd, page, width, most, causal, window, scale, typ = MANY[case]
    cache, _, table, g = make_cache(B, width, kv, page, hd, 760)
    q = torch.zeros((B * most, heads * hd), dtype=DT[typ], device=DEV)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        ops.kv_attention(q, cache, table, ints([width * page] * B), heads=heads, causal=causal, window=window, scale=scale)
        torch.cuda.synchronize()
    names = [e.name for e in prof.events() if "kv_attn" in e.name]
    if not names:
        pytest.skip("the profiler recorded no kernel")
    assert any("kv_attn_rows_kernel" in n for n in names) == (not (typ == "f32" and hd == 128)), names


def test_recorded_calls_replay_from_the_file(tmp_path):
    """norm + rotation, append and attention as a program: a replay gives what the recorded calls gave.  The cache and the lengths in the file are those of
    the moment the file was written, so the file is written before the recorded calls' own effects (the tokens they append are the same)"""
    from pgtformer_amd import export
    B, heads, kv, hd, page, width = 2, 8, 2, 64, 16, 4
    cache, _, table, g = filled(B, width, B * width, kv, page, hd, [30, 17], 771)
    tab, before, after = table.to(DEV), ints([30, 17]), ints([31, 18])
    freqs = ops.rope_freqs(hd, device=DEV)
    qkv = torch.randn((B, (heads + 2 * kv) * hd), generator=g).to(torch.bfloat16).to(DEV)
    raw, out = qkv.view(torch.uint8), torch.zeros((B, heads * hd), dtype=torch.bfloat16, device=DEV)

    def step():
        q, k = ops.qk_norm_rope(qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], before, freqs, heads=heads, kv_heads=kv)
        ops.kv_append(cache, k, qkv[:, (heads + kv) * hd:], tab, before)
        return ops.kv_attention(q, cache, tab, after, heads=heads, out=out)
    keep = (cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    state = [t.clone() for t in keep]
    persistent = export._live_cuda_storages(DEV)
    calls, _ = export.record(step, DEV)
    want = out.clone()
    for t, was in zip(keep, state):
        t.copy_(was)
    tape, layout, work = export.build_program(calls, persistent, raw, out.view(torch.uint8))
    path = str(tmp_path / "step.prog")
    export.write_program(path, tape, layout, work, raw.numel(), out.view(torch.uint8).numel(), storages=persistent)
    assert len(tape) == 3
    got = export.run_program(path, raw)
    assert torch.equal(got.view(torch.bfloat16).reshape(out.shape), want)


def test_captured_gradient_and_read():
    """a norm + rotation with its gradient, and the read of a cache, captured: every replay on new values gives what the eager calls give"""
    rows, heads, kv, hd, page, width = 700, 8, 2, 64, 16, 4
    g = torch.Generator().manual_seed(781)
    cache, _, table, _ = filled(2, width, 2 * width, kv, page, hd, [60, 33], 782)
    tab, start, freqs = table.to(DEV), ints([3, 0]), ops.rope_freqs(32, device=DEV)
    x = torch.empty((rows, (heads + kv) * hd), dtype=torch.float16, device=DEV)
    dy, pos, gain = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device=DEV), torch.ones(hd, device=DEV)

    def step():
        q, k, dq, dk = x[:, :heads * hd], x[:, heads * hd:], dy[:, :heads * hd], dy[:, heads * hd:]
        kw = dict(heads=heads, kv_heads=kv)
        return [*ops.qk_norm_rope(q, k, pos, freqs, gain, gain, **kw), *ops.qk_norm_rope_backward(dq, dk, q, k, pos, freqs, gain, gain, **kw),
                *ops.kv_read(cache, tab, start, 60, torch.float16)]

    def fill():
        x.copy_(torch.randn(x.shape, generator=g))
        dy.copy_(torch.randn(x.shape, generator=g))
        pos.copy_(torch.randint(0, 1 << 20, (rows,), generator=g))
        gain.copy_(torch.rand(hd, generator=g))
        start.copy_(torch.randint(0, 30, (2,), generator=g))
    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(4):
        fill()
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert len(outs) == 8
        for i, (a, b) in enumerate(zip(outs, want)):      # (tokens behind the last one of `filled` read as NaN)
            assert (i > 5 or not bool(b.isnan().any())) and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()), i


def test_norm_and_rotation_of_more_rows_than_a_grid_has_blocks():
    """2^26 rows and some: workgroups take several blocks of tokens; the last rows against a call of their own, the rows between by a sample"""
    rows, hd, n = (1 << 26) + 4099, 32, 5000
    x = torch.empty((rows, 2 * hd), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(DEV).manual_seed(791)
    for at in range(0, rows, 1 << 24):
        x[at:at + (1 << 24)].normal_(generator=g)
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    kw = dict(heads=1, kv_heads=1)
    freqs = ops.rope_freqs(hd, device=DEV)
    q, k = ops.qk_norm_rope(x[:, :hd], x[:, hd:], pos, freqs, **kw)
    for part in (slice(rows - n, rows), slice(0, n), slice((1 << 24) - 7, (1 << 24) + n), slice((1 << 26) - 2500, (1 << 26) + 2500)):
        a, b = ops.qk_norm_rope(x[part, :hd], x[part, hd:], pos[part], freqs, **kw)
        assert torch.equal(a, q[part]) and torch.equal(b, k[part])
    del x, q, k, pos
    torch.cuda.empty_cache()


@pytest.mark.parametrize("case", [0, 3, 10, 12])
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** -90])
def test_queries_of_any_size(case, size):
    """queries and scale that only together give ordinary scores (size a power of two: the same roundings as without it)"""
    B, kv, heads, hd, page, width, most, causal, window, scale, typ = MANY[case]
    typ = "bf16" if typ == "f16" else typ
    cache, vals, table, g = make_cache(B, width, kv, page, hd, 800 + case)
    lens, new = [width * page - b % 7 for b in range(B)], ragged(B, most, 801, 1)
    cu = offsets(new)
    q = torch.randn((cu[-1], heads * hd), generator=g, device=DEV).to(DT[typ])
    kw = dict(heads=heads, causal=causal, window=window, max_new=most)
    want, wv, amax = attention64(q, vals, table, lens, cu, heads, causal, window, scale)
    got = ops.kv_attention(q * size, cache, table, ints(lens), ints(cu), scale=scale / size, **kw)
    close(got, want.cpu(), attn_tol(typ, want, wv, amax, max(lens)).cpu())
