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
