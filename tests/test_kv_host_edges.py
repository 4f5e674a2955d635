"""Cached-attention operators without a GPU: what a fresh cache holds, outputs that a caller may not pass, sizes of more than 31 bits, grids of more threads than a
launch can have"""
import pytest
import torch

from pgtformer_amd import hip, ops
from tests.test_kv_host import P, refused


def test_a_fresh_cache_holds_zeros_under_a_valid_scale():
    """the least scale, as kv_append gives zeros; 0 would be outside the scales' range"""
    c = ops.KvCache.alloc(5, 3, 32, 128, "cpu")
    for pages, scale in ((c.k_pages, c.k_scale), (c.v_pages, c.v_scale)):
        assert not bool(pages.any()) and torch.equal(scale, torch.full((5, 3), 2.0 ** -32))


def test_an_output_is_no_other_outputs_input():
    """q's output written over k (or k's gradient over dq) is read by other workgroups later; the same tensor twice is no two outputs"""
    q, k, dq, dk = (torch.zeros(4, 512) for _ in range(4))
    pos, f = torch.zeros(4, dtype=torch.int32), ops.rope_freqs(64, device="cpu")
    kw = dict(heads=8, kv_heads=8)
    for a, b, out in ((q, k, (k, q)), (q, k, (q, q)), (q, k, (k, k)), (q, k, (k, torch.zeros(4, 512))), (q, k, (torch.zeros(4, 512), q)),
                      (q, q, (q, q)), (q, q, (q, torch.zeros(4, 512))), (q, k, (dq, dq))):
        with pytest.raises(hip.PgtError, match="overlaps"):
            ops.qk_norm_rope(a, b, pos, f, **kw, out=out)
    for out in ((dk, dq), (k, q), (dk, q), (dq, q), (dq, dq), (torch.zeros(4, 512), dq)):
        with pytest.raises(hip.PgtError, match="overlaps"):
            ops.qk_norm_rope_backward(dq, dk, q, k, pos, f, **kw, out=out)
    wide = torch.zeros(4, 2048)
    a, b, c, d = wide.chunk(4, 1)
    for outs, ins in (((q, k), (q, k)), ((dq, dk), (dq, dk, q, k)), ((q, k), (dq, dk, q, k)), ((dq, k), (dq, dk, q, k)), ((a, b), (a, b)), ((c, d), (a, b)),
                      ((a, d), (a, b, c, d)), ((q,), (q,)), ((q, k), ())):
        ops._apart(outs, ins, "t")
    for outs, ins in (((b, a), (a, b)), ((a, a), ()), ((b, d), (a, b, c, d)), ((wide[:, 8:520], d), (a, b))):
        with pytest.raises(hip.PgtError, match="overlaps"):
            ops._apart(outs, ins, "t")


def test_sizes_past_31_bits_are_refused():
    """the C entry points take int32: a stride of 2^32 + 512 would arrive there as 512, a window of 2^32 + 5 as 5"""
    far = lambda *shape, ld, dt=torch.float32: torch.empty_strided(shape, (ld, 1), dtype=dt, device="meta")      # noqa: E731
    c = ops.KvCache.alloc(4, 2, 16, 64, "cpu")
    q, k, lens, table = torch.zeros(4, 512), torch.zeros(4, 128), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 2), dtype=torch.int32)
    for ld in (1 << 31, (1 << 32) + 512):
        for call in (lambda: ops.kv_attention(far(4, 512, ld=ld), c, table, lens, heads=8), lambda: ops.kv_attention(q, c, table, lens, heads=8, out=far(4, 512, ld=ld)),
                     lambda: ops.kv_attention(q, c, far(2, 2, ld=ld, dt=torch.int32), lens, heads=8), lambda: ops.kv_append(c, far(4, 128, ld=ld), k, table, lens),
                     lambda: ops.kv_append(c, k, far(4, 128, ld=ld), table, lens),
                     lambda: ops.kv_read(c, table, lens, 4, torch.float32, out=(far(4, 128, ld=ld), k)),
                     lambda: ops.qk_norm_rope(far(4, 512, ld=ld), k, None, None, heads=8, kv_heads=2),
                     lambda: ops.qk_norm_rope_backward(q, far(4, 128, ld=ld), q, k, None, None, heads=8, kv_heads=2)):
            with pytest.raises(hip.PgtError, match="31 bits"):
                call()
    for rows in (1 << 31, 1 << 33):
        with pytest.raises(hip.PgtError, match="31 bits"):
            ops.kv_read(c, table, lens, rows, torch.float32)
    for kw in (dict(window=1 << 32), dict(window=(1 << 32) + 5), dict(causal=(1 << 32) + 1), dict(causal=1 << 31), dict(causal=-1), dict(window=-1)):
        with pytest.raises(hip.PgtError, match="causal="):
            ops.kv_attention(q, c, table, lens, heads=8, **kw)


def test_launches_of_2_to_the_32_threads_are_refused():
    """ragged rows without max_new ask for a launch that covers all rows of every sequence"""
    kv = dict(dtype=0, k=P, ldk=512, v=P, ldv=512, kp=P, vp=P, ks=P, vs=P, pages=4, page=16, kv=8, hd=64, table=P, ldt=8, width=8, lens=P, cu=P, B=64,
              rows=1 << 20, n=1 << 20, stream=None)      # 2^26 workgroups of 64 threads
    for name in ("pgt_kv_append", "pgt_kv_read"):
        refused(name, kv, [dict(), dict(page=128, hd=128, ldk=1024, ldv=1024, B=512)])      # 2^26 of 512
    att = dict(dtype=0, q=P, ldq=512, kp=P, vp=P, ks=P, vs=P, pages=4, page=16, kv=8, hd=64, table=P, ldt=3, width=3, lens=P, cu=P, B=2048, rows=1 << 16, n=1 << 16,
               heads=8, scale=0.1, causal=1, window=0, out=P, ldo=512, ws=P, nb=1 << 30, stream=None)      # 2^22 workgroups of 512 threads, or 2^26 of 256
    refused("pgt_kv_attention", att, [dict(B=4096), dict(dtype=1, B=4096), dict(dtype=0, B=1 << 14, rows=1 << 18, n=1 << 14, hd=128, ldq=1024, ldo=1024)])


def test_a_scale_that_leaves_fp32_is_refused():
    att = dict(dtype=0, q=P, ldq=512, kp=P, vp=P, ks=P, vs=P, pages=4, page=16, kv=2, hd=64, table=P, ldt=3, width=3, lens=P, cu=None, B=2, rows=8, n=4,
               heads=8, scale=0.1, causal=1, window=0, out=P, ldo=512, ws=P, nb=1 << 30, stream=None)
    refused("pgt_kv_attention", att, [dict(scale=2.5e38), dict(scale=-3.4e38)])      # times log2 e: infinite
