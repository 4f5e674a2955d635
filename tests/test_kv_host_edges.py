"""Cached-attention operators without a GPU: what a fresh cache holds, outputs that a caller may not pass"""
import pytest
import torch

from pgtformer_amd import hip, ops


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
