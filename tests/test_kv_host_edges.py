"""Cached-attention operators without a GPU: what a fresh cache holds"""
import torch

from pgtformer_amd import ops


def test_a_fresh_cache_holds_zeros_under_a_valid_scale():
    """the least scale, as kv_append gives zeros; 0 would be outside the scales' range"""
    c = ops.KvCache.alloc(5, 3, 32, 128, "cpu")
    for pages, scale in ((c.k_pages, c.k_scale), (c.v_pages, c.v_scale)):
        assert not bool(pages.any()) and torch.equal(scale, torch.full((5, 3), 2.0 ** -32))
