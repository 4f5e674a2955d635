"""Cached-attention operators without a GPU: refusals of the Python layer and of the C entry points (every call here is refused before a
launch), workspace sizes, the 64-bit reference forms against each other."""
import ctypes as C
import math

import pytest
import torch

from pgtformer_amd import hip, ops
from tests import kv_ref


def cache(pages=4, kv=2, page=16, hd=64):
    return ops.KvCache.alloc(pages, kv, page, hd, "cpu")


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_cache_layout_and_its_refusals():
    c = cache(5, 3, 32, 128)
    assert c.k_pages.shape == (5, 3, 8, 32, 16) and c.v_pages.shape == (5, 3, 2, 128, 16) and c.k_scale.shape == (5, 3)
    assert (c.pages, c.page, c.kv_heads, c.hd) == (5, 32, 3, 128)
    for kw in (dict(page=24), dict(page=256), dict(hd=96), dict(pages=0), dict(kv=0)):
        with pytest.raises(hip.PgtError):
            cache(**kw)
    good = (c.k_pages, c.v_pages, c.k_scale, c.v_scale)
    for i, t in ((0, c.k_pages[..., 0]), (0, c.k_pages.float()), (1, c.v_pages[:4]), (1, c.k_pages), (2, c.k_scale[:, :2]), (3, c.v_scale.double()),
                 (2, c.k_scale.t()), (0, c.k_pages.transpose(0, 1))):
        with pytest.raises(hip.PgtError):
            ops.KvCache(*good[:i], t, *good[i + 1:])


def test_tensors_off_the_gpu_are_refused():
    c, q, lens, table = cache(), torch.zeros(2, 8 * 64), i32(2), i32(2, 2)
    kv = torch.zeros(2, 2 * 64)
    for f in (lambda: ops.kv_attention(q, c, table, lens, heads=8), lambda: ops.kv_append(c, kv, kv, table, lens),
              lambda: ops.kv_read(c, table, lens, 2, torch.float32), lambda: ops.qk_norm_rope(q, q, None, None, heads=8, kv_heads=8),
              lambda: ops.qk_norm_rope_backward(q, q, q, q, None, None, heads=8, kv_heads=8)):
        with pytest.raises(hip.PgtError, match="GPU"):
            f()


def test_argument_refusals_of_the_python_layer():
    c, lens, table = cache(), i32(2), i32(2, 2)
    q, kv = torch.zeros(4, 8 * 64), torch.zeros(4, 2 * 64)
    f = ops.rope_freqs(64, device="cpu")
    wide = torch.zeros(4, 20 * 64)
    bad = [
        lambda: ops.kv_attention(q[:, :64], c, table, lens, heads=8),                       # wrong width
        lambda: ops.kv_attention(q[:3], c, table, lens, heads=8),                           # 3 rows over 2 sequences
        lambda: ops.kv_attention(q, c, table, lens, heads=8, max_new=5),                    # not rows / B
        lambda: ops.kv_attention(q, c, table, lens, i32(2), heads=8),                       # cu of B entries
        lambda: ops.kv_attention(q, c, table, lens, i32(3), heads=8, max_new=9),            # more than there are rows
        lambda: ops.kv_attention(q, c, table.long(), lens, heads=8),
        lambda: ops.kv_attention(q, c, table[0], lens, heads=8),
        lambda: ops.kv_attention(q, c, table.t(), i32(2), heads=8),                         # a transposed table
        lambda: ops.kv_attention(q, c, table, lens.float(), heads=8),
        lambda: ops.kv_attention(q, c, table, lens, heads=8, out=torch.zeros(4, 8 * 64, dtype=torch.float16)),
        lambda: ops.kv_attention(q[:2], c, table, lens, heads=8, out=torch.zeros(1, 8 * 64).expand(2, -1)),      # overlapping rows
        lambda: ops.kv_attention(wide[:2, :512], c, table, lens, heads=8, out=wide[:2, 64:576]),                 # output over the input
        lambda: ops.kv_attention(wide[:2, :512], c, table, lens, heads=8, out=wide[1:3, :512]),
        lambda: ops.kv_append(c, kv, kv.half(), table, lens),
        lambda: ops.kv_append(c, kv, kv[:2], table, lens),
        lambda: ops.kv_append(c, kv.t(), kv.t(), table, lens),
        lambda: ops.kv_append(c, kv[:1].expand(4, -1), kv, table, lens),                    # broadcast rows
        lambda: ops.kv_read(c, table, lens, 4, torch.float32, out=(kv, kv)),                # one buffer for both
        lambda: ops.kv_read(c, table, lens, 4, torch.float32, out=(kv, kv.half())),
        lambda: ops.qk_norm_rope(q, q[:2], lens, f, heads=8, kv_heads=8),
        lambda: ops.qk_norm_rope(q, kv.half(), None, None, heads=8, kv_heads=2),
        lambda: ops.qk_norm_rope(q, kv, lens, f, heads=8, kv_heads=2),                      # 2 positions for 4 rows
        lambda: ops.qk_norm_rope(q, kv, None, f, heads=8, kv_heads=2),                      # a rotation without positions
        lambda: ops.qk_norm_rope(q, kv, i32(4).long(), f, heads=8, kv_heads=2),
        lambda: ops.qk_norm_rope(q, kv, i32(4), f.float(), heads=8, kv_heads=2),
        lambda: ops.qk_norm_rope(q, kv, i32(4), f, torch.ones(32), heads=8, kv_heads=2),    # a gain of another length
        lambda: ops.qk_norm_rope(q, kv, i32(4), f, heads=7, kv_heads=2),
        lambda: ops.qk_norm_rope(q, kv, i32(4), f, heads=8, kv_heads=4),
        lambda: ops.qk_norm_rope(wide[:, :512], kv, i32(4), f, heads=8, kv_heads=2, out=(wide[:, 8:520], torch.zeros(4, 128))),
        lambda: ops.qk_norm_rope(wide[:, :512], kv, i32(4), f, heads=8, kv_heads=2, out=(wide[:, :512], wide[:, 448:576])),
        lambda: ops.qk_norm_rope_backward(q, kv.half(), q, kv, i32(4), f, heads=8, kv_heads=2),
        lambda: ops.qk_norm_rope_backward(q[:3], kv, q, kv, i32(4), f, heads=8, kv_heads=2),
        lambda: ops.rope_freqs(12, device="cpu"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(hip.PgtError) as e:
            call()
        assert "GPU only" not in str(e.value), (i, str(e.value))      # refused for what it is, not for where it lives


def test_outputs_that_are_inputs_or_columns_of_one_buffer_pass_the_overlap_check():
    wide = torch.zeros(4, 20 * 64)
    q, k = wide[:, :512], wide[:, 512:640]
    ops._apart((q, k), (q, k), "t")
    ops._apart((wide[:, 640:1152], wide[:, 1152:1280]), (q, k), "t")
    ops._apart((torch.zeros(4, 8),), (q,), "t")
    ops._apart((wide[2:, :512],), (wide[:2, :512],), "t")


P = 0x1000      # never dereferenced: every call below is refused on the host


def entry(name, base, **kw):
    a = dict(base, **kw)
    return getattr(hip.lib(), name)(*a.values()), hip.lib().pgt_last_error().decode()


def refused(name, base, changes):
    for kw in changes:
        rc, msg = entry(name, base, **kw)
        assert rc == -22 and msg, (name, kw, rc)


def test_c_entry_points_refuse():
    rope = dict(dtype=1, q=P, ldq=512, k=P, ldk=128, rows=4, heads=8, kv=2, hd=64, pos=P, freqs=P, rot=64, inter=0, qg=None, kg=None, eps=1e-6, qo=P,
                ldqo=512, ko=P, ldko=128, stream=None)
    changes = [dict(dtype=2), dict(dtype=9), dict(hd=48), dict(rot=12), dict(rot=72), dict(rot=-8), dict(rows=-1), dict(heads=-1), dict(heads=0, kv=0),
               dict(eps=-1.0), dict(eps=math.nan), dict(q=None), dict(ko=None), dict(pos=None), dict(freqs=None), dict(ldq=504), dict(ldko=120), dict(ldk=132),
               dict(q=P + 2), dict(ko=P + 8), dict(heads=1 << 26)]
    refused("pgt_qk_norm_rope", rope, changes)
    bwd = dict(dtype=1, dq=P, lddq=512, dk=P, lddk=128, **{k: v for k, v in rope.items() if k not in ("dtype", "stream")}, dqg=P, dkg=P, ws=P, nb=1 << 20, stream=None)
    refused("pgt_qk_norm_rope_backward", bwd, changes + [dict(dq=None), dict(lddk=120), dict(dk=P + 4), dict(ws=None), dict(nb=100), dict(ws=P + 4)])
    kv = dict(dtype=0, k=P, ldk=128, v=P, ldv=128, kp=P, vp=P, ks=P, vs=P, pages=4, page=16, kv=2, hd=64, table=P, ldt=3, width=3, lens=P, cu=None, B=2,
              rows=8, n=4, stream=None)
    changes = [dict(dtype=2), dict(page=24), dict(page=0), dict(page=256), dict(hd=32), dict(kv=0), dict(pages=0), dict(B=-1), dict(rows=-1), dict(n=-1),
               dict(width=-1), dict(ldt=2), dict(kp=None), dict(vs=None), dict(vp=P + 8), dict(k=None), dict(lens=None), dict(table=None), dict(n=5),
               dict(ldk=120), dict(ldv=130), dict(v=P + 4), dict(B=1 << 20, rows=1 << 30, n=1 << 10, kv=1 << 16, ldk=1 << 23, ldv=1 << 23)]
    refused("pgt_kv_append", kv, changes)
    refused("pgt_kv_read", kv, changes)
    att = dict(dtype=0, q=P, ldq=512, kp=P, vp=P, ks=P, vs=P, pages=4, page=16, kv=2, hd=64, table=P, ldt=3, width=3, lens=P, cu=None, B=2, rows=8, n=4,
               heads=8, scale=0.1, causal=1, window=0, out=P, ldo=512, ws=P, nb=1 << 30, stream=None)
    refused("pgt_kv_attention", att, [dict(dtype=2), dict(page=24), dict(hd=32), dict(kv=3), dict(heads=0), dict(heads=7), dict(kv=0), dict(pages=0), dict(B=-1),
                                      dict(rows=-1), dict(n=5), dict(width=-1), dict(ldt=1), dict(causal=-1), dict(window=-1), dict(causal=0, window=3),
                                      dict(scale=math.inf), dict(scale=math.nan), dict(kp=None), dict(ks=None), dict(vp=P + 4), dict(q=None),
                                      dict(out=None), dict(lens=None), dict(table=None), dict(ldq=500), dict(ldo=514), dict(out=P + 8),
                                      dict(width=4000, ldt=4000, ws=None), dict(width=4000, ldt=4000, nb=64), dict(width=4000, ldt=4000, ws=P + 8),
                                      dict(width=1 << 27, ldt=1 << 27), dict(width=(1 << 27) - 1, ldt=1 << 27), dict(width=1 << 24, ldt=1 << 24, page=128)])
    # nothing to do is not an error (and launches nothing)
    assert entry("pgt_qk_norm_rope", rope, rows=0)[0] == 0
    for name, base in (("pgt_kv_append", kv), ("pgt_kv_read", kv), ("pgt_kv_attention", att)):
        for kw in (dict(B=0), dict(rows=0, n=0)):
            assert entry(name, base, **kw)[0] == 0, (name, kw)


def test_native_launchers_decline_what_is_not_plainly_right():
    """nothing is launched, nothing raised: ops.py then says what is wrong"""
    e = hip.ops_ext()
    q, k, lens, table = torch.zeros(4, 512), torch.zeros(4, 128), i32(2), i32(2, 3)
    c = cache()
    cc = (c.k_pages, c.v_pages, c.k_scale, c.v_scale, c.pages, c.page, c.kv_heads, c.hd)
    for dev in (0, -1, 1 << 40, "cuda"):
        assert e.qk_norm_rope(dev, 0, q, k, None, None, None, None, 8, 2, 1e-6, False) is None      # tensors of the host
        assert e.qk_norm_rope_backward(dev, 0, q, k, None, None, None, None, 8, 2, 1e-6, False, q, k) is None
        assert e.kv_append(dev, 0, *cc, table, lens, None, k, k, None) is None
        assert e.kv_read(dev, 0, *cc, table, lens, None, 4, None, torch.float16) is None
        assert e.kv_attention(dev, 0, *cc, table, lens, None, q, 8, None, 1, 0, None) is None
    assert e.qk_norm_rope(0, 0, None, 3, "x", [], {}, (), 8.5, 1 << 70, "e", 1) is None
    assert e.kv_read(0, 0, *cc, table, lens, None, -4, None, torch.float16) is None
    for bad in (lambda: e.kv_append(0, 0), lambda: e.qk_norm_rope(), lambda: e.bind(1, 2)):
        with pytest.raises(TypeError):
            bad()


def test_workspace_sizes():
    L = hip.lib()
    assert L.pgt_qk_norm_rope_backward_workspace_bytes(0, 64) == 0
    assert 0 < L.pgt_qk_norm_rope_backward_workspace_bytes(1 << 20, 256) <= 1024 * 2 * 256 * 4
    f = L.pgt_kv_attention_workspace_bytes      # (dtype, B, max_new, heads, kv_heads, hd, width, page, causal, window)
    for dtype in (0, 1, 3):
        assert f(dtype, 0, 1, 8, 8, 64, 4, 16, 1, 0) == 0 and f(dtype, 1, 1, 8, 3, 64, 4, 16, 1, 0) == 0 and f(dtype, 1, 1, 8, 8, 64, 4, 24, 1, 0) == 0
        assert f(dtype, 1, 1, 8, 8, 64, 1, 16, 1, 0) == 0       # one tile: nothing to join
        long = f(dtype, 1, 1, 32, 8, 128, 8192, 16, 1, 0)
        assert isinstance(long, int) and long >= f(dtype, 1, 1, 32, 8, 128, 8192, 16, 1, 4096) > 0 and f(dtype, 1, 1, 32, 8, 128, 8192, 16, 1, 64) == 0
        assert f(dtype, 64, 2048, 32, 8, 128, 512, 32, 1, 0) == 0      # enough rows to fill the chip
    assert C.sizeof(C.c_size_t) == 8


def test_reference_forms_agree_with_each_other():
    """the 64-bit append against a direct quantisation of whole pages, and attention over one page against a dense softmax"""
    g = torch.Generator().manual_seed(0)
    ref = kv_ref.Cache(3, 1, 16, 64)
    x = torch.randn((20, 64), generator=g) * 5
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    ref.append(x, x, table, [0], [0, 20])
    for pid, part in ((2, x[:16]), (0, x[16:])):
        e = math.ceil(math.log2(float(part.abs().max()) / 448))
        assert int(ref.e[0][pid, 0]) == e
        want = (part / 2.0 ** e).to(torch.float8_e4m3fn).double()
        assert torch.equal(ref.code[0][pid, :part.shape[0], 0], want)
    q = torch.randn((1, 128), generator=g)
    out, _, _ = kv_ref.attention(q, ref, table, [20], [0, 1], 2, 1, 0, 0.3)
    k, _ = ref.tokens(0, table, 0, 0, 20)
    for h in range(2):
        w = torch.softmax(k[:, 0] @ q[0, h * 64:(h + 1) * 64].double() * 0.3, 0)
        assert torch.allclose(out[0, h * 64:(h + 1) * 64], w @ k[:, 0], rtol=0, atol=1e-12)
