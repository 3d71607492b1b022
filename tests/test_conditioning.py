"""CPU: what cross_attention, embedding and embedding_grad refuse, and what their C entry points refuse before any launch."""
from ctypes import byref

import pytest
import torch

import favae_hip
from favae_hip import XattnDesc
from favae_hip import ops as K


class OnGpu:
    """a CPU tensor that says it is on the GPU, for checks that come before the first kernel"""

    def __init__(self, t):
        self.t = t

    is_cuda = True

    def __getattr__(self, n):
        return getattr(self.t, n)


def qkv(q, k, v=None, dtype=torch.float32):
    return tuple(OnGpu(torch.zeros(s, dtype=dtype)) for s in (q, k, v or k))


def test_no_cpu_fallback():
    t = torch.zeros(1, 2, 4, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        K.cross_attention(t, t, t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        K.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        K.embedding_grad(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 4)


@pytest.mark.parametrize("shapes, what", [
    (((2, 4, 8, 32), (2, 5, 3, 32)), "evenly"), (((2, 4, 8, 32), (3, 5, 8, 32)), "B, Lk"), (((2, 4, 8, 32), (2, 5, 8, 64)), "B, Lk"),
    (((2, 4, 8, 32), (2, 5, 8, 32), (2, 6, 8, 32)), "B, Lk"), (((4, 8, 32), (5, 8, 32)), "B, Lk"), (((2, 4, 8, 36), (2, 5, 8, 36)), "multiple of 8"),
    (((2, 4, 8, 136), (2, 5, 8, 136)), "multiple of 8"), (((2, 4, 8, 0), (2, 5, 8, 0)), "multiple of 8"), (((2, 4, 0, 32), (2, 5, 0, 32)), "evenly")])
def test_cross_attention_refuses_shapes(shapes, what):
    with pytest.raises(ValueError, match=what):
        K.cross_attention(*qkv(*shapes))


def test_cross_attention_refuses_types_masks_and_scales():
    q, k, v = qkv((2, 4, 8, 32), (2, 5, 8, 32))
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        K.cross_attention(*qkv((2, 4, 8, 32), (2, 5, 8, 32), dtype=torch.float64))
    with pytest.raises(RuntimeError, match="differ"):
        K.cross_attention(q, OnGpu(k.t.half()), OnGpu(v.t.half()))
    for bad in (torch.zeros(2, 5), torch.zeros(2, 4, dtype=torch.bool), torch.zeros(5, dtype=torch.bool), torch.zeros(2, 5, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="key_padding_mask"):                # additive masks, other shapes, bytes
            K.cross_attention(q, k, v, bad)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            K.cross_attention(q, k, v, None, bad)


def test_embedding_refusals():
    w, ids = OnGpu(torch.zeros(4, 8)), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="int64 or int32"):
        K.embedding(ids.float(), w)
    with pytest.raises(ValueError, match="int64 or int32"):
        K.embedding(ids.to(torch.int16), w)
    with pytest.raises(ValueError, match="V, C"):
        K.embedding(ids, OnGpu(torch.zeros(4)))
    with pytest.raises(ValueError, match="V, C"):
        K.embedding(ids, OnGpu(torch.zeros(0, 8)))
    for p in (4, -5):
        with pytest.raises(ValueError, match="padding_idx"):
            K.embedding(ids, w, 1.0, p)
    g = OnGpu(torch.zeros(3, 8))
    with pytest.raises(ValueError, match="at least one row"):
        K.embedding_grad(g, ids, 0)
    with pytest.raises(ValueError, match="ids.shape"):
        K.embedding_grad(g, ids[:2], 4)
    with pytest.raises(ValueError, match="padding_idx"):
        K.embedding_grad(g, ids, 4, 1.0, 4)
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        K.embedding_grad(OnGpu(torch.zeros(3, 8, dtype=torch.float64)), ids, 4)


def desc(**kw):
    f = dict(B=2, Lq=4, Lk=5, H=8, Hkv=2, D=32, dtype=1, scale=0.5, q_sb=1024, q_sl=256, q_sh=32, k_sb=320, k_sl=64, k_sh=32, v_sb=320, v_sl=64,
             v_sh=32, pad_sb=0)
    f.update(kw)
    return XattnDesc(**f)


def test_c_entry_points_refuse_before_they_launch():
    lib = favae_hip.load()
    P = 1 << 12                                                                  # an aligned address that no refused call touches
    bad_arg, unsupported, workspace = 1, 3, 4

    def fwd(d, q=P, k=P, v=P, o=P, ws=None, n=0):
        return lib.favae_xattn_fwd(byref(d) if d else None, q, k, v, None, o, None, None, ws, n, None)

    def bwd(d, q=P, dq=P, dk=P, dv=P, ws=P, n=1 << 40):
        return lib.favae_xattn_bwd(byref(d) if d else None, q, P, P, None, P, P, P, dq, dk, dv, ws, n, None)

    assert fwd(None) == bad_arg and fwd(desc(), q=None) == bad_arg and fwd(desc(), o=None) == bad_arg
    assert bwd(None) == bad_arg and bwd(desc(), dq=None) == bad_arg and bwd(desc(), ws=None) == bad_arg
    assert bwd(desc(), dk=None) == bad_arg and bwd(desc(), dv=None) == bad_arg   # both or neither
    for d in (desc(D=36), desc(D=136), desc(D=0), desc(H=7), desc(Hkv=0), desc(B=0), desc(Lq=0), desc(Lk=0), desc(dtype=3), desc(dtype=-1),
              desc(scale=0.0), desc(scale=-1.0), desc(scale=float("inf")), desc(scale=float("nan")), desc(q_sl=260), desc(k_sb=-320),
              desc(v_sh=4), desc(dtype=0, k_sl=66), desc(Lq=1 << 30), desc(k_sl=0), desc(v_sl=24), desc(q_sl=1 << 23)):
        assert fwd(d) == unsupported and bwd(d) == unsupported
        assert lib.favae_xattn_fwd_workspace(byref(d)) == 0 and lib.favae_xattn_bwd_workspace(byref(d)) == 0
    assert fwd(desc(), q=P + 8) == unsupported and fwd(desc(), o=P + 4) == unsupported and bwd(desc(), dq=P + 2) == unsupported
    assert bwd(desc(), n=16) == workspace
    long = desc(B=1, Lq=1, H=2, Lk=1 << 16)                                      # splits its keys
    need = lib.favae_xattn_fwd_workspace(byref(long))
    assert need > 0 and fwd(long) == workspace and fwd(long, ws=P, n=need - 1) == workspace

    def efwd(ids=P, w=P, ws=8, V=4, out=P, T=3, C=8, dt=0):
        return lib.favae_embed_fwd(ids, 1, w, ws, V, out, T, C, dt, 1.0, None)

    def ebwd(ids=P, g=P, T=3, V=4, C=8, dt=0, dw=P, ws=P, n=1 << 40):
        return lib.favae_embed_bwd(ids, 1, g, T, V, C, dt, 1.0, -1, dw, ws, n, None)

    for f in (efwd(ids=None), efwd(w=None), efwd(out=None), efwd(ws=-8), ebwd(ids=None), ebwd(g=None), ebwd(dw=None), ebwd(ws=None)):
        assert f == bad_arg
    for f in (efwd(T=0), efwd(V=0), efwd(C=0), efwd(dt=3), efwd(T=1 << 31), efwd(V=1 << 31), ebwd(T=0), ebwd(V=0), ebwd(C=0), ebwd(dt=-1),
              ebwd(T=1 << 31), ebwd(dw=P + 4), ebwd(ws=P + 8)):
        assert f == unsupported
    assert ebwd(n=lib.favae_embed_bwd_workspace(3, 4, 8) - 1) == workspace and lib.favae_embed_bwd_workspace(0, 4, 8) == 0


def test_rows_of_very_many_heads_are_refused():
    """the dense outputs' rows of H D elements have to stay under 2^24 bytes, whatever the strides of the inputs"""
    lib = favae_hip.load()
    for dtype, heads in ((0, 1 << 16), (1, 1 << 17)):                            # times 64 columns
        at, under = (desc(B=1, Lq=1, Lk=1, H=h, Hkv=8, D=64, dtype=dtype) for h in (heads, heads - 8))
        assert lib.favae_xattn_bwd_workspace(byref(at)) == 0 and lib.favae_xattn_bwd_workspace(byref(under)) > 0
        assert lib.favae_xattn_fwd(byref(at), 1 << 12, 1 << 12, 1 << 12, None, 1 << 12, None, None, None, 0, None) == 3


def test_scales_that_leave_32_bits_in_powers_of_two_are_refused():
    """scores are taken times scale / ln 2"""
    lib = favae_hip.load()
    for scale, ok in ((2.3e38, True), (2.4e38, False), (3.4e38, False)):
        d = desc(scale=scale)
        assert (lib.favae_xattn_bwd_workspace(byref(d)) > 0) == ok
        if not ok:
            assert lib.favae_xattn_fwd(byref(d), 1 << 12, 1 << 12, 1 << 12, None, 1 << 12, None, None, None, 0, None) == 3


def test_embedding_gradients_too_wide_for_a_launch_are_refused_before_the_first():
    """the sums' launch is what they are too wide for; the sort before it must not have run"""
    lib, P = favae_hip.load(), 1 << 12
    for T, C, dt in ((4096, (1 << 24) - 1, 0), (1 << 17, 1 << 24, 1), (1 << 17, (1 << 22) + 1, 2)):
        assert lib.favae_embed_bwd(P, 1, P, T, 4, C, dt, 1.0, -1, P, P, 1 << 62, None) == 3
