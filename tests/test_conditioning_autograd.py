"""CPU: cross_attention, embedding and embedding_grad stay visible to autograd and to the tracer whatever their inputs require, with the
launches stubbed: a launch fills its output with the number of the call."""
import ctypes
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from favae_hip import ops as K


@pytest.fixture
def launches(monkeypatch):
    """names of the launches so far; launch n fills the first output with n"""
    names = []

    def fill(p, count):
        ctypes.memmove(p, (ctypes.c_float * count)(*([float(len(names))] * count)), 4 * count)

    def call(name, *a):
        names.append(name)
        if name == "favae_xattn_fwd":
            d = a[0]._obj
            fill(a[5], d.B * d.Lq * d.H * d.D)
        elif name == "favae_xattn_bwd":
            d = a[0]._obj
            fill(a[8], d.B * d.Lq * d.H * d.D)
            for p in (a[9], a[10]):
                if p:
                    fill(p, d.B * d.Lk * d.Hkv * d.D)
        elif name == "favae_embed_fwd":
            fill(a[5], a[6] * a[7])
        elif name == "favae_embed_bwd":
            fill(a[9], a[4] * a[5])

    monkeypatch.setattr(K, "call", call)
    monkeypatch.setattr(K, "_require_float_gpu", lambda what, *t: None)
    monkeypatch.setattr(K, "_on_device", lambda fn, device, *a: fn(*a))
    return names


def tensors():
    return torch.randn(2, 4, 8, 32), torch.randn(2, 5, 8, 32), torch.randn(2, 5, 8, 32)


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_through_attention_raises(launches, which, leaf):
    """a tangent on q, k or v is refused, not dropped"""
    x = list(tensors())
    with fwAD.dual_level():
        x[which] = fwAD.make_dual(x[which].requires_grad_(leaf), torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="forward mode"):
            K.cross_attention(*x)


def test_forward_mode_through_embedding_raises(launches):
    ids = torch.tensor([[0, 3], [1, 1]])
    with fwAD.dual_level():
        w = fwAD.make_dual(torch.randn(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward mode"):
            K.embedding(ids, w)
        g = fwAD.make_dual(torch.randn(2, 2, 8), torch.ones(2, 2, 8))
        with pytest.raises(NotImplementedError, match="forward mode"):
            K.embedding_grad(g, ids, 4)


def traced(fn, *args):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                                          # the checks of sizes are constants of a trace
        return torch.jit.trace(fn, args, check_trace=False)


def test_a_traced_program_launches(launches):
    """its results are those of its own launches, not the memory they would have been written to"""
    q, k, v = tensors()
    ids, w, g = torch.tensor([0, 3, 1]), torch.randn(4, 8), torch.randn(3, 8)
    for fn, args in ((lambda q, k, v: K.cross_attention(q, k, v), (q, k, v)), (lambda ids, w: K.embedding(ids, w), (ids, w)),
                     (lambda g, ids: K.embedding_grad(g, ids, 4), (g, ids))):
        t = traced(fn, *args)
        for _ in range(2):
            n = len(launches)
            out = t(*args)
            assert len(launches) == n + 1 and bool((out == n + 1.0).all())


def test_a_program_traced_without_gradients_has_them_later(launches):
    """traced over plain tensors and run over leaves: what the backward pass needs is kept then"""
    q, k, v = tensors()
    with torch.no_grad():
        t = traced(lambda q, k, v: K.cross_attention(q, k, v), q, k, v)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(t(*leaves), leaves, torch.ones_like(q))
    n = len(launches)
    assert launches[-1] == "favae_xattn_bwd" and all(bool((x == n).all()) for x in grads)
    ids, w = torch.tensor([0, 3, 1]), torch.randn(4, 8)
    t = traced(lambda ids, w: K.embedding(ids, w), ids, w)
    leaf = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(t(ids, leaf), leaf, torch.ones(3, 8))
    assert launches[-1] == "favae_embed_bwd" and bool((dw == len(launches)).all())


def test_embedding_grad_keeps_its_history(launches):
    """a gradient of a gradient is refused where it is asked for; the first derivative alone is not disturbed"""
    ids = torch.tensor([0, 3, 1])
    dw = K.embedding_grad(torch.randn(3, 8, requires_grad=True), ids, 4)
    assert dw.requires_grad and bool((dw == 1.0).all())
    with pytest.raises(RuntimeError, match="no derivative"):
        dw.sum().backward()
    assert not K.embedding_grad(torch.randn(3, 8), ids, 4).requires_grad
    with torch.no_grad():
        assert not K.embedding_grad(torch.randn(3, 8, requires_grad=True), ids, 4).requires_grad


def test_nothing_is_kept_where_no_gradient_can_be_asked_for(launches, monkeypatch):
    """inference allocates the output alone: no copy before its rounding, no log-sums"""
    seen = []
    fwd = K._xattn_fwd
    monkeypatch.setattr(K, "_xattn_fwd", lambda *a: seen.append(a[5]) or fwd(*a))
    q, k, v = tensors()
    assert K.cross_attention(q, k, v).grad_fn is None
    out = K.cross_attention(q, k, v.requires_grad_())
    with torch.no_grad():
        K.cross_attention(q, k, v)
    with torch.inference_mode():
        K.cross_attention(q, k, v)
    assert out.grad_fn is not None and seen == [False, True, False, False]


def test_a_learnt_scale_is_refused(launches):
    """it would get no gradient; one that needs none is a number like any other"""
    q, k, v = tensors()
    ids, w, g = torch.tensor([0, 3, 1]), torch.randn(4, 8), torch.randn(3, 8)
    learnt = torch.tensor(0.5, requires_grad=True)
    for f in (lambda s: K.cross_attention(q, k, v, None, s), lambda s: K.embedding(ids, w, s), lambda s: K.embedding_grad(g, ids, 4, s)):
        with pytest.raises(ValueError, match="no gradient"):
            f(learnt)
        f(learnt.detach())
        f(0.5)
