"""GPU: cross attention and token embedding where a call is easily answered wrongly: what autograd and the tracer see of it, infinities and
NaN, probabilities far below a row's largest, sequences without keys, rows split over many workgroups.

Tolerances are those of test_gpu_conditioning.oracle (64 bits on the CPU), where a test does not derive its own."""
import math
import warnings

import pytest
import torch

from test_gpu_conditioning import DEV, DT, check, half_step, mask_of, oracle, rnd, run

pytestmark = pytest.mark.gpu


def ops():
    from favae_hip import ops as K
    return K


def test_traced_programs_give_the_eager_results():
    """with other values than the traced ones, and with leaves where the traced inputs were plain"""
    K = ops()
    q, k, v = (rnd(s, i, torch.float32).to(DEV) for i, s in enumerate(((2, 9, 4, 32), (2, 40, 2, 32), (2, 40, 2, 32))))
    ids, w, g = torch.randint(0, 50, (3, 7)).to(DEV), rnd((50, 24), 4, torch.float32).to(DEV), rnd((3, 7, 24), 5, torch.float32).to(DEV)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                                          # the checks of sizes are constants of a trace
        attend = torch.jit.trace(lambda q, k, v: K.cross_attention(q, k, v), (q, k, v), check_trace=False)
        embed = torch.jit.trace(lambda ids, w: K.embedding(ids, w, 2.0), (ids, w), check_trace=False)
        grad = torch.jit.trace(lambda g, ids: K.embedding_grad(g, ids, 50), (g, ids), check_trace=False)
    for _ in range(3):
        q, k, v, w, g = (t * -1.5 for t in (q, k, v, w, g))
        ids = ids.add(1).remainder(50)
        assert torch.equal(attend(q, k, v), K.cross_attention(q, k, v)) and torch.equal(embed(ids, w), K.embedding(ids, w, 2.0))
        assert torch.equal(grad(g, ids), K.embedding_grad(g, ids, 50))
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        a, b = (torch.autograd.grad(f(*leaves), leaves, q) for f in (attend, K.cross_attention))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_call_without_gradients_gives_the_same_bits():
    """plain inputs (nothing is kept) and leaves, in every form of the forward pass"""
    K = ops()
    for dt in DT.values():
        for Lq, Lk, G, D in ((1, 300, 1, 64), (1, 5000, 4, 64), (10, 300, 4, 64), (200, 70, 1, 64), (200, 300, 1, 64), (300, 3000, 1, 128)):
            q, k, v = rnd((1, Lq, 2 * G, D), 1, dt).to(DEV), rnd((1, Lk, 2, D), 2, dt).to(DEV), rnd((1, Lk, 2, D), 3, dt).to(DEV)
            out = K.cross_attention(q, k, v)
            assert out.grad_fn is None and torch.equal(K.cross_attention(q, k.requires_grad_(), v), out)
