"""GPU: cross attention and token embedding, forward and backward, against plain 64-bit implementations on the CPU.

Tolerances, with u = half a step of the element type (2^-8, 2^-11, 2^-24) and e = 2^-24:
  * a 16-bit result carries its own rounding (u of its value) and that of the probabilities or score gradients that enter its last product
    (u of the sum of the products' magnitudes); fp32 elements have neither, only 32-bit arithmetic;
  * 32-bit arithmetic: a score is a sum of D products, so it is off by at most (D + 8) e of the sum of their magnitudes, and a probability
    by that plus a few e relative; sums over n keys or rows add at most n e of the sum of magnitudes.
bounds() evaluates this elementwise in 64 bits.  Norms: independent roundings of at most u have an rms of at most u / sqrt(3) each."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def ops():
    from favae_hip import ops as K
    return K


def rnd(shape, seed, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dt)


def oracle(q, k, v, pad, scale, do):
    """values, and elementwise bounds of their 32-bit and rounding errors, of out, dq, dk, dv (64 bits)"""
    dt = q.dtype
    u = half_step(dt)
    w = 0.0 if dt == torch.float32 else u                                       # rounding of probabilities and score gradients
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    q, k, v, do = (t.double().permute(0, 2, 1, 3) for t in (q, k, v, do))       # (B, heads, L, D)
    if pad is not None:                                                          # what stands in padded places takes no part
        k, v = (torch.where(pad[:, None, :, None], torch.zeros((), dtype=torch.float64), t) for t in (k, v))
    ke, ve = (t.repeat_interleave(G, 1) for t in (k, v))
    s = scale * q @ ke.transpose(2, 3)
    sa = scale * q.abs() @ ke.abs().transpose(2, 3)
    if pad is not None:
        s = s.masked_fill(pad[:, None, None, :], -math.inf)
    m = s.amax(3, keepdim=True)
    m = torch.where(m.isinf(), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    p = p / p.sum(3, keepdim=True).clamp_min(1e-300)
    rp = E * (24 + Lk + (D + 8) * (sa + (p * sa).sum(3, keepdim=True)))         # relative error of a probability
    o = p @ ve
    oa = p @ ve.abs()
    be = {"out": (p * rp) @ ve.abs() + (w + E * (Lk + 8)) * oa + u * o.abs()}
    dp = do @ ve.transpose(2, 3)
    dpa = do.abs() @ ve.abs().transpose(2, 3)
    delta = (do * o).sum(3, keepdim=True)
    derr = (do.abs() * ((p * rp) @ ve.abs() + (w + E * (Lk + D + 16)) * oa)).sum(3, keepdim=True)
    ds = scale * p * (dp - delta)
    dse = scale * p * (rp * (dp - delta).abs() + E * (D + 8) * dpa + derr) + (w + 4 * E) * ds.abs()
    fold = lambda t: t.view(B, Hkv, G, Lk, D).sum(2)  # noqa: E731
    n = G * Lq
    dq, dk, dv = ds @ ke, fold(ds.transpose(2, 3) @ q), fold(p.transpose(2, 3) @ do)
    be["dq"] = (dse + E * (Lk + 8) * ds.abs()) @ ke.abs() + u * dq.abs()
    be["dk"] = fold((dse + E * (n + 8) * ds.abs()).transpose(2, 3) @ q.abs()) + u * dk.abs()
    be["dv"] = fold((p * (rp + w + E * (n + 8))).transpose(2, 3) @ do.abs()) + u * dv.abs()
    val = {"out": o, "dq": dq, "dk": dk, "dv": dv}
    if dt == torch.float16:                                                      # results under the smallest normal number round to its grid
        be = {n: t + 2.0 ** -25 for n, t in be.items()}
    return {n: t.permute(0, 2, 1, 3) for n, t in val.items()}, {n: t.permute(0, 2, 1, 3) for n, t in be.items()}


def check(got, val, bound, dt, norms=True):
    for n, t in got.items():
        x = t.detach().cpu().double()
        assert x.shape == val[n].shape and t.dtype == dt, n
        off = (x - val[n]).abs()
        assert bool((off <= bound[n] + 1e-300).all()), (n, float((off / (bound[n] + 1e-300)).max()))
        norm = float(val[n].norm())
        if norms and norm > 0 and x.numel() >= 512:
            rel = float(off.norm()) / norm
            assert rel <= (4e-6 if dt == torch.float32 else half_step(dt)), (n, rel)


def run(q, k, v, pad, scale, do):
    K = ops()
    q, k, v = (t.to(DEV).requires_grad_() for t in (q, k, v))
    pad = None if pad is None else pad.to(DEV)
    out = K.cross_attention(q, k, v, pad, scale)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do.to(DEV))
    with torch.no_grad():
        again = K.cross_attention(q, k, v, pad, scale)                           # the call without a backward pass: the same result
    assert torch.equal(again, out)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def mask_of(kind, B, Lk, seed):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed)
    if kind == "holes":
        return torch.rand((B, Lk), generator=g) < 0.5
    n = torch.randint(0 if kind == "empty" else 1, Lk + 1, (B, 1), generator=g)
    if kind == "empty":
        n[0] = 0
    return torch.arange(Lk)[None] >= n


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 77, 4, 2, 64), (2, 5, 130, 4, 1, 40), (1, 33, 64, 2, 2, 32), (2, 129, 65, 3, 3, 96), (1, 257, 300, 2, 1, 128),
          (3, 64, 31, 8, 2, 16), (1, 700, 129, 2, 2, 64), (2, 130, 1100, 2, 1, 72), (1, 3, 2500, 4, 2, 128), (1, 1, 4099, 4, 1, 104),
          (1, 20, 700, 2, 1, 128), (2, 30, 300, 1, 1, 96), (1, 150, 400, 2, 2, 96), (1, 16, 513, 3, 3, 32), (1, 140, 40, 1, 1, 8)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("mask", ["none", "tail", "holes", "empty"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_cross_attention_against_64_bits(shape, mask, dtype):
    B, Lq, Lk, H, Hkv, D = shape
    dt = DT[dtype]
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of(mask, B, Lk, 5)
    scale = D ** -0.5
    got = run(q, k, v, pad, scale, do)
    check(got, *oracle(q, k, v, pad, scale, do), dt)
    if pad is not None:
        assert not got["dk"].cpu()[pad].any() and not got["dv"].cpu()[pad].any()
        for b in pad.all(1).nonzero()[:, 0].tolist():
            assert not got["out"][b].any() and not got["dq"][b].any()


@pytest.mark.parametrize("dtype", list(DT))
def test_many_row_tiles_take_the_two_tile_kernel(dtype):
    """enough rows and heads for the wider row tiling, with ragged lengths"""
    dt = DT[dtype]
    B, Lq, Lk, H, Hkv, D = 32, 261, 70, 16, 16, 24
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of("empty", B, Lk, 6)
    check(run(q, k, v, pad, 0.3, do), *oracle(q, k, v, pad, 0.3, do), dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Lq", [1, 100])
def test_what_padded_rows_hold_reaches_nothing(dtype, Lq):
    dt = DT[dtype]
    B, Lk, H, D = 2, 150, 2, 64
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, H, D), 2, dt), rnd((B, Lk, H, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of("holes", B, Lk, 9)
    val, bound = oracle(q, k, v, pad, 0.125, do)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dt).min):
        k2, v2 = k.clone(), v.clone()
        k2[pad], v2[pad] = bad, bad
        check(run(q, k2, v2, pad, 0.125, do), val, bound, dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [40, 88, 128])
def test_padded_tiles_between_live_ones(dtype, D):
    """a tile of keys that is all padding between two that are not, and scattered padding in both: the bits of a run with zeros there"""
    dt = DT[dtype]
    B, Lq, Lk, H, Hkv = 2, 70, 300, 4, 2
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of("holes", B, Lk, 7)
    pad[:, 128:256] = True
    k[pad] = v[pad] = 0.0
    clean = run(q, k, v, pad, D ** -0.5, do)
    check(clean, *oracle(q, k, v, pad, D ** -0.5, do), dt)
    k[pad], v[pad] = math.inf, math.nan
    for n, t in run(q, k, v, pad, D ** -0.5, do).items():
        assert torch.equal(t, clean[n]), n


@pytest.mark.parametrize("dtype", list(DT))
def test_layouts_are_read_where_they_are(dtype):
    """views of a packed projection, head-major tensors, states shared by the batch, odd offsets: results of the dense copies, and gradients
    that go back through the views (a shared tensor's is the sum over its readers)"""
    K, dt = ops(), DT[dtype]
    B, Lq, Lk, H, D = 3, 50, 90, 4, 32
    q0, k0, v0 = rnd((B, Lq, H, D), 1, dt).to(DEV), rnd((B, Lk, H, D), 2, dt).to(DEV), rnd((B, Lk, H, D), 3, dt).to(DEV)
    do = rnd((B, Lq, H, D), 4, dt).to(DEV)

    def grads(leaves, q, k, v):
        out = K.cross_attention(q, k, v)
        return (out,) + torch.autograd.grad(out, leaves, do)

    ref = grads(*(lambda a: (a, *a))([t.clone().requires_grad_() for t in (q0, k0, v0)]))
    kv = torch.stack((k0, v0), 2).requires_grad_()                               # packed
    q = q0.clone().requires_grad_()
    got = grads((q, kv), q, *kv.unbind(2))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], torch.stack(ref[2:], 2))
    hm = [t.transpose(1, 2).contiguous().requires_grad_() for t in (q0, k0, v0)]  # head-major memory
    got = grads(hm, *(t.transpose(1, 2) for t in hm))
    assert all(torch.equal(a, b) for a, b in zip(got, (ref[0], *(t.transpose(1, 2) for t in ref[1:]))))
    flat = k0[:, :1].expand(-1, Lk, -1, -1)                                      # a length stride of 0: copied
    assert torch.equal(K.cross_attention(q0, flat, v0), K.cross_attention(q0, flat.contiguous(), v0))
    big = torch.zeros(B, Lk, H, D + 1, dtype=dt, device=DEV)                     # rows that begin at odd addresses: copied
    big[..., 1:] = k0
    assert torch.equal(K.cross_attention(q0, big[..., 1:], v0), ref[0])
    odd = torch.zeros(q0.numel() + 1, dtype=dt, device=DEV)[1:].view_as(q0).copy_(q0)
    assert odd.data_ptr() % 16 and torch.equal(K.cross_attention(odd, k0, v0), ref[0])
    one = [k0[:1].clone().requires_grad_(), v0[:1].clone().requires_grad_()]     # one sequence of states for the whole batch
    out = K.cross_attention(q0, *(t.expand(B, -1, -1, -1) for t in one))
    g = torch.autograd.grad(out, one, do)
    dense = [t.detach().expand(B, -1, -1, -1).clone().requires_grad_() for t in one]
    out2 = K.cross_attention(q0, *dense)
    g2 = torch.autograd.grad(out2, dense, do)
    assert torch.equal(out, out2) and all(torch.equal(a, b.sum(0, keepdim=True)) for a, b in zip(g, g2))
    s = q0.clone().requires_grad_()                                              # the same tensor in all three places
    gs = torch.autograd.grad(K.cross_attention(s, s, s), s, do)[0]
    a, b, c = (q0.clone().requires_grad_() for _ in range(3))
    parts = torch.autograd.grad(K.cross_attention(a, b, c), (a, b, c), do)
    lim = 4 * half_step(dt) * (sum(t.abs() for t in parts))                      # three roundings of a sum of three
    assert bool(((gs.float() - sum(t.float() for t in parts)).abs() <= lim.float() + 1e-30).all())


def test_mask_strides():
    K = ops()
    q, k = rnd((4, 9, 2, 32), 1, torch.float32).to(DEV), rnd((4, 40, 2, 32), 2, torch.float32).to(DEV)
    pad = mask_of("holes", 4, 40, 3).to(DEV)
    ref = K.cross_attention(q, k, k, pad)
    wide = torch.zeros(4, 100, dtype=torch.bool, device=DEV)
    wide[:, 30:70] = pad
    assert torch.equal(K.cross_attention(q, k, k, wide[:, 30:70]), ref)
    assert torch.equal(K.cross_attention(q, k, k, pad.t().contiguous().t()), ref)
    assert torch.equal(K.cross_attention(q, k, k, pad[:1].expand(4, -1)), K.cross_attention(q, k, k, pad[:1].repeat(4, 1)))


def test_gradients_against_differences():
    """central differences of a 64-bit restatement at the kernel's inputs: the gradients are those of the formula"""
    B, Lq, Lk, H, Hkv, D = 1, 3, 6, 2, 1, 8
    q, k, v, do = rnd((B, Lq, H, D), 1, torch.float32), rnd((B, Lk, Hkv, D), 2, torch.float32), rnd((B, Lk, Hkv, D), 3, torch.float32), rnd((B, Lq, H, D), 4, torch.float32)
    pad = torch.tensor([[False, True, False, False, False, True]])
    got = run(q, k, v, pad, 0.4, do)

    def f(q, k, v):
        return float((oracle(q, k, v, pad, 0.4, do)[0]["out"] * do.double()).sum())

    base = [t.double() for t in (q, k, v)]
    h = 1e-5                                                                     # third derivatives of order 1: error about h^2
    for i, n in enumerate(("dq", "dk", "dv")):
        flat = got[n].cpu().double().reshape(-1)
        for j in range(0, flat.numel(), 5):
            x = [t.clone() for t in base]
            x[i].view(-1)[j] += h
            hi = f(*x)
            x[i].view(-1)[j] -= 2 * h
            lo = f(*x)
            assert abs((hi - lo) / (2 * h) - float(flat[j])) <= 2e-5


@pytest.mark.parametrize("dtype, gain", [("fp16", 2.0 ** -20), ("fp16", 2.0 ** 9), ("bf16", 2.0 ** -60), ("bf16", 2.0 ** 60), ("fp32", 2.0 ** -60), ("fp32", 2.0 ** 60)])
def test_small_and_large_gradients_keep_their_precision(dtype, gain):
    """score gradients far from 1: a power of two on dout comes out as that power on the gradients, but for results that leave the type's
    normal range (their bound is half a step of its subnormal grid)"""
    dt = DT[dtype]
    B, Lq, Lk, H, D = 2, 130, 700, 2, 64
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, H, D), 2, dt), rnd((B, Lk, H, D), 3, dt, 4.0), rnd((B, Lq, H, D), 4, dt)
    if gain < 1 and dtype == "fp16":                                             # keep dout itself normal
        do = torch.where(do.abs() < 2.0 ** 6 * 2.0 ** -14 / gain * 2.0 ** -14, torch.full_like(do, 0.25), do)
    do = (do.double() * gain).to(dt)
    got = run(q, k, v, None, 0.125, do)
    val, bound = oracle(q, k, v, None, 0.125, do)
    check(got, val, bound, dt, norms=gain > 1 or dtype != "fp16")


@pytest.mark.parametrize("dtype", list(DT))
def test_large_scores_and_ties(dtype):
    """scores of hundreds (a softmax that is almost one key), and scores that are all alike"""
    dt = DT[dtype]
    B, Lq, Lk, H, D = 1, 70, 300, 2, 64
    q, k, v, do = rnd((B, Lq, H, D), 1, dt, 6.0), rnd((B, Lk, H, D), 2, dt, 6.0), rnd((B, Lk, H, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    check(run(q, k, v, None, 0.125, do), *oracle(q, k, v, None, 0.125, do), dt, norms=False)
    k = k[:, :1].expand(-1, Lk, -1, -1).contiguous()
    got = run(q, k, v, None, 0.125, do)
    val, bound = oracle(q, k, v, None, 0.125, do)
    check({n: got[n] for n in ("out", "dk", "dv")}, val, bound, dt, norms=False)


def test_infinite_and_nan_values_among_live_keys_stay_in_their_rows():
    K = ops()
    for dt in DT.values():
        q, k, v = rnd((2, 40, 2, 32), 1, dt).to(DEV), rnd((2, 50, 2, 32), 2, dt).to(DEV), rnd((2, 50, 2, 32), 3, dt).to(DEV)
        ref = K.cross_attention(q, k, v)
        q2 = q.clone()
        q2[0, 3, 1, 5] = math.nan
        out = K.cross_attention(q2, k, v)
        assert bool(out[0, 3, 1].isnan().all())
        out[0, 3, 1] = ref[0, 3, 1]
        assert torch.equal(out, ref)
        v2 = v.clone()
        v2[1, 7, 0, 9] = math.inf
        out = K.cross_attention(q, k, v2)
        assert not bool(torch.isfinite(out[1, :, 0, 9]).any())
        out[1, :, 0, 9] = ref[1, :, 0, 9]
        assert torch.equal(out, ref)


@pytest.mark.parametrize("shape", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_empty_axes(shape):
    K = ops()
    B, Lq, Lk = shape
    q = torch.randn(B, Lq, 4, 32, device=DEV, requires_grad=True)
    k, v = (torch.randn(B, Lk, 2, 32, device=DEV, requires_grad=True) for _ in range(2))
    out = K.cross_attention(q, k, v, torch.zeros(B, Lk, dtype=torch.bool, device=DEV))
    assert out.shape == q.shape and not out.any()
    g = torch.autograd.grad(out.sum(), (q, k, v))
    assert all(a.shape == b.shape and not a.any() for a, b in zip(g, (q, k, v)))


@pytest.mark.parametrize("Lk, step", [(700, 2 ** 22), (70, 2 ** 25)])
def test_offsets_beyond_32_bits(Lk, step):
    """rows of a long cache more than 2^32 bytes (and 2^31 elements) from its start, read in place and (rows very far apart) copied first"""
    K = ops()
    D = 32
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 10 GB")
    cache = torch.empty((Lk * step + 2 * D,), dtype=torch.float16, device=DEV)
    k, v = cache.as_strided((1, Lk, 1, D), (0, step, D, 1)), cache.as_strided((1, Lk, 1, D), (0, step, D, 1), D)
    kd, vd = rnd((1, Lk, 1, D), 1, torch.float16).to(DEV), rnd((1, Lk, 1, D), 2, torch.float16).to(DEV)
    k.copy_(kd)
    v.copy_(vd)
    for Lq in (1, 100):
        q, do = rnd((1, Lq, 1, D), 3, torch.float16).to(DEV).requires_grad_(), rnd((1, Lq, 1, D), 4, torch.float16).to(DEV)
        a = K.cross_attention(q, k, v)
        b = K.cross_attention(q, kd, vd)
        assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, q, do)[0], torch.autograd.grad(b, q, do)[0])


def test_every_run_gives_the_same_bits_and_touches_nothing_else():
    K = ops()
    q, k, v, do = (rnd(s, i, torch.bfloat16).to(DEV) for i, s in enumerate(((2, 300, 4, 64), (2, 900, 2, 64), (2, 900, 2, 64), (2, 300, 4, 64))))
    before = [t.clone() for t in (q, k, v, do)]
    pad = mask_of("holes", 2, 900, 5).to(DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    first = None
    for _ in range(4):
        out = K.cross_attention(*leaves, pad)
        got = (out.detach(),) + torch.autograd.grad(out, leaves, do)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    assert all(torch.equal(a, b.detach()) for a, b in zip(before, (q, k, v, do)))


def test_second_derivatives_are_refused():
    K = ops()
    q = torch.randn(1, 4, 1, 32, device=DEV, requires_grad=True)
    g = torch.autograd.grad(K.cross_attention(q, q, q).sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)


# ---- embedding ------------------------------------------------------------------------------------------------------------------------
EMB = [(1, 1, 1), (7, 5, 3), (64, 1, 40), (1000, 17, 64), (4097, 300, 100), (5000, 70000, 36), (40000, 10, 8), (3000, 40000, 520), (33, 7, 2049),
       (70000, 257, 16)]


def emb_check(dw, ids, dout, V, scale, padding, dt):
    """dw against 64-bit sums; a sum of n terms in 32 bits is off by at most n e of their magnitudes, its product with scale by e"""
    n = ids.numel()
    g = dout.double().reshape(n, -1)
    keep = torch.ones(n, dtype=torch.bool) if padding is None else ids.reshape(-1) != padding
    keep &= (ids.reshape(-1) >= 0) & (ids.reshape(-1) < V)
    at = ids.reshape(-1)[keep].long()
    ref = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, at, g[keep])
    mag = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, at, g[keep].abs())
    cnt = torch.bincount(at, minlength=V).double()[:, None]
    u = half_step(dt)
    lim = abs(scale) * (u * ref.abs() + E * (cnt + 2) * mag) + (2.0 ** -25 if dt == torch.float16 else 0)
    assert dw.dtype == dt
    x = dw.cpu().double()
    assert bool(((x - scale * ref).abs() <= lim).all())
    assert not x[cnt[:, 0] == 0].any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", EMB, ids=lambda s: "x".join(map(str, s)))
def test_embedding_and_its_gradient(size, dtype):
    K, dt = ops(), DT[dtype]
    T, V, C = size
    g = torch.Generator().manual_seed(T)
    ids = (torch.rand(T, generator=g) ** 3 * V).long().clamp_(0, V - 1)          # low ids are hot
    w, do = rnd((V, C), 1, dt), rnd((T, C), 2, dt)
    scale, padding = 1.7, (int(ids[T // 2]) if T > 2 else None)
    wd = w.to(DEV).requires_grad_()
    for idt in (torch.int64, torch.int32):
        out = K.embedding(ids.to(DEV, idt), wd, scale, padding)
        exact = w[ids].double() * float(torch.tensor(scale, dtype=torch.float32))
        # the product in 32 bits and its rounding, or both at once (the compiler may fuse them: -0.51025390625 * 1.7 lies 2.4e-8 beyond the
        # middle of two fp16 numbers, and its fp32 value in the middle), so equality with either would be too much to ask
        lim = (half_step(dt) * (1 + 2 * E) + 2 * E) * exact.abs() + (2.0 ** -25 if dtype == "fp16" else 0)
        assert out.dtype == dt and bool(((out.detach().cpu().double() - exact).abs() <= lim).all())
        (dw,) = torch.autograd.grad(out, wd, do.to(DEV))
        emb_check(dw, ids, do, V, scale, padding, dt)
        assert torch.equal(dw, K.embedding_grad(do.to(DEV), ids.to(DEV, idt), V, scale, padding))


@pytest.mark.parametrize("T", [1, 31, 32, 33, 1023, 1024, 1025, 300001])
def test_one_id_for_all_tokens(T):
    """a run over every chunk of the sorted tokens"""
    K = ops()
    do = rnd((T, 12), 3, torch.float32)
    ids = torch.full((T,), 5)
    emb_check(K.embedding_grad(do.to(DEV), ids.to(DEV), 9, 0.5), ids, do, 9, 0.5, None, torch.float32)
    assert not K.embedding_grad(do.to(DEV), ids.to(DEV), 9, 0.5, 5).any()        # all of them padding


@pytest.mark.parametrize("C", [5, 64, 264])
def test_runs_of_many_chunks(C):
    """runs around 16, 64 and 128 chunks of 32 sorted tokens, which end at a chunk's border, one before or one behind it"""
    K = ops()
    lengths = [32 * n + x for n in (1, 2, 16, 17, 63, 64, 65, 128, 129, 200, 600) for x in (-1, 0, 1)]
    ids = torch.repeat_interleave(torch.arange(len(lengths)) + 300, torch.tensor(lengths))      # two digits
    ids = torch.cat([torch.zeros(130000 - len(ids), dtype=torch.long), ids])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))]
    do = rnd((len(ids), C), 4, torch.float32)
    emb_check(K.embedding_grad(do.to(DEV), ids.to(DEV), 400), ids, do, 400, 1.0, None, torch.float32)


def test_order_of_equal_ids_is_fixed():
    """1, 2^24, -2^24, 1 in fp32 depends on its order: the sum runs over ascending tokens, every time"""
    K = ops()
    do = torch.tensor([1.0, 2.0 ** 24, -2.0 ** 24, 1.0])[:, None].repeat(1, 64)
    ids = torch.tensor([3, 3, 3, 3])
    for _ in range(3):
        assert torch.equal(K.embedding_grad(do.to(DEV), ids.to(DEV), 4)[3].cpu(), torch.full((64,), 1.0))
    do, ids = rnd((100000, 24), 1, torch.float32).to(DEV), torch.randint(0, 5000, (100000,)).to(DEV)
    first = K.embedding_grad(do, ids, 5000)
    assert all(torch.equal(first, K.embedding_grad(do, ids, 5000)) for _ in range(3))


def test_ids_outside_the_table():
    K = ops()
    w = rnd((10, 16), 1, torch.float32).to(DEV)
    ids = torch.tensor([[0, 9], [10, -1], [2 ** 40, -2 ** 40], [3, 2 ** 32 + 3]]).to(DEV)
    out = K.embedding(ids, w)
    bad = (ids < 0) | (ids >= 10)
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], w[ids[~bad]])
    do = torch.ones(4, 2, 16, device=DEV)
    dw = K.embedding_grad(do, ids, 10)
    assert torch.equal(dw.sum(1), torch.tensor([16.0, 0, 0, 16, 0, 0, 0, 0, 0, 16], device=DEV))
    assert not K.embedding_grad(do, torch.full_like(ids, -7), 10).any()
    assert torch.equal(K.embedding_grad(do, ids, 10, 1.0, -1), K.embedding_grad(do, ids, 10, 1.0, 9))     # -1: the last row


def test_embedding_layouts_and_empty_inputs():
    K = ops()
    table = rnd((50, 80), 1, torch.bfloat16).to(DEV)
    ids = torch.randint(0, 50, (6, 7)).to(DEV)
    for w in (table[:, 8:40], table[:, 3:20], table.t()[:50, :50].t(), table[::2][:, :16]):
        i = ids % w.shape[0]
        leaf = w.detach().requires_grad_()
        out = K.embedding(i.t(), leaf)
        assert torch.equal(out.detach(), w[i.t()])
        do = rnd(out.shape, 2, torch.bfloat16).to(DEV)
        a = torch.autograd.grad(out, leaf, do)[0]
        emb_check(a, i.t().cpu(), do.cpu(), w.shape[0], 1.0, None, torch.bfloat16)
    out = K.embedding(ids, table.clone().requires_grad_())
    assert torch.equal(torch.autograd.grad(out.sum(), out.grad_fn.next_functions[0][0].variable)[0].float().sum(1) / 80,
                       torch.bincount(ids.reshape(-1), minlength=50).float())    # the gradient of a sum is an expanded scalar
    none = K.embedding(ids[:0], table.requires_grad_())
    assert none.shape == (0, 7, 80) and not torch.autograd.grad(none.sum(), table)[0].any()
    assert K.embedding(ids[0, 0], table).shape == (80,)


# ---- as they are used ------------------------------------------------------------------------------------------------------------------
def chain(ids, table, x, blk, pad):
    return blk(x, ops().embedding(ids, table, table.shape[1] ** 0.5, 0), pad)


def plain_chain(ids, table, x, blk, pad):
    """CrossAttnBlock over embedded tokens in 64 bits on the CPU"""
    P = {n: p.detach().cpu().double().requires_grad_() for n, p in blk.named_parameters()}
    ctx = F.embedding(ids, table, padding_idx=0) * table.shape[1] ** 0.5
    B, C, H, W = x.shape
    h = F.group_norm(x, 32, P["norm.weight"], P["norm.bias"], 1e-5).flatten(2).transpose(1, 2)
    heads = blk.num_heads
    q = F.linear(h, P["q.weight"], P["q.bias"]).view(B, H * W, heads, -1).transpose(1, 2)
    k, v = F.linear(ctx, P["kv.weight"], P["kv.bias"]).view(B, ids.shape[1], 2, heads, -1).permute(2, 0, 3, 1, 4)
    s = q @ k.transpose(2, 3) * (C // heads) ** -0.5
    a = torch.softmax(s.masked_fill(pad[:, None, None], -math.inf), 3).nan_to_num(0.0)
    o = (a @ v).transpose(1, 2).reshape(B, H * W, C)
    return x + F.linear(o, P["proj.weight"], P["proj.bias"]).transpose(1, 2).reshape(B, C, H, W), P


def make_block():
    from models.codec import CrossAttnBlock
    torch.manual_seed(3)
    return CrossAttnBlock(64, 48, num_heads=4).to(DEV)


def test_block_over_embedded_tokens_against_64_bits():
    """ids -> embedding -> CrossAttnBlock -> loss, with every gradient down to the table.  The block's convs are the framework's fp32-grade
    ones (3.7e-7 rms of their range); the chain has five of them and a softmax: 1e-4 of each tensor's largest value, as for AttnBlock"""
    blk = make_block()
    ids = torch.randint(1, 90, (3, 21), generator=torch.Generator().manual_seed(1))
    ids[0, 15:] = 0
    ids[2, 3:] = 0
    pad = ids == 0
    x, table, do = rnd((3, 64, 8, 8), 2, torch.float32), rnd((90, 48), 3, torch.float32, 0.3), rnd((3, 64, 8, 8), 4, torch.float32)
    xd, td = x.to(DEV).requires_grad_(), table.to(DEV).requires_grad_()
    y = chain(ids.to(DEV), td, xd, blk, pad.to(DEV))
    y.backward(do.to(DEV))
    x64, t64 = x.double().requires_grad_(), table.double().requires_grad_()
    y64, P = plain_chain(ids, t64, x64, blk, pad)
    y64.backward(do.double())
    pairs = [("y", y, y64), ("x", xd.grad, x64.grad), ("table", td.grad, t64.grad)] + [(n, p.grad, P[n].grad) for n, p in blk.named_parameters()]
    for n, a, b in pairs:
        assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= 1e-4 * float(b.detach().abs().max()), n
    assert not td.grad[0].any()


def test_other_stream_and_two_graphs_with_replays():
    """one decoding step and one training step on a side stream and as captured graphs that live side by side, replayed in turn with eager
    work and synchronisation between them: every result is the eager one"""
    K = ops()
    q, k, v = (rnd(s, i, torch.bfloat16).to(DEV) for i, s in enumerate(((2, 1, 4, 64), (2, 3000, 2, 64), (2, 3000, 2, 64))))
    qt, kt, vt, do = (rnd(s, i, torch.float32).to(DEV) for i, s in enumerate(((2, 200, 4, 32), (2, 600, 4, 32), (2, 600, 4, 32), (2, 200, 4, 32))))
    ids, dout = torch.randint(0, 3000, (700,)).to(DEV), rnd((700, 40), 9, torch.float32).to(DEV)
    pad = mask_of("tail", 2, 3000, 3).to(DEV)

    def step():
        with torch.no_grad():
            return (K.cross_attention(q, k, v, pad),)

    def train():
        leaves = [t.detach().requires_grad_() for t in (qt, kt, vt)]
        out = K.cross_attention(*leaves)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do) + (K.embedding_grad(dout, ids, 3000),)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        on_side = step() + train()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_side, step() + train()))
    graphs = []
    for fn in (step, train):
        with torch.cuda.stream(side):
            fn()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = fn()
        graphs.append((g, fn, res))
    for n in range(3):
        for t in (q, k, v, qt, kt, vt, do, dout):
            t.mul_(-1.25 if n != 1 else 0.7)
        ids.add_(1).remainder_(3000)
        for g, fn, res in graphs + graphs[::-1]:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, fn()))
