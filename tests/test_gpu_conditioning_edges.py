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


# every form of the forward pass: (Lq, Lk, query heads of a key head, D)
FORMS = {"token": (1, 300, 1, 64), "split token": (1, 5000, 4, 64), "wide token": (3, 500, 1, 128), "few rows": (20, 700, 1, 64),
         "wide few rows": (30, 600, 2, 128), "resident keys": (100, 70, 1, 64), "resident wide": (150, 60, 1, 128), "many rows": (200, 300, 1, 64),
         "many wide rows": (140, 300, 1, 128), "split rows": (70, 3000, 1, 64)}


def case(dtype, form, seed=1):
    Lq, Lk, G, D = FORMS[form]
    dt = DT[dtype]
    return rnd((2, Lq, 2 * G, D), seed, dt), rnd((2, Lk, 2, D), seed + 1, dt), rnd((2, Lk, 2, D), seed + 2, dt), rnd((2, Lq, 2 * G, D), seed + 3, dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_an_infinite_value_is_an_infinity(form, dtype):
    """every probability is above exp(-20) here and far from underflow, so one infinity among a column's values is the column's sum, two of
    opposite signs are a NaN, and no other column, head or sequence is touched"""
    K = ops()
    Lq, Lk, G, D = FORMS[form]
    q, k, v, _ = (t.to(DEV) for t in case(dtype, form))
    scale = D ** -0.5
    ref = K.cross_attention(q, k, v, None, scale)
    for sign in (1, -1):
        for j in (0, 7, Lk - 1):
            v2 = v.clone()
            v2[1, j, 1, 9] = sign * math.inf
            v2[1, Lk // 2, 1, 9] = sign * math.inf
            out = K.cross_attention(q, k, v2, None, scale)
            assert bool((out[1, :, G:, 9] == sign * math.inf).all())
            out[1, :, G:, 9] = ref[1, :, G:, 9]
            assert torch.equal(out, ref)
    v2[1, Lk // 3, 1, 9] = math.inf
    out = K.cross_attention(q, k, v2, None, scale)
    assert bool(out[1, :, G:, 9].isnan().all())
    out[1, :, G:, 9] = ref[1, :, G:, 9]
    assert torch.equal(out, ref)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_an_infinite_key_takes_no_part_or_all(form, dtype):
    """a score of -infinity is a key that is not there (its value and key get gradients of 0, and 0 times the infinity is a NaN in the
    query's gradient, in that column), one of +infinity a NaN row, as the signs of the queries say"""
    Lq, Lk, G, D = FORMS[form]
    q, k, v, do = case(dtype, form)
    q[..., 5] = q[..., 5].abs() + 0.125
    pad = torch.zeros(2, Lk, dtype=torch.bool)
    pad[1, 11] = True
    val, bound = oracle(q, k, v, pad, D ** -0.5, do)
    k2 = k.clone()
    k2[1, 11, :, 5] = -math.inf
    got = run(q, k2, v, None, D ** -0.5, do)
    assert bool(got["dq"][1, :, :, 5].isnan().all())
    got["dq"][1, :, :, 5] = val["dq"][1, :, :, 5].to(DEV, DT[dtype])
    check(got, val, bound, DT[dtype], norms=False)
    q[1, ::2, :, 5] *= -1
    out = ops().cross_attention(*(t.to(DEV) for t in (q, k2, v)), None, D ** -0.5)
    assert bool(out[1, ::2].isnan().all())
    val, bound = oracle(q, k, v, pad, D ** -0.5, do)
    out[1, ::2] = val["out"][1, ::2].to(DEV, DT[dtype])
    check({"out": out}, val, bound, DT[dtype], norms=False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_an_infinite_output_gradient(form, dtype):
    """reaches its column of the values' gradient as an infinity, its row and its head's keys as no finite number, and nothing else"""
    Lq, Lk, G, D = FORMS[form]
    q, k, v, do = case(dtype, form)
    clean = run(q, k, v, None, D ** -0.5, do)
    for sign in (1, -1):
        do2 = do.clone()
        do2[1, Lq // 2, -1, 3] = sign * math.inf
        got = run(q, k, v, None, D ** -0.5, do2)
        assert bool((got["dv"][1, :, 1, 3] == sign * math.inf).all())
        assert not bool(torch.isfinite(got["dq"][1, Lq // 2, -1]).any() or torch.isfinite(got["dk"][1, :, 1]).any())
        got["dv"][1, :, 1, 3] = clean["dv"][1, :, 1, 3]
        got["dq"][1, Lq // 2, -1] = clean["dq"][1, Lq // 2, -1]
        got["dk"][1, :, 1] = clean["dk"][1, :, 1]
        for n, t in got.items():
            assert torch.equal(t, clean[n]), n


@pytest.mark.parametrize("form", list(FORMS))
def test_the_largest_fp32_keys_are_numbers(form):
    """keys between bf16's largest (3.3895e38) and fp32's, beside queries of 2^-124: scores of ordinary size"""
    Lq, Lk, G, D = FORMS[form]
    q, k, v, do = case("fp32", form)
    q[..., 5] = torch.where(q[..., 5] > 0, 2.0 ** -124, -2.0 ** -124)
    k[:, ::3, :, 5] = torch.linspace(3.39e38, torch.finfo(torch.float32).max, len(k[0, ::3]))[None, :, None]
    do *= 2.0 ** -8                                                              # the queries' gradient in column 5 stays in the type
    got = run(q, k, v, None, D ** -0.5, do)
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    val, bound = oracle(q, k, v, None, D ** -0.5, do)
    # the keys' gradients in column 5 are sums of products with 2^-124 and lie below the smallest normal number, on the grid of 2^-149: each
    # of the roundings of such a sum (six products of every row, the scale, the split sums) is off by half a step of it, 2^-150
    bound["dk"][..., 5] += (6 * G * Lq + 8) * 2.0 ** -150
    check(got, val, bound, torch.float32, norms=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", list(FORMS))
def test_the_largest_values_are_numbers(form, dtype):
    """values next to the type's largest (fp32: beyond bf16's, 3.3895e38), as keys beside queries of 2^-124, and as values under no output
    gradient (whose product with them would leave the type): their sums with undivided probabilities leave 32 bits, the results do not"""
    Lq, Lk, G, D = FORMS[form]
    q, k, v, do = case(dtype, form)
    low, most = 3.39e38 if dtype == "fp32" else 3.3e38, torch.finfo(DT[dtype]).max
    q[..., 5] = torch.where(q[..., 5] > 0, 2.0 ** -124, -2.0 ** -124)
    k[:, ::3, :, 5] = torch.linspace(low, most, len(k[0, ::3]))[None, :, None].to(DT[dtype])
    v[:, 1::5, :, 2] = -torch.linspace(low, most, len(v[0, 1::5]))[None, :, None].to(DT[dtype])
    do[..., 2] = 0.0
    do *= 2.0 ** -8                                                              # the queries' gradient in column 5 stays in the type
    got = run(q, k, v, None, D ** -0.5, do)
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    val, bound = oracle(q, k, v, None, D ** -0.5, do)
    bound["dk"][..., 5] += (6 * G * Lq + 8) * 2.0 ** -150                        # below the normal numbers, as in the test of the largest keys
    if dtype == "bf16":
        bound["dk"][..., 5] += 2.0 ** -134                                       # and rounded to bf16's grid there, 2^-133
    check(got, val, bound, DT[dtype], norms=False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("gap", [21.5, 24.3, 26.7])
@pytest.mark.parametrize("form", list(FORMS))
def test_small_probabilities_keep_their_bits(form, gap, dtype):
    """a key that takes almost everything and whose value is 0, and all others alike, 2^gap below it: nothing averages the rounding of their
    probabilities, which is that of a normal number of the type"""
    Lq, Lk, G, D = FORMS[form]
    dt = DT[dtype]
    q, k, v, do = case(dtype, form)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[..., 1:] = 0.0
    k[:, 1, :, 0] = gap * math.log(2.0)
    v = (v.abs() * 1024 + 512).to(dt)                                            # results that are normal numbers
    v[:, 1] = 0.0
    check(run(q, k, v, None, 0.125, do), *oracle(q, k, v, None, 0.125, do), dt, norms=False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_sequences_without_keys_give_zeros_whatever_their_queries_hold(form, dtype):
    """and gradients of zeros; a sequence that has keys is not touched"""
    Lq, Lk, G, D = FORMS[form]
    q, k, v, do = case(dtype, form)
    pad = torch.zeros(2, Lk, dtype=torch.bool)
    pad[0] = True
    clean = run(q, k, v, pad, D ** -0.5, do)
    q[0, :, ::2] = math.nan
    q[0, :, 1::2, 3] = -math.inf
    k[0, ::2], v[0, 1::2] = math.inf, math.nan
    got = run(q, k, v, pad, D ** -0.5, do)
    for n, t in got.items():
        assert not t[0].any() and not t[0].isnan().any(), n
        assert torch.equal(t, clean[n]), n


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_scores_of_any_finite_size(form, dtype):
    """scores of 1e8 (fp16) and 1e12, whose spacing in 32 bits is more than a softmax can resolve: a row is its largest score's value where
    the next one is out of reach of the scores' own rounding, (D + 8) 2^-24 of the products' magnitudes, and an average of values elsewhere"""
    Lq, Lk, G, D = FORMS[form]
    dt = DT[dtype]
    q, k, v, _ = case(dtype, form)
    gain = 1e4 if dtype == "fp16" else 1e6
    q, k = (q.double() * gain).to(dt), (k.double() * gain).to(dt)
    out = ops().cross_attention(*(t.to(DEV) for t in (q, k, v)), None, 0.125).cpu().double()
    qh, kh, vh = q.double().transpose(1, 2), *(t.double().repeat_interleave(G, 2).transpose(1, 2) for t in (k, v))
    s, mag = 0.125 * qh @ kh.transpose(2, 3), 0.125 * qh.abs() @ kh.abs().transpose(2, 3)
    top = s.topk(2, 3)
    clear = top.values[..., 0] - top.values[..., 1] > 2 * (D + 8) * 2.0 ** -24 * mag.amax(3) + 1000
    best = torch.gather(vh, 2, top.indices[..., :1].expand(-1, -1, -1, D)).transpose(1, 2)
    assert float(clear.double().mean()) > 0.9 and bool(torch.isfinite(out).all())
    assert torch.equal(out[clear.transpose(1, 2)], best[clear.transpose(1, 2)])
    assert bool((out.abs() <= vh.abs().amax(2)[:, None] * (1 + 2 * half_step(dt))).all())


def test_block_over_no_states_is_the_identity_and_its_bias():
    """a prompt of length 0, as one that is all padding: the same result, and gradients of zeros for what nothing depends on"""
    from models.codec import CrossAttnBlock
    torch.manual_seed(3)
    blk = CrossAttnBlock(64, 48, num_heads=4).to(DEV)
    x, do = rnd((3, 64, 8, 8), 2, torch.float32).to(DEV).requires_grad_(), rnd((3, 64, 8, 8), 4, torch.float32).to(DEV)
    results = []
    for states, pad in ((torch.zeros(3, 0, 48, device=DEV), torch.zeros(3, 0, dtype=torch.bool, device=DEV)), (torch.zeros(3, 0, 48, device=DEV), None),
                        (torch.ones(3, 5, 48, device=DEV), torch.ones(3, 5, dtype=torch.bool, device=DEV))):
        states.requires_grad_()
        y = blk(x, states, pad)
        leaves = [x, states] + list(blk.parameters())
        results.append([y] + list(torch.autograd.grad(y, leaves, do)))
        names = ["y", "x", "states"] + [n for n, _ in blk.named_parameters()]
        assert torch.equal(y, x + blk.proj.bias[:, None, None]) and torch.equal(results[-1][1], do)
        for n, t in zip(names, results[-1]):
            assert bool(torch.isfinite(t).all()) and (n in ("y", "x", "proj.bias") or not t.any()), n
    for n, a, b in zip(names, results[0], results[2]):
        assert n == "states" or torch.equal(a, b), n


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["tail", "holes", "empty"])
@pytest.mark.parametrize("D", [40, 64, 128])
def test_many_row_tiles_and_heads_over_many_keys(dtype, kind, D):
    """the general form (more keys than stay in LDS) with ragged lengths, several row tiles of every head and many heads"""
    dt = DT[dtype]
    B, Lq, Lk, H, Hkv = 4, 333, 450, 8, 4
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of(kind, B, Lk, 6)
    check(run(q, k, v, pad, D ** -0.5, do), *oracle(q, k, v, pad, D ** -0.5, do), dt)


@pytest.mark.parametrize("dtype", list(DT))
def test_resident_keys_under_many_row_tiles(dtype):
    """keys that stay in LDS while every workgroup goes through several row tiles, the last one partial; ragged lengths"""
    dt = DT[dtype]
    B, Lq, Lk, H, Hkv, D = 16, 1030, 70, 16, 16, 24
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of("empty", B, Lk, 6)
    check(run(q, k, v, pad, 0.3, do), *oracle(q, k, v, pad, 0.3, do), dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 8, 70000, 1, 1, 64), (1, 70000, 64, 1, 1, 64), (1, 3, 30000, 2, 1, 128), (1, 20000, 3, 2, 1, 128), (2, 1, 40000, 4, 2, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_hundreds_of_splits(shape, dtype):
    """few queries over long keys (dq is summed over many splits) and few keys under many rows (dk and dv are)"""
    dt = DT[dtype]
    B, Lq, Lk, H, Hkv, D = shape
    q, k, v, do = rnd((B, Lq, H, D), 1, dt), rnd((B, Lk, Hkv, D), 2, dt), rnd((B, Lk, Hkv, D), 3, dt), rnd((B, Lq, H, D), 4, dt)
    pad = mask_of("holes", B, Lk, 5)
    first = run(q, k, v, pad, D ** -0.5, do)
    check(first, *oracle(q, k, v, pad, D ** -0.5, do), dt)
    for n, t in run(q, k, v, pad, D ** -0.5, do).items():
        assert torch.equal(t, first[n]), n


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_infinite_values_beside_padding(form, dtype):
    """the pass with care sees the same mask: infinities and NaN among padded keys and one infinity among live ones, another sequence all
    padding"""
    K = ops()
    Lq, Lk, G, D = FORMS[form]
    q, k, v, _ = (t.to(DEV) for t in case(dtype, form))
    pad = mask_of("holes", 2, Lk, 7).to(DEV)
    pad[0], pad[1, 4] = True, False
    k[pad], v[pad] = 0.0, 0.0
    ref = K.cross_attention(q, k, v, pad)
    k[pad], v[pad] = math.nan, -math.inf
    v[1, 4, 1, 9] = math.inf
    out = K.cross_attention(q, k, v, pad)
    assert bool((out[1, :, G:, 9] == math.inf).all())
    out[1, :, G:, 9] = ref[1, :, G:, 9]
    assert torch.equal(out, ref)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", list(FORMS))
def test_rows_without_a_score_and_nan_inputs(form, dtype):
    """a row that has keys, all of whose scores are -infinity, is the formula's NaN (0 / 0), whatever stands beside the last key; a NaN in a
    query is its row's, in a key its head's, in a value its column's"""
    K = ops()
    Lq, Lk, G, D = FORMS[form]
    q, k, v, _ = (t.to(DEV) for t in case(dtype, form))
    k[..., 5] = k[..., 5].abs() + 0.125
    ref = K.cross_attention(q, k, v)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    q2[1, Lq // 2, 0, 5], q2[0, 0, -1, 3] = -math.inf, math.nan
    out = K.cross_attention(q2, k, v)
    assert bool(out[1, Lq // 2, 0].isnan().all()) and bool(out[0, 0, -1].isnan().all())
    out[1, Lq // 2, 0], out[0, 0, -1] = ref[1, Lq // 2, 0], ref[0, 0, -1]
    assert torch.equal(out, ref)
    some = k.clone()                                                             # the same by infinite keys; one key without an infinity is enough
    some[:, :, 0, 5] = -math.inf
    q3 = q.clone()
    q3[..., 5] = q3[..., 5].abs() + 0.125
    assert bool(K.cross_attention(q3, some, v)[:, :, :G].isnan().all())
    some[1, 40, 0] = k[1, 40, 0]
    # p v / p, p near 1: the product, the reciprocal, its product and a join's are off by 2^-24 each; p and the result are rounded to 16 bits
    lim = (4 * 2.0 ** -24 + (0 if dtype == "fp32" else 2 * half_step(DT[dtype]))) * v[1, 40, 0].double().abs()
    assert bool(((K.cross_attention(q3, some, v)[1, :, :G].double() - v[1, 40, 0].double()).abs() <= lim).all())
    k2[0, Lk // 2, 1, 7], v2[0, 3, 0, 2] = math.nan, math.nan
    out = K.cross_attention(q, k2, v2)
    assert bool(out[0, :, G:].isnan().all()) and bool(out[0, :, :G, 2].isnan().all())
    out[0, :, G:], out[0, :, :G, 2] = ref[0, :, G:], ref[0, :, :G, 2]
    assert torch.equal(out, ref)
