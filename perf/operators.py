"""Measured cases of the conditioning operators: attention of image tokens to another sequence's states, and the token embedding that such
a sequence starts from.

    cross_attention(q, k, v)   out[b,i,h] = sum_j p[b,h,i,j] v[b,j,h'],  p = softmax_j over the keys that are not padding of
                               scale * <q[b,i,h], k[b,j,h']>,  h' = h // (H // Hkv); a row without keys gives zeros
    embedding(ids, weight)     out[t] = scale * weight[ids[t]];  its gradient dweight[v] = scale * sum of dout[t] over ids[t] == v

With `own` false run() computes them in elementary torch operations, in 32 bits, rounded once; with `own` true it makes the calls of
favae_hip.ops.  A "train" case is one forward and one backward pass and returns the output with every gradient.
"""
import math
import os
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    """the framework's operators, imported once (its package root is fa-vae_amd/)"""
    pkg = os.path.join(os.getcwd(), "fa-vae_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from favae_hip import ops
    return ops


# ---------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------
def _attend(name, op, dtype, B, Lq, Lk, H, Hkv, D, mask, packed=False):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D, "mask": mask, "packed": packed}


def _embed(name, op, dtype, B, L, V, C, ids, scale):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "L": L, "V": V, "C": C, "ids": ids, "scale": scale}


def listed():
    return [
        # one decoding step of a batch that attends to short padded prompts: a call whose latency counts
        _attend("token to prompt", "attend", "bf16", 32, 1, 77, 8, 8, 64, "tail", True),
        # one decoding step over long states with shared key / value heads: the states' bytes are the work
        _attend("token to long states", "attend", "fp16", 4, 1, 30011, 32, 8, 128, "tail"),
        # sampling: a 64 x 64 feature map of 8 heads attends to a padded prompt
        _attend("map to prompt", "attend", "bf16", 16, 4096, 77, 8, 8, 64, "tail", True),
        # the framework's own type and wide heads, no padding
        _attend("fp32 wide heads", "attend", "fp32", 4, 2048, 2048, 4, 4, 128, "none"),
        # training at the 16 x 16 latent of the 256 x 256 models, batch 32, in the framework's own type
        _attend("train latents to prompt", "attend_train", "fp32", 32, 256, 77, 8, 8, 64, "tail", True),
        # training, a 64 x 64 map to a 32 x 32 map: the largest products
        _attend("train map to map", "attend_train", "bf16", 8, 4096, 1024, 8, 8, 64, "none", True),
        # ragged sizes, shared heads, scattered padding, a head size between the powers of two
        _attend("train odd sizes", "attend_train", "fp16", 3, 1021, 515, 12, 4, 80, "holes"),
        # small windows of which some have no key at all
        _attend("train empty rows", "attend_train", "bf16", 16, 64, 130, 8, 2, 32, "empty"),
        # one token of one sequence: pure latency
        _embed("embed one token", "embed", "bf16", 1, 1, 1024, 256, "uniform", 1.0),
        # long prompts of a batch, rows scaled by sqrt(C)
        _embed("embed long rows", "embed", "fp16", 16, 4096, 16384, 1024, "zipf", 32.0),
        # the codes of a batch of 16 images (64 x 64 indices of 256 dimensions), trained in the framework's own type
        _embed("train codes", "embed_train", "fp32", 16, 4096, 8192, 256, "uniform", 1.0),
        # text tokens of a large vocabulary: a few rows are hot, many are never met, the padding row gets no gradient
        _embed("train text tokens", "embed_train", "bf16", 64, 1024, 49999, 768, "zipf", 27.712812921102035),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if rng.random() < 0.6:
        train = rng.random() < 0.5
        Hkv, G = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 4))
        D = rng.choice((32, 64, 64, 128, 8 * rng.randint(1, 16)))
        Lq = 1 if rng.random() < 0.2 else _log(rng, 1, 4096)
        Lk = _log(rng, 1, 8192)
        B = _log(rng, 1, 32)
        H, products = Hkv * G, 7 if train else 2
        while B * H * Lq * Lk > 2e8 or B * H * Lq * Lk * D * products > 1e11 or B * Lq * H * D > 1.6e7 or B * Lk * Hkv * D > 3e7:
            B, Lq, Lk = (B // 2, Lq, Lk) if B > 1 else (1, max(1, Lq // 2), (Lk + 1) // 2)
        return {"op": "attend_train" if train else "attend", "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D,
                "mask": rng.choice(("none", "tail", "holes", "empty")), "packed": rng.random() < 0.5}
    train = rng.random() < 0.6
    B, L, V = _log(rng, 1, 64), _log(rng, 1, 1024), _log(rng, 8, 50000)
    C = rng.choice((64, 128, 256, 512, 768, 1024, rng.randint(1, 1024)))
    while (B * L * (2 if train else 1) + (V if train else 0)) * C > (7e7 if dtype == "fp32" else 1.4e8):
        L, V = L // 2, V // 2
    return {"op": "embed_train" if train else "embed", "dtype": dtype, "B": B, "L": L, "V": V, "C": C,
            "ids": rng.choice(("uniform", "zipf")), "scale": rng.choice((1.0, 0.5, math.sqrt(C)))}


def _lengths(case):
    """keys of each batch element that are not padding, before they are shuffled ("holes": about that many, scattered)"""
    B, Lk = case["B"], case["Lk"]
    if case["mask"] == "none":
        return [Lk] * B
    n = [max(1, Lk - (b * Lk) // (2 * B)) for b in range(B)]
    if case["mask"] == "empty":
        n = [0 if b % 4 == 3 else n[b] for b in range(B)]
    return n


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"].startswith("attend"):
        keys = sum(_lengths(case))
        rows = case["B"] * case["Lq"] * case["H"] * case["D"] * es             # q, or any other tensor of its shape
        cols = keys * case["Hkv"] * case["D"] * es                             # k or v
        mask = 0 if case["mask"] == "none" else case["B"] * case["Lk"]
        product = 2.0 * case["H"] * case["Lq"] * keys * case["D"]
        if case["op"] == "attend":
            return {"bytes": 2 * rows + 2 * cols + mask, "flops": 2 * product}
        return {"bytes": 4 * rows + 4 * cols + mask, "flops": 7 * product}     # + dout, dq; dk, dv; five products of the backward pass
    T, C, V = case["B"] * case["L"], case["C"], case["V"]
    forward = 8 * T + (T + min(T, V)) * C * es
    if case["op"] == "embed":
        return {"bytes": forward, "flops": T * C}
    return {"bytes": forward + (T + V) * C * es, "flops": 3.0 * T * C}


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------
def _rows_of(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DT[case["dtype"]]
    train = case["op"].endswith("train")
    if case["op"].startswith("attend"):
        B, Lq, Lk, H, Hkv, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "D"))
        q = _rows_of(gen, (B, Lq, H, D), dt)
        if case["packed"]:                                                     # keys and values of ONE projection, as views of it
            k, v = _rows_of(gen, (B, Lk, 2, Hkv, D), dt).unbind(2)
        else:
            k, v = _rows_of(gen, (B, Lk, Hkv, D), dt), _rows_of(gen, (B, Lk, Hkv, D), dt)
        pad = None
        if case["mask"] != "none":
            n = torch.tensor(_lengths(case), device="cuda")[torch.randperm(B, generator=gen, device="cuda")]
            if case["mask"] == "holes":
                at = torch.rand((B, Lk), generator=gen, device="cuda").argsort(1)
            else:
                at = torch.arange(Lk, device="cuda").expand(B, Lk)
            pad = at >= n[:, None]
        if train:
            q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        return {"op": case["op"], "q": q, "k": k, "v": v, "pad": pad, "scale": 1.0 / math.sqrt(D),
                "dout": _rows_of(gen, (B, Lq, H, D), dt) if train else None}
    B, L, V, C = (case[k] for k in ("B", "L", "V", "C"))
    weight = _rows_of(gen, (V, C), dt)
    u = torch.rand((B, L), generator=gen, device="cuda", dtype=torch.float64)
    if case["ids"] == "zipf":                                                  # density ~ 1 / rank over a shuffled vocabulary
        rank = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        ids = torch.randperm(V, generator=gen, device="cuda")[rank]
    else:
        ids = (u * V).long().clamp_(0, V - 1)
    padding = int(ids[0, -1]) if case["ids"] == "zipf" else None               # some row of the table serves as padding
    if padding is not None:                                                    # a quarter of the sequences end in padding
        ids[::4, (L + 1) // 2:] = padding
    return {"op": case["op"], "ids": ids, "weight": weight, "scale": case["scale"], "padding": padding,
            "dout": _rows_of(gen, (B, L, C), dt) if train else None}


# ---------------------------------------------------------------------------------------------------------------------------------
# the operators in plain form
# ---------------------------------------------------------------------------------------------------------------------------------
def _by_head(t, Hkv):
    """(B, L, H, D) -> (B, Hkv, G L, D) in 32 bits: the G query heads that share a key / value head follow one another"""
    B, L, H, D = t.shape
    return t.float().view(B, L, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, (H // Hkv) * L, D)


def _by_token(t, L, dtype):
    B, Hkv, R, D = t.shape
    return t.view(B, Hkv, R // L, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, Hkv * (R // L), D).to(dtype)


def _plain_probabilities(q, k, pad, scale):
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    if pad is not None:
        s = s.masked_fill(pad[:, None, None, :], -math.inf)
    m = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    n = e.sum(3, keepdim=True)
    return e / torch.where(n == 0, torch.ones_like(n), n)


@torch.no_grad()
def _plain_attend(s):
    Lq, Hkv, dt = s["q"].shape[1], s["k"].shape[2], s["q"].dtype
    q, k, v = (_by_head(t, Hkv) for t in (s["q"], s["k"], s["v"]))
    p = _plain_probabilities(q, k, s["pad"], s["scale"])
    o = torch.matmul(p, v)
    out = _by_token(o, Lq, dt)
    if s["dout"] is None:
        return out
    do = _by_head(s["dout"], Hkv)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(3, keepdim=True)) * s["scale"]
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    return out, _by_token(dq, Lq, dt), dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt)


@torch.no_grad()
def _plain_embed(s):
    w, ids = s["weight"], s["ids"]
    out = (w[ids].float() * s["scale"]).to(w.dtype)
    if s["dout"] is None:
        return out
    C = w.shape[1]
    dout = s["dout"].reshape(-1, C).float()
    if s["padding"] is not None:
        dout = dout * (ids.reshape(-1, 1) != s["padding"])
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids.reshape(-1), dout)
    return out, (dw * s["scale"]).to(w.dtype)


def run(state):
    if not own:
        return _plain_attend(state) if state["op"].startswith("attend") else _plain_embed(state)
    K = _ops()
    if state["op"].startswith("attend"):
        q, k, v = state["q"], state["k"], state["v"]
        out = K.cross_attention(q, k, v, state["pad"], state["scale"])
        return out if state["dout"] is None else (out.detach(),) + torch.autograd.grad(out, (q, k, v), state["dout"])
    out = K.embedding(state["ids"], state["weight"], state["scale"], state["padding"])
    if state["dout"] is None:
        return out
    return out, K.embedding_grad(state["dout"], state["ids"], state["weight"].shape[0], state["scale"], state["padding"])


# ---------------------------------------------------------------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------
def _exact_attend(s):
    """each batch element and head by itself, over the keys that are not padding only; gradients by differentiation"""
    B, _, H, D = s["q"].shape
    group = H // s["k"].shape[2]
    q, k, v = (s[n].detach().double().requires_grad_() for n in ("q", "k", "v"))
    rows = []
    for b in range(B):
        keep = torch.arange(k.shape[1], device="cuda") if s["pad"] is None else (~s["pad"][b]).nonzero()[:, 0]
        heads = []
        for h in range(H):
            kb, vb = (t[b, :, h // group][keep] for t in (k, v))
            if keep.numel() == 0:
                heads.append(q[b, :, h] * 0.0)
                continue
            w = torch.softmax((q[b, :, h] @ kb.t()) * s["scale"], 1)
            heads.append(w @ vb)
        rows.append(torch.stack(heads, 1))
        if s["dout"] is not None:                                              # element by element, so that the graphs stay small
            rows[-1].backward(s["dout"][b].double())
            rows[-1] = rows[-1].detach()
        else:
            rows[-1] = rows[-1].detach()
    out = torch.stack(rows, 0)
    return out if s["dout"] is None else (out, q.grad, k.grad, v.grad)


def _exact_embed(s):
    w, ids = s["weight"].detach().double(), s["ids"].reshape(-1)
    out = (torch.index_select(w, 0, ids) * s["scale"]).view(*s["ids"].shape, w.shape[1])
    if s["dout"] is None:
        return out
    g = s["dout"].double().reshape(-1, w.shape[1])
    keep = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids != s["padding"]
    order = torch.argsort(ids[keep], stable=True)                              # sums of runs of equal ids, as differences of prefix sums per run
    key, g = ids[keep][order], g[keep][order]
    row, count = torch.unique_consecutive(key, return_counts=True)
    sums = torch.segment_reduce(g, "sum", lengths=count) if row.numel() else g
    dw = torch.zeros_like(w)
    dw[row] = sums * s["scale"]
    return out, dw


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"].startswith("attend"):
        if s["dout"] is None:
            with torch.no_grad():
                return _exact_attend(s)
        return _exact_attend(s)
    with torch.no_grad():
        return _exact_embed(s)
