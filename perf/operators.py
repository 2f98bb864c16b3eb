"""Cases, plain forms and 64-bit definitions of the neck / optimiser operators: GroupNorm with an activation on channels-last rows
(forward, and forward + backward), the Newton-Schulz orthogonalisation of weight-gradient matrices and the Muon update built on it.

`own = False`: elementary torch operations in fp32.  `own = True`: the library's kernels through its public entry points."""
import math
import random

import torch

own = False

NS_COEFFS = (3.4445, -4.7750, 2.0315)        # quintic Newton-Schulz step X <- a X + b (X X^T) X + c (X X^T)^2 X
NS_STEPS = 5
NS_EPS = 1e-7
GN_EPS = 1e-5
LR, MOMENTUM, DECAY = 0.02, 0.95, 1e-4
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the projected 15 x 20 level of ONE 640 x 480 frame: single-image inference, where the call's latency counts
        dict(name="gn_fwd_frame", op="gn_fwd", N=1, HW=300, C=256, G=32, dtype="f32", act="relu", sliced=False),
        # the 60 x 80 level of a training batch of 16, read out of the token buffer that holds all four levels
        dict(name="gn_fwd_level", op="gn_fwd", N=16, HW=4800, C=256, G=32, dtype="bf16", act="silu", sliced=True),
        # the 120 x 160 level of eight 1280 x 960 frames
        dict(name="gn_fwd_hires", op="gn_fwd", N=8, HW=19200, C=256, G=32, dtype="f16", act="gelu", sliced=False),
        # a narrow head on an odd crop: 11 x 11 tokens, 12 channels per group
        dict(name="gn_train_crop", op="gn_train", N=3, HW=121, C=96, G=8, dtype="f32", act="silu", sliced=False),
        # one training step's normalisation of the 60 x 80 level at batch 16
        dict(name="gn_train_level", op="gn_train", N=16, HW=4800, C=256, G=32, dtype="bf16", act="silu", sliced=False),
        # ... and of the 120 x 160 level of eight 1280 x 960 frames, kept in fp32 up to the normalisation
        dict(name="gn_train_hires", op="gn_train", N=8, HW=19200, C=256, G=32, dtype="f32", act="gelu", sliced=False),
        # the last Linear of a class-specific translation head (22 classes x 3)
        dict(name="orth_head", op="orth", shapes="1x66x256", dtype="f32"),
        # the first FFN Linears of ten transformer layers, one stacked call
        dict(name="orth_ffn", op="orth", shapes="10x1024x256", dtype="bf16"),
        # a generic large square matrix
        dict(name="orth_square", op="orth", shapes="1x2048x2048", dtype="f32"),
        # one odd matrix: no dimension a multiple of anything
        dict(name="muon_odd", op="muon", shapes="1x257x131", dtype="f32"),
        # every matrix of the five encoder layers: sampling offsets, the three 256 x 256 projections, the two FFN Linears
        dict(name="muon_encoder", op="muon", shapes="5x512x256+15x256x256+5x1024x256+5x256x1024", dtype="f32"),
        # four generic wide FFN weights
        dict(name="muon_wide", op="muon", shapes="4x4096x1024", dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["gn_fwd", "gn_train", "orth", "muon"])
    if op in ("gn_fwd", "gn_train"):
        while True:
            N, HW, G = _log(rng, 1, 16), _log(rng, 8, 19200), rng.choice([1, 2, 4, 8, 16, 32])
            C = G * rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 32])
            if 16 <= C <= 512 and N * HW * C <= 16 * 4800 * 256 and HW * (C // G) >= 16:
                # (a ReLU's gradient jumps at 0, where two right roundings of z may fall on either side: the drawn training passes are smooth)
                acts = ["none", "gelu", "silu"] + (["relu"] if op == "gn_fwd" else [])
                return dict(op=op, N=N, HW=HW, C=C, G=G, dtype=rng.choice(["f32", "bf16", "f16"]), act=rng.choice(acts), sliced=rng.random() < 0.4)
    while True:
        m, n, k = _log(rng, 2, 2048), _log(rng, 2, 2048), _log(rng, 1, 16)
        if k * min(m, n) ** 2 * max(m, n) <= 4 * 1024 * 1024 * 1024:
            return dict(op=op, shapes=f"{k}x{m}x{n}", dtype="f32" if op == "muon" else rng.choice(["f32", "bf16", "f16"]))


def _stacks(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split("+")]


def _gradient(g, k, m, n, scale):
    """k weight-gradient-like matrices: sums of 2 min(m, n) + 8 outer products of decaying weight."""
    r = 2 * min(m, n) + 8
    w = (1.0 + torch.arange(r, device="cuda", dtype=torch.float32)).pow(-0.25)
    a = torch.randn(k, m, r, generator=g, device="cuda") * w
    b = torch.randn(k, r, n, generator=g, device="cuda")
    return torch.matmul(a, b) * (scale / math.sqrt(r))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")    # noqa: E731
    if case["op"] in ("gn_fwd", "gn_train"):
        N, HW, C = case["N"], case["HW"], case["C"]
        train = case["op"] == "gn_train"
        S = HW + HW // 3 + 1 if case["sliced"] else HW
        # conv outputs: channels with means and spreads of their own
        x = (rnd(N, S, C) * (0.5 + rnd(C).abs()) + 0.5 * rnd(C)).to(dt)
        x = x[:, S - HW:]
        w, b = 1.0 + 0.2 * rnd(C), 0.2 * rnd(C)
        st = dict(op=case["op"], x=x, w=w, b=b, G=case["G"], act=case["act"])
        if train:
            st["dy"] = (rnd(N, HW, C) * 0.01).to(dt)
            for t in (x, w, b):
                t.requires_grad_(True)
        return st
    stacks = _stacks(case)
    if case["op"] == "orth":
        (k, m, n), = stacks
        return dict(op="orth", g=_gradient(g, k, m, n, 1e-3).to(dt))
    p = [rnd(k, m, n) / math.sqrt(n) for k, m, n in stacks]
    gr = [_gradient(g, k, m, n, 1e-3) for k, m, n in stacks]
    mo = [0.3 * t.roll(1, -1) + 0.5 * t for t in gr]
    lists = [[t[i] for t in s for i in range(t.shape[0])] for s in (p, gr, mo)]
    return dict(op="muon", p=p, g=gr, m=mo, lists=lists)


# ---- plain forms ------------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_gn(st):
    x, w, b, G = (st["x"].detach().float(), st["w"].detach(), st["b"].detach(), st["G"])
    N, HW, C = x.shape
    xg = x.reshape(N, HW, G, C // G)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    d = xg - mean
    rstd = (d.square().mean(dim=(1, 3), keepdim=True) + GN_EPS).rsqrt()
    xhat = (d * rstd).reshape(N, HW, C)
    z = xhat * w + b
    y = _act(z, st["act"]).to(st["x"].dtype)
    if "dy" not in st:
        return y
    dz = st["dy"].float() * _act_grad(z, st["act"])
    db = dz.sum(dim=(0, 1))
    dw = (dz * xhat).sum(dim=(0, 1))
    dh = (dz * w).reshape(N, HW, G, C // G)
    hg = xhat.reshape(N, HW, G, C // G)
    dx = rstd * (dh - dh.mean(dim=(1, 3), keepdim=True) - hg * (dh * hg).mean(dim=(1, 3), keepdim=True))
    return y, dx.reshape(N, HW, C).to(st["x"].dtype), dw, db


def _plain_ns(G):
    """G (k, m, n) fp32 -> the orthogonalised stack."""
    X = G.mT if G.shape[-2] > G.shape[-1] else G
    X = X / (X.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NS_EPS)
    a, b, c = NS_COEFFS
    for _ in range(NS_STEPS):
        A = torch.matmul(X, X.mT)
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    return X.mT if G.shape[-2] > G.shape[-1] else X


def _plain_muon(p, g, m):
    m.mul_(MOMENTUM).add_(g, alpha=1.0 - MOMENTUM)
    u = MOMENTUM * m + (1.0 - MOMENTUM) * g
    s = math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
    p.mul_(1.0 - LR * DECAY).add_(_plain_ns(u), alpha=-LR * s)


def run(state):
    op = state["op"]
    if not own:
        if op in ("gn_fwd", "gn_train"):
            return _plain_gn(state)
        if op == "orth":
            return _plain_ns(state["g"].float()).to(state["g"].dtype).contiguous()
        with torch.no_grad():
            [_plain_muon(p, g, m) for p, g, m in zip(state["p"], state["g"], state["m"])]
        return state["p"], state["m"]
    from poet_amd import functional, ops
    if op == "gn_fwd":
        return functional.group_norm_act(state["x"], state["w"], state["b"], state["G"], act=state["act"], eps=GN_EPS)
    if op == "gn_train":
        y = functional.group_norm_act(state["x"], state["w"], state["b"], state["G"], act=state["act"], eps=GN_EPS)
        return (y.detach(), *torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["dy"]))
    if op == "orth":
        return ops.orthogonalize(state["g"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
    params, grads, moments = state["lists"]
    ops.muon_step(params, grads, moments, lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
    return state["p"], state["m"]


def work(case):
    if case["op"] in ("gn_fwd", "gn_train"):
        n, esz = case["N"] * case["HW"] * case["C"], 4 if case["dtype"] == "f32" else 2
        if case["op"] == "gn_fwd":                # x in, y out
            return dict(bytes=2 * n * esz + 8 * case["C"], flops=12 * n)
        return dict(bytes=4 * n * esz + 16 * case["C"], flops=36 * n)        # x, dy in, y, dx out
    nbytes = flops = 0
    for k, m, n in _stacks(case):
        d, r = min(m, n), max(m, n)
        # X X^T and its square are symmetric: half of their products are free
        flops += k * NS_STEPS * (d * d * r + d * d * d + 2 * d * d * r)
        nbytes += k * m * n * ((8 if case["dtype"] == "f32" else 4) if case["op"] == "orth" else 20)
    return dict(bytes=nbytes, flops=flops)


# ---- the definitions in 64 bits -----------------------------------------------------------------------
def _exact_ns(G):
    """Newton-Schulz in float64, from the right: X <- X (a I + b K + c K^2), K = X^T X (the same polynomial of the singular values)."""
    X = G / (torch.linalg.vector_norm(G, dim=(-2, -1), keepdim=True) + NS_EPS)
    a, b, c = NS_COEFFS
    eye = torch.eye(X.shape[-1], dtype=torch.float64, device=X.device)
    for _ in range(NS_STEPS):
        K = X.mT @ X
        X = X @ (a * eye + K @ (b * eye + c * K))
    return X


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("gn_fwd", "gn_train"):
        x, w, b = (st[k].detach().double().requires_grad_(True) for k in ("x", "w", "b"))
        z = x.transpose(1, 2).reshape(x.shape[0], st["G"], -1)
        var, mean = torch.var_mean(z, dim=-1, correction=0, keepdim=True)
        z = ((z - mean) / torch.sqrt(var + GN_EPS)).reshape(x.shape[0], x.shape[2], x.shape[1])
        z = (z * w[:, None] + b[:, None]).transpose(1, 2)
        y = {"none": lambda t: t, "relu": lambda t: t.clamp(min=0), "silu": lambda t: t * torch.sigmoid(t),
             "gelu": lambda t: t * torch.special.ndtr(t)}[case["act"]](z)
        if case["op"] == "gn_fwd":
            return y.detach()
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), st["dy"].double()))
    if case["op"] == "orth":
        return _exact_ns(st["g"].double())
    ps, ms = [], []
    for p, g, m in zip(st["p"], st["g"], st["m"]):
        p, g, m = p.double(), g.double(), m.double()
        m = m + (1.0 - MOMENTUM) * (g - m)
        o = _exact_ns(g + MOMENTUM * (m - g))
        ps.append(p - LR * DECAY * p - LR * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5 * o)
        ms.append(m)
    return ps, ms
