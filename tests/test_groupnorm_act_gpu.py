"""GroupNorm + activation on channels-last rows against its definition in float64, forward and backward.

Tolerances (u = 2^-24, fp32's half step; s = sqrt(var + eps), R = |mean| / s, h = (x - mean) / s, z = gamma h + beta):
  * a group's mean is off by a few u (|mean| + s), so h is off by K u (1 + R)(1 + |h|) with K = 16 for the handful of roundings of
    x - mean, rstd and the per-lane / per-chunk combination (a lane sums at most 64 samples against its own first sample);
  * the activations are 1.13-Lipschitz at most and evaluated to a few u of max(|z|, 1); the result is rounded once: half a step of its type;
  * a gradient sum over a lane's <= 64 rows, then a tree, is off by 128 u of the sum of magnitudes (plus the error of h in each term,
    act'' <= 1)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ["none", "relu", "gelu", "silu"]


@pytest.fixture(scope="module")
def fn():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from poet_amd import functional
    return functional


@pytest.fixture(scope="module")
def ops(fn):
    from poet_amd import ops as _ops
    return _ops


def act64(z, act):
    return {"none": lambda t: t, "relu": lambda t: t.clamp(min=0), "silu": lambda t: t / (1 + torch.exp(-t)),
            "gelu": lambda t: 0.5 * t * torch.erfc(-t * math.sqrt(0.5))}[act](z)


def dact64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def ref(x, w, b, G, act, eps, dy=None):
    """Everything in float64 on the CPU, with the magnitudes the tolerances need."""
    x, w, b = x.detach().cpu().double(), w.detach().cpu().double(), b.detach().cpu().double()
    N, HW, C = x.shape
    g = x.view(N, HW, G, C // G)
    mean = g.mean((1, 3), keepdim=True)
    s = ((g - mean).square().mean((1, 3), keepdim=True) + eps).sqrt()
    h = ((g - mean) / s).reshape(N, HW, C)
    R = (mean.abs() / s).expand(N, HW, G, C // G).reshape(N, HW, C)
    rstd = (1 / s).expand(N, HW, G, C // G).reshape(N, HW, C)
    z = h * w + b
    y = act64(z, act)
    dh = 16 * U * (1 + R) * (1 + h.abs())
    out = dict(y=y, z=z, tol_y=1.13 * (dh * w.abs()) + 16 * U * (1 + z.abs() + b.abs()))
    if dy is not None:
        dy = dy.detach().cpu().double()
        avg = lambda t: t.reshape(N, HW, G, C // G).mean((1, 3), keepdim=True).expand(N, HW, G, C // G).reshape(N, HW, C)   # noqa: E731
        dz = dy * dact64(z, act)
        e_dz = dy.abs() * (dh * w.abs() + 16 * U * (1 + z.abs())) * (0 if act in ("none", "relu") else 1) + 4 * U * dz.abs()
        out["db"], out["dw"] = dz.sum((0, 1)), (dz * h).sum((0, 1))
        out["tol_db"] = (128 * U * dz.abs() + e_dz).sum((0, 1))
        out["tol_dw"] = (128 * U * (dz * h).abs() + e_dz * h.abs() + dz.abs() * dh).sum((0, 1))
        p = dz * w
        m1, m2 = avg(p), avg(p * h)
        out["dx"] = rstd * (p - m1 - h * m2)
        e_p = e_dz * w.abs() + 4 * U * p.abs()
        e1 = avg(128 * U * p.abs() + e_p)
        e2 = avg(128 * U * (p * h).abs() + e_p * h.abs() + p.abs() * dh)
        out["tol_dx"] = rstd * (e_p + e1 + h.abs() * e2 + dh * m2.abs()) + 32 * U * (1 + R) * rstd * (p.abs() + m1.abs() + (h * m2).abs())
    return out


def check(got, want, tol, what):
    got_, eps = got.detach().cpu().double(), torch.finfo(got.dtype).eps
    tol = tol + (eps / 2) * (want.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    bad = (got_ - want).abs() - tol
    assert torch.isfinite(got_).all(), what
    assert bad.max().item() <= 0, f"{what}: off by {(got_ - want).abs().flatten()[bad.argmax()].item():.3e}, allowed {tol.flatten()[bad.argmax()].item():.3e}"


def make(N, HW, C, dtype, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)     # noqa: E731
    x = (r(N, HW, C) * (0.5 + r(C).abs()) + mean * r(C)).to(dtype)
    return x.cuda(), (1 + 0.3 * r(C)).cuda(), (0.3 * r(C)).cuda(), (0.1 * r(N, HW, C)).to(dtype).cuda()


def away_from_kink(x, w, b, G, act, dy, eps=1e-5):
    """A ReLU's gradient jumps at z = 0, where a rounding of z decides it: no gradient arrives within 1e-3 of it."""
    if act != "relu":
        return dy
    z = ref(x, w, b, G, act, eps)["z"].cuda()
    return torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)


def run_case(fn, x, w, b, G, act, dy, eps=1e-5, what=""):
    dy = away_from_kink(x, w, b, G, act, dy, eps)
    xg, wg, bg = x.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = fn.group_norm_act(xg, wg, bg, G, act=act, eps=eps)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)
    r = ref(x, w, b, G, act, eps, dy)
    check(y, r["y"], r["tol_y"], what + " y")
    check(dx, r["dx"], r["tol_dx"], what + " dx")
    check(dw, r["dw"], r["tol_dw"], what + " dgamma")
    check(db, r["db"], r["tol_db"], what + " dbeta")
    with torch.no_grad():
        assert torch.equal(fn.group_norm_act(x, w, b, G, act=act, eps=eps), y)


SHAPES = [(1, 1, 8, 1), (1, 1, 32, 4), (2, 7, 96, 8), (3, 121, 96, 8), (1, 300, 256, 32), (2, 1000, 66, 33), (1, 50, 2100, 1), (2, 33, 4096, 2),
          (1, 9, 3, 3), (1, 40, 5000, 1250), (5, 17, 40, 5), (1, 2047, 24, 2), (2, 513, 320, 32), (1, 3, 260, 1), (16, 80, 256, 32), (3, 1201, 256, 32)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("N,HW,C,G", SHAPES)
def test_shapes(fn, N, HW, C, G, dtype):
    act = ACTS[(N + HW + C) % 4]
    x, w, b, dy = make(N, HW, C, DTYPES[dtype], seed=HW + C)
    run_case(fn, x, w, b, G, act, dy, what=f"{(N, HW, C, G)} {act} {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("act", ACTS)
def test_activations(fn, act, dtype):
    x, w, b, dy = make(2, 260, 64, DTYPES[dtype], seed=3)
    w = w * 3                                             # z out to the tails
    run_case(fn, x, w, b, 8, act, dy, what=f"{act} {dtype}")


@pytest.mark.parametrize("G", [1, 32, 256])
def test_many_rows(fn, G):
    x, w, b, dy = make(2, 19200, 256, torch.float32, seed=5)
    run_case(fn, x, w, b, G, "gelu", dy, what=f"many rows G={G}")


@pytest.mark.parametrize("kind", ["token slice", "interleaved images", "wide rows", "unaligned", "expanded dy"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(fn, kind, dtype):
    dt = DTYPES[dtype]
    N, HW, C, G = 3, 77, 64, 8
    x, w, b, dy = make(N, HW, C, dt, seed=9)
    if kind == "token slice":
        buf = torch.full((N, 200, C), 7.0, dtype=dt, device="cuda")
        buf[:, 30:30 + HW] = x
        x = buf[:, 30:30 + HW]
    elif kind == "interleaved images":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
        dy = dy.transpose(0, 1).contiguous().transpose(0, 1)
    elif kind == "wide rows":
        buf = torch.full((N, HW, 2 * C), 7.0, dtype=dt, device="cuda")
        buf[..., C:] = x
        x = buf[..., C:]
    elif kind == "unaligned":
        buf = torch.full((N * HW * C + 1,), 7.0, dtype=dt, device="cuda")
        buf[1:] = x.flatten()
        x = buf[1:].view(N, HW, C)
    else:
        dy = dy[:1, :1].expand(N, HW, C)
    run_case(fn, x, w, b, G, "silu", dy, what=f"{kind} {dtype}")


def test_output_views_leave_their_surroundings(ops):
    """y and dx as rows of a larger buffer: nothing else of the buffer changes; y may be x itself."""
    N, HW, C, G = 2, 85, 64, 8
    x, w, b, dy = make(N, HW, C, torch.float32, seed=11)
    r = ref(x, w, b, G, "relu", 1e-5)
    buf = torch.full((N, 200, C), 7.0, device="cuda")
    stats = torch.empty(N, G, 2, device="cuda")
    ops.groupnorm_act_fwd(x, w, b, buf[:, 40:40 + HW], G, "relu", stats=stats)
    check(buf[:, 40:40 + HW], r["y"], r["tol_y"], "y view")
    assert (buf[:, :40] == 7).all() and (buf[:, 40 + HW:] == 7).all()
    buf.fill_(7.0)
    dw, db = torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "relu", dx=buf[:, 3:3 + HW], dgamma=dw, dbeta=db)
    assert (buf[:, :3] == 7).all() and (buf[:, 3 + HW:] == 7).all()
    y = x.clone()
    ops.groupnorm_act_fwd(y, w, b, y, G, "relu")
    check(y, r["y"], r["tol_y"], "in place")


@pytest.mark.parametrize("xt,yt", [("bf16", "f32"), ("f32", "bf16")])
def test_mixed_types(ops, xt, yt):
    N, HW, C, G = 2, 150, 128, 16
    x, w, b, dy = make(N, HW, C, DTYPES[xt], seed=13)
    dy = dy.to(DTYPES[yt])
    y, dx, stats = torch.empty(N, HW, C, dtype=DTYPES[yt], device="cuda"), torch.empty_like(x), torch.empty(N, G, 2, device="cuda")
    dw, db = torch.full((C,), 2.0, device="cuda"), torch.full((C,), -1.0, device="cuda")
    ops.groupnorm_act_fwd(x, w, b, y, G, "gelu", stats=stats)
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "gelu", dx=dx, dgamma=dw, dbeta=db, accumulate=True)
    r = ref(x, w, b, G, "gelu", 1e-5, dy)
    check(y, r["y"], r["tol_y"], "y")
    check(dx, r["dx"], r["tol_dx"], "dx")
    check(dw, r["dw"] + 2, r["tol_dw"], "dgamma, added")
    check(db, r["db"] - 1, r["tol_db"], "dbeta, added")
    # parts of the gradient alone, the same bits
    dx2, dw2, db2 = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "gelu", dx=dx2)
    assert torch.equal(dx, dx2)
    dw.fill_(2.0)
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "gelu", dgamma=dw2, dbeta=db2)
    check(dw2, r["dw"], r["tol_dw"], "dgamma alone")


def test_offsets_and_outliers(fn):
    """Means a thousand spreads away, an outlier as the first sample, constant groups."""
    x, w, b, dy = make(2, 300, 64, torch.float32, seed=17)
    run_case(fn, x + 1000.0, w, b, 8, "silu", dy, what="far mean")
    x2 = x.clone()
    x2[0, 0] = 3e4
    run_case(fn, x2, w, b, 8, "silu", dy, what="outlier in the first row")
    x3 = x.clone()
    x3[1, :, :8] = 2.5
    y = fn.group_norm_act(x3, w, b, 8, act="none")
    assert torch.equal(y[1, :, :8], b[:8].expand(300, 8))                       # zero variance: exactly beta


def test_non_finite_values_stay_in_their_group(fn):
    x, w, b, _ = make(2, 90, 64, torch.float32, seed=19)
    clean = fn.group_norm_act(x, w, b, 8, act="relu")
    for v in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[1, 44, 17] = v                                                    # group 2 of image 1
        y = fn.group_norm_act(x2, w, b, 8, act="relu")
        assert torch.isnan(y[1, :, 16:24]).all()
        keep = torch.ones(2, 1, 64, dtype=torch.bool, device="cuda").expand(2, 90, 64).clone()
        keep[1, :, 16:24] = False
        assert torch.equal(y[keep], clean[keep])


def test_gradient_against_differences(fn):
    """Directional derivatives of sum(y c) by central differences of the float64 definition: truncation h^2 ~ 1e-8 of the values."""
    x, w, b, c = make(2, 30, 24, torch.float32, seed=23)
    xg, wg, bg = (t.clone().requires_grad_(True) for t in (x, w, b))
    g = torch.autograd.grad(fn.group_norm_act(xg, wg, bg, 4, act="gelu"), (xg, wg, bg), c)
    gen = torch.Generator().manual_seed(1)
    base = [t.cpu().double() for t in (x, w, b)]
    c64, step = c.cpu().double(), 1e-4

    def f(p):
        N, HW, C = p[0].shape
        q = p[0].view(N, HW, 4, C // 4)
        m = q.mean((1, 3), keepdim=True)
        q = ((q - m) / ((q - m).square().mean((1, 3), keepdim=True) + 1e-5).sqrt()).reshape(N, HW, C)
        return (act64(q * p[1] + p[2], "gelu") * c64).sum()

    for i in range(3):
        v = torch.randn(base[i].shape, generator=gen).double()
        hi, lo = [t.clone() for t in base], [t.clone() for t in base]
        hi[i] += step * v
        lo[i] -= step * v
        d = ((f(hi) - f(lo)) / (2 * step)).item()
        got = (g[i].cpu().double() * v).sum().item()
        scale = (g[i].cpu().double() * v).abs().sum().item()
        assert abs(got - d) <= 1e-5 * scale, (i, got, d)


def test_streams_graph_and_repeatability(fn):
    """Bit-identical when repeated, on another stream, and over replays of a captured graph with eager work between."""
    x, w, b, dy = make(4, 1200, 256, torch.bfloat16, seed=29)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))

    def step():
        y = fn.group_norm_act(x, w, b, 32, act="silu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(want, side))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        with torch.no_grad():
            for o in out:
                o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out)), k
        assert all(torch.equal(p, q) for p, q in zip(want, step()))


def test_shapes_of_the_module(fn):
    from poet_amd import GroupNormAct
    m = GroupNormAct(8, 64, act="silu").cuda()
    ref_m = torch.nn.GroupNorm(8, 64)
    assert list(m.state_dict()) == list(ref_m.state_dict())
    img = torch.randn(2, 64, 9, 11, device="cuda")
    want = ref(img.permute(0, 2, 3, 1).reshape(2, 99, 64), m.weight, m.bias, 8, "silu", 1e-5)
    for x in (img.permute(0, 2, 3, 1), img.to(memory_format=torch.channels_last).permute(0, 2, 3, 1)):
        y = m(x)
        assert y.shape == (2, 9, 11, 64)
        check(y.reshape(2, 99, 64), want["y"], want["tol_y"], "module")
    v = m(torch.randn(5, 64, device="cuda"))
    assert v.shape == (5, 64)
    assert m(torch.empty(0, 9, 64, device="cuda")).shape == (0, 9, 64)
    e = torch.empty(2, 0, 64, device="cuda", requires_grad=True)
    m(e).sum().backward()
    assert e.grad.shape == (2, 0, 64) and (m.weight.grad == 0).all()


def test_refusals(fn, ops):
    x, w, b, dy = make(2, 10, 64, torch.float32)
    for call, err in [(lambda: fn.group_norm_act(x, w, b, 7), ValueError),
                      (lambda: fn.group_norm_act(x, w, b, 8, act="tanh"), ValueError),
                      (lambda: fn.group_norm_act(x, w.half(), b, 8), ValueError),
                      (lambda: fn.group_norm_act(x, w[:32], b, 8), ValueError),
                      (lambda: fn.group_norm_act(x.double(), w, b, 8), TypeError),
                      (lambda: fn.group_norm_act(x[0, 0], w, b, 8), ValueError),
                      (lambda: fn.group_norm_act(x.cpu(), w, b, 8), Exception),
                      (lambda: ops.groupnorm_act_fwd(x.half(), w, b, torch.empty_like(x), 8), Exception),
                      (lambda: ops.groupnorm_act_fwd(x, w, b, torch.empty(10, 64, device="cuda").expand(2, 10, 64), 8), ValueError),
                      (lambda: ops.groupnorm_act_bwd(dy, x, torch.empty(2, 8, device="cuda"), w, b, 8, dx=x.clone()), ValueError)]:
        with pytest.raises(err):
            call()
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fn.group_norm_act(xg, w, b, 8, act="silu").sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):                       # differentiable once
        g.sum().backward()


def test_more_than_the_cache_holds(ops):
    """Over 200 MB the second pass runs from the last row to the first: the same results, image by image against float64 on the GPU."""
    N, HW, C, G = 3, 70001, 256, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(N, HW, C, generator=g, device="cuda") + 1.5
    dy = torch.randn(N, HW, C, generator=g, device="cuda") * 0.1
    w, b = torch.rand(C, generator=g, device="cuda") + 0.5, torch.randn(C, generator=g, device="cuda") * 0.1
    y, dx, st, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty(N, G, 2, device="cuda"), torch.empty_like(w), torch.empty_like(b)
    ops.groupnorm_act_fwd(x, w, b, y, G, "silu", stats=st)
    ops.groupnorm_act_bwd(dy, x, st, w, b, G, "silu", dx=dx, dgamma=dw, dbeta=db)
    sw, sb = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
    for n in range(N):
        q = x[n].double().view(HW, G, C // G)
        m = q.mean((0, 2), keepdim=True)
        s = ((q - m).square().mean((0, 2), keepdim=True) + 1e-5).sqrt()
        h = ((q - m) / s).view(HW, C)
        z = h * w.double() + b.double()
        sig = torch.sigmoid(z)
        # (K u per element as above: K = 16 for y; the group's two means sum 560 008 terms, lanes of <= 64 rows and then trees)
        assert (y[n].double() - z * sig).norm() <= 16 * U * (z * sig).norm()
        dz = dy[n].double() * sig * (1 + z * (1 - sig))
        p = (dz * w.double()).view(HW, G, C // G)
        hg = h.view(HW, G, C // G)
        want = ((p - p.mean((0, 2), keepdim=True) - hg * (p * hg).mean((0, 2), keepdim=True)) / s).view(HW, C)
        assert (dx[n].double() - want).norm() <= 32 * U * want.norm()
        sw += (dz * h).sum(0)
        sb += dz.sum(0)
    assert (dw.double() - sw).norm() <= 128 * U * HW ** 0.5 * sw.norm() and (db.double() - sb).norm() <= 128 * U * HW ** 0.5 * sb.norm()


@pytest.mark.parametrize("N,HW,C,G", [(1, 30, 64, 8), (2, 5000, 64, 2)])
def test_in_place(ops, N, HW, C, G):
    """y on x; dx on x or on dy: the bits of the call with its own outputs, on both the one-launch and the chunked path."""
    x, w, b, dy = make(N, HW, C, torch.float32)
    y, stats = torch.empty_like(x), torch.empty(N, G, 2, device="cuda")
    ops.groupnorm_act_fwd(x, w, b, y, G, "silu", stats)
    dx, (dw, db) = torch.empty_like(x), torch.empty(2, C, device="cuda")
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "silu", dx, dw, db)
    for own in (lambda: (x.clone(), dy.clone(), 0), lambda: (x.clone(), dy.clone(), 1)):
        xc, dyc, which = own()
        dw2, db2 = torch.empty(2, C, device="cuda")
        ops.groupnorm_act_bwd(dyc, xc, stats, w, b, G, "silu", (xc, dyc)[which], dw2, db2)
        assert torch.equal((xc, dyc)[which], dx) and torch.equal(dw2, dw) and torch.equal(db2, db)
    xc = x.clone()
    assert torch.equal(ops.groupnorm_act_fwd(xc, w, b, xc, G, "silu"), y)
    big = torch.zeros(N, HW + 1, C, device="cuda")
    big[:, :HW] = x
    keep = big.clone()
    with pytest.raises(ValueError):
        ops.groupnorm_act_fwd(big[:, :HW], w, b, big[:, 1:], G, "silu")
    with pytest.raises(ValueError):
        ops.groupnorm_act_bwd(dy, big[:, :HW], stats, w, b, G, "silu", big[:, 1:])
    with pytest.raises(ValueError):
        ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "silu", None, dw, dw)
    assert torch.equal(big, keep)


def test_more_images_than_one_launch_of_groups_holds(fn):
    """2^17 images of 32 groups: past what the one-launch path may start, the chunked one takes over."""
    x, w, b, dy = make(4, 1, 64, torch.float32)
    n = (1 << 17) + 4
    big = x.repeat(n // 4, 1, 1)
    got = fn.group_norm_act(big, w, b, 32, act="gelu")
    r = ref(x, w, b, 32, "gelu", 1e-5)
    check(got[-4:], r["y"], r["tol_y"], "last images")
    assert torch.equal(got.view(-1, 4, 1, 64), got[:4].expand(n // 4, 4, 1, 64))
