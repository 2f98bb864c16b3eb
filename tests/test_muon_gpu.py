"""Newton-Schulz orthogonalisation and the Muon update against their definition in float64.

Tolerance.  A step X' = a X + b X X^T X + c (X X^T)^2 X uses X 1, 3 and 5 times; with every product off by a relative g (two operand
roundings of 2^-22 each, and fp32 sums of K terms: 4 sqrt(K) 2^-24) it adds at most g (|a| + 3 |b| s^2 + 5 |c| s^4) |X|_F, s = |X|_2, and carries an
earlier error on by at most D = max(|p'|, |p(x) / x|) on [0, s].  The bound is summed over the float64 iterates; an output of fewer bits
adds half a step of its type per element."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFS = (3.4445, -4.7750, 2.0315)
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from poet_amd import ops as _ops
    return _ops


def exact(u, steps=5, coeffs=COEFFS, eps=1e-7):
    """(result, bound on the Frobenius norm of its error)."""
    u = u.detach().cpu().double()
    turned = u.shape[0] > u.shape[1]
    X = u.t() if turned else u
    X = X / (X.norm() + eps)
    cs = coeffs if hasattr(coeffs[0], "__len__") else [coeffs] * steps
    err = 2.0 ** -21 * X.norm().item()
    for a, b, c in cs:
        K = max(X.shape)
        g = 2 * 2.0 ** -22 + 4 * math.sqrt(K) * 2.0 ** -24
        s = torch.linalg.matrix_norm(X, 2).item()
        x = torch.linspace(0, s, 500, dtype=torch.float64)
        D = max((a + 3 * b * x ** 2 + 5 * c * x ** 4).abs().max().item(), (a + b * x ** 2 + c * x ** 4).abs().max().item())
        err = D * err + g * (abs(a) + 3 * abs(b) * s ** 2 + 5 * abs(c) * s ** 4) * X.norm().item()
        A = X @ X.t()
        X = a * X + (b * A + c * (A @ A)) @ X
    return (X.t() if turned else X), err


def check(got, u, what, **kw):
    want, err = exact(u, **kw)
    g = got.detach().cpu().double()
    assert torch.isfinite(g).all(), what
    tol = err + torch.finfo(got.dtype).eps / 2 * want.norm().item() + (2.0 ** -25 * math.sqrt(want.numel()) if got.dtype == torch.float16 else 0)
    off = (g - want).norm().item()
    assert off <= tol, f"{what}: off by {off:.3e} of {want.norm().item():.3e}, allowed {tol:.3e}"
    return off / max(want.norm().item(), 1e-30)


def matrix(m, n, seed=0, kind="gauss"):
    g = torch.Generator().manual_seed(seed)
    if kind == "gauss":
        return torch.randn(m, n, generator=g)
    d = min(m, n)
    i = torch.arange(d, dtype=torch.float32)
    s = {"power": 1 / (1 + i), "wide": 10.0 ** (-7 * i / d), "lowrank": (i < max(1, d // 8)).float()}[kind]
    U = torch.linalg.qr(torch.randn(m, d, generator=g))[0]
    V = torch.linalg.qr(torch.randn(n, d, generator=g))[0]
    return (U * s) @ V.t()


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 256), (66, 256), (64, 64), (65, 63), (128, 129), (257, 131), (256, 1024), (1024, 256), (200, 2000), (513, 513),
          (31, 4097), (1100, 1300), (2048, 1024)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(ops, m, n, dtype):
    g = matrix(m, n, seed=m + n).to(DT[dtype]).cuda() * 1e-3
    keep = g.clone()
    check(ops.orthogonalize(g), g, f"{(m, n)} {dtype}")
    assert torch.equal(g, keep)


@pytest.mark.parametrize("kind", ["power", "wide", "lowrank"])
@pytest.mark.parametrize("m,n", [(96, 96), (256, 640), (1000, 160)])
def test_spectra(ops, m, n, kind):
    g = matrix(m, n, seed=3, kind=kind).cuda()
    check(ops.orthogonalize(g), g, f"{kind} {(m, n)}")


def test_result_is_nearly_orthogonal(ops):
    """Singular values of a well-conditioned matrix end inside the fixed band of the quintic."""
    o = ops.orthogonalize(matrix(256, 1024, seed=1).cuda())
    s = torch.linalg.svdvals(o.cpu().double())
    assert 0.6 < s.min() and s.max() < 1.25


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_scale_of_the_input(ops, scale):
    g = (matrix(70, 130, seed=5).double() * scale).float().cuda()
    o = ops.orthogonalize(g, eps=0.0)
    check(o, g, f"scale {scale}", eps=0.0)


def test_zero_and_non_finite_matrices(ops):
    a, z, b, c = matrix(40, 90, 1).cuda(), torch.zeros(100, 30, device="cuda"), matrix(64, 64, 2).cuda(), matrix(130, 130, 4).cuda()
    alone = ops.orthogonalize([a])[0]
    b[3, 5], c[0, 0] = float("nan"), float("-inf")
    oa, oz, ob, oc = ops.orthogonalize([a, z, b, c])
    assert torch.equal(oa, alone) and (oz == 0).all() and torch.isnan(ob).all() and torch.isnan(oc).all()


def test_list_equals_single_calls(ops):
    """30 matrices (more than one launch of records) of mixed shapes: the bits of a call of their own, whatever tile the list takes."""
    shapes = [(1, 5), (256, 256), (300, 70), (66, 256), (5, 900)] * 6
    gs = [matrix(m, n, seed=i).cuda() for i, (m, n) in enumerate(shapes)]
    outs = ops.orthogonalize(gs)
    for g, o in zip(gs, outs):
        check(o, g, f"list {tuple(g.shape)}")
        assert torch.equal(o, ops.orthogonalize(g))
    assert all(torch.equal(p, q) for p, q in zip(outs, ops.orthogonalize(gs)))


@pytest.mark.parametrize("shape,count", [((200, 200), 3), ((200, 200), 10), ((200, 200), 14), ((200, 400), 8), ((70, 300), 60), ((300, 300), 4), ((1100, 1030), 2)])
def test_every_tile_choice_on_a_dirty_workspace(ops, shape, count):
    """Both kinds of product with either tile edge, at sizes that end inside a tile; what the padding of the planes held before the call
    (here NaN) does not reach a result, and the result is that of a call of its own."""
    gs = [matrix(*shape, seed=i).cuda() for i in range(count)]
    torch.full((1 << 27,), float("nan"), device="cuda")                       # freed at once: the workspaces below come out of it
    outs = ops.orthogonalize(gs)
    for g, o in zip(gs, outs):
        check(o, g, f"{shape} x {count}")
    for i in (0, count - 1):
        torch.full((1 << 27,), float("nan"), device="cuda")
        assert torch.equal(outs[i], ops.orthogonalize(gs[i]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_batches_views_and_out(ops, dtype):
    dt = DT[dtype]
    base = torch.stack([matrix(90, 200, seed=i) for i in range(6)]).to(dt).cuda()
    want = [ops.orthogonalize(base[i]) for i in range(6)]
    o = ops.orthogonalize(base.view(2, 3, 90, 200))
    assert o.shape == (2, 3, 90, 200) and all(torch.equal(o.view(6, 90, 200)[i], want[i]) for i in range(6))
    wide = torch.full((90, 512), 3.0, dtype=dt, device="cuda")
    wide[:, 100:300] = base[0]
    assert torch.equal(ops.orthogonalize(wide[:, 100:300]), want[0])                     # strided rows
    assert torch.equal(ops.orthogonalize(base[0].t().contiguous().t()), want[0])         # columns first: copied
    assert torch.equal(ops.orthogonalize(base[:, :, :].flip(0)[0]), want[5])
    dst = torch.full((90, 512), 3.0, dtype=dt, device="cuda")
    ops.orthogonalize(base[1], out=dst[:, 7:207])
    assert torch.equal(dst[:, 7:207], want[1]) and (dst[:, :7] == 3).all() and (dst[:, 207:] == 3).all()
    g = base[2].clone()
    assert ops.orthogonalize(g, out=g) is g and torch.equal(g, want[2])                  # in place
    e = ops.orthogonalize(base[:1].expand(3, 90, 200))
    assert all(torch.equal(e[i], want[0]) for i in range(3))
    assert ops.orthogonalize(base[:0]).shape == (0, 90, 200) and ops.orthogonalize([]) == []
    assert ops.orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)


def test_other_coefficients(ops):
    g = matrix(100, 140, seed=9).cuda()
    cubic = (1.5, -0.5, 0.0)
    check(ops.orthogonalize(g, steps=12, coeffs=cubic), g, "cubic", steps=12, coeffs=cubic)
    each = [(3.0, -3.2, 1.2), COEFFS, (2.0, -1.5, 0.5)]
    check(ops.orthogonalize(g, steps=3, coeffs=each), g, "per step", steps=3, coeffs=each)
    check(ops.orthogonalize(g, steps=1), g, "one step", steps=1)


def ref_step(p, g, m, lr, mu, nesterov, wd, scale, gs=1.0, eps=1e-7):
    """One update in float64: (p, m, bound on |p - computed|_F)."""
    p2, g2 = p.reshape(p.shape[0], -1), g.reshape(p.shape[0], -1) * gs
    m2 = mu * m.reshape(p2.shape) + (1 - mu) * g2
    u = mu * m2 + (1 - mu) * g2 if nesterov else m2
    o, err = exact(u, eps=eps)
    r, c = p2.shape
    s = max(1.0, r / c) ** 0.5 if scale == "spectral" else 0.2 * max(r, c) ** 0.5
    new = p2 * (1 - lr * wd) - lr * s * o
    # (the update direction itself carries two fp32 roundings: D <= 3.45 per step of a relative 2^-23)
    return new.reshape(p.shape), m2.reshape(p.shape), lr * s * (err + 3.45 ** 5 * 2.0 ** -22) + 3 * 2.0 ** -24 * p2.norm().item()


SETS = {"encoder": [(512, 256), (256, 256), (256, 256), (1024, 256), (256, 1024)], "heads": [(256, 256), (66, 256), (132, 256), (3, 256)],
        "conv": [(256, 64, 3, 3), (256, 512, 1, 1)], "many": [(40, 60)] * 27, "large": [(1500, 1100)]}


@pytest.mark.parametrize("nesterov,scale", [(True, "spectral"), (False, "rms")])
@pytest.mark.parametrize("which", list(SETS))
def test_muon_steps(ops, which, nesterov, scale):
    gen = torch.Generator().manual_seed(2)
    ps = [torch.randn(*s, generator=gen) * 0.05 for s in SETS[which]]
    dev = [p.clone().cuda() for p in ps]
    mom = [torch.zeros_like(p) for p in dev]
    hi = [torch.zeros_like(p, dtype=torch.bfloat16) for p in dev]
    lo = [torch.zeros_like(p, dtype=torch.bfloat16) for p in dev]
    ref = [(p.double(), torch.zeros_like(p).double(), 0.0) for p in ps]
    for _ in range(2):
        gs = [torch.randn(*s, generator=gen) * 1e-3 for s in SETS[which]]
        ops.muon_step(dev, [g.cuda() for g in gs], mom, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale, p_bf16=hi, p_bf16_lo=lo)
        new = []
        for (p, m, e), g in zip(ref, gs):
            p, m, e2 = ref_step(p, g.double(), m, 0.02, 0.9, nesterov, 0.1, scale)
            new.append((p, m, e + e2))
        ref = new
    for i, (p, m, e) in enumerate(ref):
        got = dev[i].cpu().double()
        assert (got - p).norm().item() <= e, (which, i, (got - p).norm().item(), e)
        assert ((mom[i].cpu().double() - m).abs() <= 6 * 2.0 ** -24 * (m.abs() + 1e-3)).all()
        assert torch.equal(hi[i], dev[i].to(torch.bfloat16)) and torch.equal(lo[i], (dev[i] - hi[i].float()).to(torch.bfloat16))


def test_muon_scales_clip_and_lr_words(ops):
    gen = torch.Generator().manual_seed(4)
    p0, g0 = torch.randn(80, 50, generator=gen) * 0.1, torch.randn(80, 50, generator=gen)
    sq = torch.zeros(1025, device="cuda")
    g = g0.cuda()
    ops.sqnorm(g.view(-1), sq)
    p, m = p0.cuda(), torch.zeros(80, 50, device="cuda")
    word = torch.tensor([-0.25], device="cuda")                                  # (its sign is the caller's)
    ops.muon_step([p], [g], [m], lr=0.02, lr_scale=[word], sqnorm_buf=sq, max_norm=0.1, grad_scale=0.5)
    total = g0.double().norm().item() * 0.5
    gs = 0.5 * min(1.0, 0.1 / (total + 1e-6))
    want, wm, e = ref_step(p0.double(), g0.double(), torch.zeros(80, 50).double(), 0.005, 0.95, True, 0.0, "spectral", gs=gs)
    assert (p.cpu().double() - want).norm().item() <= e
    assert ((m.cpu().double() - wm).abs() <= 16 * 2.0 ** -24 * wm.abs() + 1e-12).all()


def test_muon_leaves_its_neighbours(ops):
    """Matrices that lie side by side in one buffer, with gaps: nothing outside them changes."""
    buf = {k: torch.full((40000,), v, device="cuda") for k, v in (("p", 1.0), ("g", 1e-3), ("m", 0.0))}
    gen = torch.Generator(device="cuda").manual_seed(1)
    buf["g"] += 1e-3 * torch.randn(40000, generator=gen, device="cuda")
    spans = [(0, 33, 65), (2145 + 64, 130, 100), (20000 + 1, 64, 128)]
    lists = {k: [b[o:o + r * c].view(r, c) for o, r, c in spans] for k, b in buf.items()}
    ops.muon_step(lists["p"], lists["g"], lists["m"], lr=0.02)
    inside = torch.zeros(40000, dtype=torch.bool, device="cuda")
    for o, r, c in spans:
        inside[o:o + r * c] = True
    assert (buf["p"][~inside] == 1).all() and (buf["m"][~inside] == 0).all() and (buf["m"][inside] != 0).any()


def test_streams_and_graph(ops):
    """The same bits on another stream and over the replays of a captured step, with eager work between the replays; two captured
    graphs have workspaces of their own."""
    shapes = [(256, 256), (300, 1030), (66, 256)]
    g = [matrix(*s, seed=i).cuda() * 1e-2 for i, s in enumerate(shapes)]
    want = ops.orthogonalize(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, side))

    def fresh():
        return [matrix(*sh, seed=50 + i).cuda() for i, sh in enumerate(shapes)], [torch.zeros(*sh, device="cuda") for sh in shapes]

    pe, me = fresh()
    pg, mg = fresh()
    graphs = []
    for k in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.muon_step(pg, g, mg, lr=0.01 * (k + 1), weight_decay=0.1)
        graphs.append(gr)
    for r in range(4):
        graphs[r % 2].replay()
        torch.cuda.synchronize()
        ops.muon_step(pe, g, me, lr=0.01 * (r % 2 + 1), weight_decay=0.1)
        assert all(torch.equal(a, b) for a, b in zip(pe + me, pg + mg)), r


def test_refusals(ops):
    g = matrix(8, 16).cuda()
    v = torch.zeros(16, device="cuda")
    p, m = g.clone(), torch.zeros_like(g)
    step = lambda **kw: ops.muon_step([p], [g], [m], **{"lr": 0.1, **kw})       # noqa: E731
    for call, err in [(lambda: ops.orthogonalize(v), ValueError), (lambda: ops.orthogonalize([v]), ValueError),
                      (lambda: ops.orthogonalize(g.double()), TypeError), (lambda: ops.orthogonalize(g.cpu()), Exception),
                      (lambda: ops.orthogonalize([g, g.half()]), ValueError), (lambda: ops.orthogonalize(g, steps=0), ValueError),
                      (lambda: ops.orthogonalize(g, steps=17), ValueError), (lambda: ops.orthogonalize(g, steps=3, coeffs=[(1, 0, 0)] * 2), ValueError),
                      (lambda: ops.orthogonalize(g, coeffs=(50.0, 0.0, 0.0)), Exception), (lambda: ops.orthogonalize(g, coeffs=(float("nan"), 0.0, 0.0)), Exception),
                      (lambda: ops.orthogonalize(g, out=torch.empty(16, 8, device="cuda")), ValueError),
                      (lambda: ops.orthogonalize(g, out=torch.empty(16, 8, device="cuda").t()), ValueError),
                      (lambda: ops.orthogonalize([g, g], out=[p, p]), ValueError), (lambda: step(scale="max"), ValueError),
                      (lambda: step(momentum=1.0), ValueError), (lambda: step(steps=0), ValueError), (lambda: step(p_bf16_lo=[p.bfloat16()]), ValueError),
                      (lambda: ops.muon_step([p, p], [g, g], [m, torch.zeros_like(m)], lr=0.1), ValueError),
                      (lambda: ops.muon_step([p], [g], [p], lr=0.1), ValueError), (lambda: ops.muon_step([p], [g.half()], [m], lr=0.1), ValueError),
                      (lambda: ops.muon_step([p.t()], [g.t()], [m.t()], lr=0.1), ValueError), (lambda: ops.muon_step([v], [v], [v.clone()], lr=0.1), ValueError),
                      (lambda: ops.muon_step([p], [g], [], lr=0.1), ValueError)]:
        with pytest.raises(err):
            call()
    assert torch.equal(p, g) and (m == 0).all()
    ops.muon_step([], [], [], lr=0.1)


def test_outputs_side_by_side_and_outputs_that_overlap(ops):
    """Views of one buffer as outputs: columns of the same rows, interleaved batches, and what would write an element twice or into another
    matrix's input, refused before anything runs."""
    buf = torch.zeros(40, 96, device="cuda")
    gs = [matrix(40, 32, i).cuda() for i in range(3)]
    ops.orthogonalize(gs, out=[buf[:, 32 * i:32 * (i + 1)] for i in range(3)])
    for i, g in enumerate(gs):
        assert torch.equal(buf[:, 32 * i:32 * (i + 1)], ops.orthogonalize(g))
    src = buf.clone()
    cols = [src[:, :32], src[:, 32:64], src[:, 64:]]
    want = [ops.orthogonalize(c) for c in cols]
    ops.orthogonalize(cols, out=cols)                                            # in place, on column views
    assert all(torch.equal(c, w) for c, w in zip(cols, want))
    g3 = torch.stack(gs)
    out3 = torch.zeros(40, 3, 32, device="cuda").transpose(0, 1)                 # the batch between rows and columns
    ops.orthogonalize(g3, out=out3)
    assert torch.equal(out3, ops.orthogonalize(g3))
    flat = torch.randn(5 * 40 * 32, device="cuda")
    a, b, c = flat[:1280].view(40, 32), flat[1280:2560].view(40, 32), flat[2000:3280].view(40, 32)
    keep = flat.clone()
    wide, half = torch.zeros(40, 32, device="cuda"), [g.bfloat16() for g in gs[:2]]
    for call in (lambda: ops.orthogonalize([a, gs[0]], out=[b, c]), lambda: ops.orthogonalize([a, b], out=[b, torch.empty_like(a)]),
                 lambda: ops.orthogonalize([a, b], out=[torch.empty_like(a), a]), lambda: ops.orthogonalize(torch.stack([a, b]), out=b.expand(2, 40, 32)),
                 lambda: ops.orthogonalize(half, out=[wide, half[1]]), lambda: ops.orthogonalize(half, out=[half[0], wide]),
                 lambda: ops.muon_step([a], [a], [torch.zeros_like(a)], lr=0.1), lambda: ops.muon_step([a], [b], [b], lr=0.1),
                 lambda: ops.muon_step([a, b], [gs[0], gs[1]], [torch.zeros_like(a), c], lr=0.1),
                 lambda: ops.muon_step([a], [b], [gs[0]], lr=0.1, p_bf16=[flat.view(torch.bfloat16)[100:1380]])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(flat, keep) and (wide == 0).all()
    ops.muon_step([a, b], [gs[0], gs[0]], [torch.zeros_like(a), torch.zeros_like(a)], lr=0.1)      # (one gradient for two matrices is fine)
    assert not torch.equal(flat, keep)


@pytest.mark.parametrize("shapes", [[(1100, 1030)] * 6, [(256, 256)] * 9 + [(900, 256)] * 4 + [(200, 410)] * 3 + [(700, 300), (260, 1500), (300, 300)], [(400, 2600), (2500, 500), (600, 600), (520, 300)]])
def test_mixed_lists_on_a_dirty_workspace(ops, shapes):
    """Large tiles in both products; lists of several lengths, which are not worked on in their order: still the bits of calls of their own."""
    gs = [matrix(m, n, seed=i).cuda() for i, (m, n) in enumerate(shapes)]
    torch.full((1 << 27,), float("nan"), device="cuda")
    outs = ops.orthogonalize(gs)
    again = ops.orthogonalize(gs[::-1])[::-1]
    for i, g in enumerate(gs):
        torch.full((1 << 27,), float("nan"), device="cuda")
        assert torch.equal(outs[i], ops.orthogonalize(g)) and torch.equal(outs[i], again[i]), shapes[i]
    small = min(range(len(shapes)), key=lambda i: shapes[i][0] * shapes[i][1])
    check(outs[small], gs[small], f"{shapes[small]}")
    check(outs[-1], gs[-1], f"{shapes[-1]}")


def test_muon_step_takes_images_and_odd_alignment_of_narrow_matrices(ops):
    """Whole vectors, single elements and bf16 images of narrow and ordinary matrices: the bits of the aligned update, and images = its rounding."""
    for shape in ((24, 132), (132, 24), (66, 256), (31, 57), (260, 280)):
        p, g, m = (matrix(*shape, seed=s).cuda() for s in range(3))
        n = p.numel()
        res = []
        for off in (0, 1):                                                       # (1: nothing is 16-byte aligned)
            bufs = [torch.zeros(n + 4, device="cuda")[off:off + n].view(shape) for _ in range(3)]
            imgs = [torch.zeros(n + 4, dtype=torch.bfloat16, device="cuda")[off:off + n].view(shape) for _ in range(2)]
            for b, t in zip(bufs, (p, g, m)):
                b.copy_(t)
            ops.muon_step([bufs[0]], [bufs[1]], [bufs[2]], lr=0.02, weight_decay=0.1, p_bf16=[imgs[0]], p_bf16_lo=[imgs[1]])
            hi = bufs[0].bfloat16()
            assert torch.equal(imgs[0], hi) and torch.equal(imgs[1], (bufs[0] - hi.float()).bfloat16())
            res.append(bufs)
        assert torch.equal(res[0][2], res[1][2])                                 # the momenta
        d = (res[0][0].double() - res[1][0].double()).norm() / res[0][0].double().norm()
        assert d <= 2.0 ** -22                                                   # (|u|_F summed in another order of 64-bit terms: one step of X_0's scale at most)


def test_long_lists_of_narrow_matrices(ops):
    """More narrow matrices than a launch takes by value: the bits of calls of their own, also in place and for the update."""
    shapes = [(20, 100), (7, 33), (90, 64), (50, 60), (1, 1)] * 30
    gs = [matrix(m, n, seed=i).cuda() for i, (m, n) in enumerate(shapes)]
    outs = ops.orthogonalize(gs)
    for i, (g, o) in enumerate(zip(gs, outs)):
        if i < 5 or i >= 145:
            check(o, g, f"{shapes[i]}")
        assert torch.equal(o, ops.orthogonalize(g)), shapes[i]
    ps, ms = [matrix(m, n, seed=500 + i).cuda() for i, (m, n) in enumerate(shapes)], [torch.zeros_like(g) for g in gs]
    p1, m1 = [p.clone() for p in ps], [m.clone() for m in ms]
    ops.muon_step(ps, gs, ms, lr=0.1)
    for i in range(0, 150, 7):
        ops.muon_step([p1[i]], [gs[i]], [m1[i]], lr=0.1)
        assert torch.equal(ps[i], p1[i]) and torch.equal(ms[i], m1[i]), shapes[i]
    same = torch.stack([matrix(24, 40, seed=i) for i in range(70)]).cuda()
    want = ops.orthogonalize(same)
    assert torch.equal(want[69], ops.orthogonalize(same[69]))
    ops.orthogonalize(same, out=same)
    assert torch.equal(same, want)
