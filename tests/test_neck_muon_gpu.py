"""The operators as a training run uses them: input projection with an activation, a small neck trained by Muon, PoET trained with Muon
updates (eager and from captured graphs)."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

from tests.test_muon_gpu import exact  # noqa: E402


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from tests.product_runner import build_product
    return build_product


@pytest.mark.parametrize("act", ["relu", "silu"])
def test_input_projection_with_activation(gpu, act):
    """Two 1 x 1 levels and two chained 3 x 3 stride-2 levels: conv -> GroupNorm -> activation against torch in float64, all gradients."""
    from poet_amd import functional as Fn
    from poet_amd.ops import LevelGeom
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    N, d, cins, shapes = 2, 64, [48, 80, 80, 64], [(12, 17), (6, 9), (3, 5), (2, 3)]
    feats = [r(N, 48, 12, 17), r(N, 80, 6, 9)]
    names, params = [], []
    for l, c in enumerate(cins):
        k = 1 if l < 2 else 3
        for n, t in ((f"{l}.0.weight", r(d, c, k, k) / (c * k * k) ** 0.5), (f"{l}.0.bias", 0.1 * r(d)), (f"{l}.1.weight", 1 + 0.2 * r(d)), (f"{l}.1.bias", 0.2 * r(d))):
            names.append(n)
            params.append(t)
    geom = LevelGeom(shapes)
    dsrc = 0.1 * r(N, geom.S, d)
    ref = [p.double().requires_grad_(True) for p in params]
    P = dict(zip(names, ref))
    rows, prev = [], None
    for l in range(4):
        x = feats[l].double() if l < 2 else feats[1].double() if l == 2 else prev
        y = F.conv2d(x, P[f"{l}.0.weight"], P[f"{l}.0.bias"], stride=1 if l < 2 else 2, padding=0 if l < 2 else 1)
        prev = {"relu": F.relu, "silu": F.silu}[act](F.group_norm(y, 32, P[f"{l}.1.weight"], P[f"{l}.1.bias"]))
        rows.append(prev.flatten(2).transpose(1, 2))
    want = torch.cat(rows, 1)
    if act == "relu":                                   # (its gradient jumps at 0, where a rounding decides it)
        dsrc[want.detach().abs() < 1e-4] = 0
    wg = torch.autograd.grad(want, ref, dsrc.double())
    dev = [p.cuda().requires_grad_(True) for p in params]
    src = Fn.InputProjFn.apply([f.cuda() for f in feats], geom, 32, (torch.float32, torch.float32, False, act), tuple(names), *dev)
    assert (src.detach().cpu().double() - want.detach()).abs().max() < 1e-4
    got = torch.autograd.grad(src, dev, dsrc.cuda())
    for n, a, b in zip(names, got, wg):
        assert (a.cpu().double() - b).norm() <= 2e-4 * b.norm() + 1e-6, (n, float((a.cpu().double() - b).norm() / b.norm()))


def test_neck_trained_by_muon(gpu):
    """Linear -> GroupNorm + SiLU -> Linear, three steps of gradient, momentum and orthogonalised update, against the same run in float64.
    A gradient of relative Frobenius error 1e-5 (fp32 products and the statistics) is amplified at most 3.45 per Newton-Schulz step."""
    from poet_amd import functional as Fn, ops
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    x, t = r(3, 150, 96), r(3, 150, 40)
    W1, b1, gw, gb, W2, b2 = r(128, 96) / 10, 0.1 * r(128), 1 + 0.1 * r(128), 0.1 * r(128), r(40, 128) / 11, 0.1 * r(40)
    lr, mu = 0.02, 0.9
    dev = [p.clone().cuda().requires_grad_(True) for p in (W1, b1, gw, gb, W2, b2)]
    ref = [p.double().requires_grad_(True) for p in (W1, b1, gw, gb, W2, b2)]
    xd, td = x.cuda(), t.cuda()
    mats, rest = (0, 4), (1, 2, 3, 5)
    mom = [torch.zeros_like(dev[i]) for i in mats]
    rmom = [torch.zeros_like(ref[i]) for i in mats]
    bound = [0.0, 0.0]
    for step in range(3):
        y = Fn.LinearFn.apply(Fn.group_norm_act(Fn.LinearFn.apply(xd, dev[0], dev[1]), dev[2], dev[3], 16, act="silu"), dev[4], dev[5])
        grads = torch.autograd.grad(((y - td) ** 2).mean(), dev)
        h = F.linear(x.double(), ref[0], ref[1]).transpose(1, 2)
        ry = F.linear(F.silu(F.group_norm(h, 16, ref[2], ref[3])).transpose(1, 2), ref[4], ref[5])
        rgrads = torch.autograd.grad(((ry - t.double()) ** 2).mean(), ref)
        for a, b in zip(grads, rgrads):
            assert (a.cpu().double() - b).norm() <= (1e-5 + 0.05 * step) * b.norm()
        with torch.no_grad():
            ops.muon_step([dev[i] for i in mats], [grads[i] for i in mats], mom, lr=lr, momentum=mu)
            for i in rest:
                dev[i] -= 0.05 * grads[i]
                ref[i] -= 0.05 * rgrads[i]
            for k, i in enumerate(mats):
                rmom[k] = mu * rmom[k] + (1 - mu) * rgrads[i]
                o, err = exact(mu * rmom[k] + (1 - mu) * rgrads[i])
                s = max(1.0, ref[i].shape[0] / ref[i].shape[1]) ** 0.5
                ref[i] -= lr * s * o
                if step == 0:
                    off = (dev[i].cpu().double() - ref[i]).norm().item()
                    assert off <= lr * s * (err + 3.45 ** 5 * 1e-5) + 1e-6, (i, off)
    # later steps start from weights that differ by the above: the runs stay together to a percent of an update
    for i in mats:
        assert (dev[i].cpu().double() - ref[i]).norm() <= 0.01 * 3 * lr * ref[i].shape[0] ** 0.5


def _params(model):
    return {n: p.detach().clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_trainer_with_muon(gpu, precision):
    """One step of PoET: every matrix of the arena's list moves by the Muon formula from its own gradient, every other parameter exactly as
    AdamW moves it without Muon; images follow; the momentum is the state."""
    import poet_amd
    r = gpu("tiny", 2, True, precision, dropout=0.0)
    q = gpu("tiny", 2, True, precision, dropout=0.0)
    ta = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.1, distributed=False, muon=dict(momentum=0.9))
    tb = poet_amd.Trainer(q["model"], q["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.1, distributed=False)
    A, B = ta.arena, tb.arena
    before = _params(r["model"])
    names = set(A.muon_names)
    assert any("in_proj_weight" in n for n in names) and any("input_proj" in n for n in names) and any("linear1" in n for n in names)
    assert not any("level_embed" in n or "layers.2.weight" in n and "head" in n for n in names) and all("bias" not in n for n in names)
    for t, m in ((ta, r), (tb, q)):
        m["model"].train()
        t.step(m["samples"], m["targets"])
    torch.cuda.synchronize()
    total = A.grad.double().norm().item()
    clip = min(1.0, 0.1 / (total + 1e-6))
    for (n, p, o), (_, p2, _) in zip(A.entries, B.entries):
        k = p.numel()
        if n not in names:
            if precision == "fp32":
                assert torch.allclose(p, p2, rtol=0, atol=2e-6), n            # (two runs' gradients differ by atomics' order)
            continue
        assert (A.v[o:o + k] == 0).all(), n
        lr = 1e-3 * (0.1 if "sampling_offsets" in n else 1.0)
        parts = 3 if n.endswith("in_proj_weight") else 1
        rows = p.shape[0] // parts
        for i in range(parts):
            sl = slice(i * rows, (i + 1) * rows)
            g = A.grad[o:o + k].view(p.shape[0], -1)[sl].cpu().double() * clip
            w = before[n].view(p.shape[0], -1)[sl].cpu().double()
            assert (A.m[o:o + k].view(p.shape[0], -1)[sl].cpu().double() - 0.1 * g).abs().max() <= 1e-6 * g.abs().max() + 1e-30
            u = 0.9 * 0.1 * g + 0.1 * g
            want, err = exact(u)
            s = 0.2 * max(u.shape) ** 0.5
            new = w * (1 - lr * 0.1) - lr * s * want
            got = p.detach().view(p.shape[0], -1)[sl].cpu().double()
            # (the clip factor and the direction carry a few fp32 roundings; eps = 1e-7 of the norm makes the scale matter a little)
            assert (got - new).norm() <= lr * s * (err + 3.45 ** 5 * 2.0 ** -20) + 4e-7 * w.norm(), n
    assert torch.equal(A.flat_bf16, A.flat.to(torch.bfloat16))
    sd = A.state_dict()
    assert sd["muon"] == A.muon_names
    with pytest.raises(ValueError):
        B.load_state_dict(sd)
    A.load_state_dict(sd)


def test_muon_schedule_and_zero_rate(gpu):
    """set_lr reaches both optimisers; at a rate of zero nothing moves and AdamW still leaves the matrices' state alone."""
    import poet_amd
    r = gpu("tiny", 2, True, "fp32", dropout=0.0)
    t = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.0, distributed=False, muon=True)
    A = t.arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w0 = A.flat.clone()
    A.set_lr(0.0)
    A.step(0.0)
    torch.cuda.synchronize()
    assert torch.equal(A.flat, w0)
    for n, p, o in A.entries:
        if n in A.muon_names:
            assert (A.v[o:o + p.numel()] == 0).all() and (A.m[o:o + p.numel()] != 0).any()
    A.set_lr(5e-4)
    w1, m1 = A.flat.clone(), A.m.clone()
    A.step(0.0)
    half = A.flat - w1
    A.flat.copy_(w1)
    A.m.copy_(m1)
    A.set_lr(1e-3)
    A.step(0.0)
    for n, p, o in A.entries:
        if n in A.muon_names:
            k = p.numel()
            full = (A.flat - w1)[o:o + k]
            assert (full - 2 * half[o:o + k]).abs().max() <= 4 * 2.0 ** -24 * (w1[o:o + k].abs().max() + 1), n


def test_graphed_trainer_with_muon_and_activation(gpu):
    """The captured step (input projection with SiLU, Muon in the optimiser graph) against the eager one, over several replays."""
    import poet_amd
    runs = []
    for graphed in (False, True):
        r = gpu("tiny", 2, True, "fp32", dropout=0.0)
        r["model"].input_proj_act = "silu"
        r["model"].train()
        kw = dict(lr=1e-4, weight_decay=1e-4, max_norm=0.1, muon=dict(momentum=0.9))
        tr = poet_amd.GraphedTrainer(r["model"], r["crit"], warm=1, **kw) if graphed else poet_amd.Trainer(r["model"], r["crit"], distributed=False, **kw)
        losses = [float(tr.step(r["samples"], r["targets"])[0]) for _ in range(5)]
        torch.cuda.synchronize()
        runs.append((losses, _params(r["model"]), tr.arena))
    (la, pa, A), (lb, pb, _) = runs
    assert A.muon_names
    for x, y in zip(la, lb):
        assert abs(x - y) <= 2e-3 * abs(x), (la, lb)
    # (fp32 atomics in other kernels reorder sums from run to run; an orthogonalised update amplifies a relative 1e-6 of the gradient)
    for n in pa:
        assert (pa[n] - pb[n]).norm() <= 5 * 1e-4 * 0.2 * (max(pa[n].shape) ** 0.5 if pa[n].dim() > 1 else 5.0) * pa[n].numel() ** 0.5 * 0.2 + 1e-6, n
