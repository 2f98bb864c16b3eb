"""The Muon half of the optimiser step inside the trainers' arena."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def build():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from tests.product_runner import build_product
    return build_product


def test_a_refused_step_changes_nothing(build):
    """Coefficients that only the kernels' own check refuses (the iteration leaves its range): no AdamW half, no count, no moment."""
    import poet_amd
    r = build("tiny", 2, True, "fp32", dropout=0.0)
    A = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.1, distributed=False, muon=dict(coeffs=(50.0, 0.0, 0.0))).arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    before = [t.clone() for t in (A.flat, A.m, A.v, A.flat_bf16, A.flat_bf16_lo)]
    for _ in range(2):
        with pytest.raises(poet_amd.PoetHipError, match="range"):
            A.step(0.1)
    torch.cuda.synchronize()
    assert A.step_count == 0 and all(torch.equal(a, b) for a, b in zip(before, (A.flat, A.m, A.v, A.flat_bf16, A.flat_bf16_lo)))


def test_output_layers_step_by_adamw(build):
    """Learned reference points: their 2-row Linear is an output layer like the heads' last ones, so AdamW steps it (its second moment moves)."""
    import poet_amd
    r = build("tiny", 2, True, "fp32", dropout=0.0, ref_points_mode="learned", query_embedding_mode="learned")
    A = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, max_norm=0.0, distributed=False, muon=True).arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    A.step(0.0)
    outputs = [n for n, p, _ in A.entries if p.dim() > 1 and ("reference_points" in n or ("head" in n and ".layers.2." in n) or "query_embed" in n)]
    assert "transformer.reference_points.weight" in outputs and len(outputs) >= 4
    for n, p, o in A.entries:
        owned = n in A.muon_names
        assert owned == (p.dim() > 1 and n not in outputs and "level_embed" not in n), n
        assert ((A.v[o:o + p.numel()] != 0).any().item()) != owned, n


def _formula(A, p0, m0, mu, wd, max_norm):
    """Every Muon matrix of the arena after a step whose gradients are still there, against the float64 update from p0, m0; returns how many were compared."""
    from tests.test_muon_gpu import exact
    total = A.grad.double().norm().item()
    clip = min(1.0, max_norm / (total + 1e-6)) if max_norm else 1.0
    count = 0
    for n, p, o in A.entries:
        if n not in A.muon_names:
            continue
        lr = A.lr * (0.1 if "sampling_offsets" in n else 1.0)
        parts = 3 if n.endswith("in_proj_weight") else 1
        rows = p.shape[0] // parts
        cut = lambda flat, i: flat[o:o + p.numel()].view(p.shape[0], -1)[i * rows:(i + 1) * rows].cpu().double()      # noqa: E731
        for i in range(parts):
            g, w, m = cut(A.grad, i) * clip, cut(p0, i), cut(m0, i)
            m1 = mu * m + (1 - mu) * g
            # (three roundings of 2^-24 in m, a few more in the clip factor)
            assert (cut(A.m, i) - m1).abs().max() <= 2.0 ** -20 * (m.abs().max() + g.abs().max()) + 1e-37, n
            u = mu * m1 + (1 - mu) * g
            want, err = exact(u)
            s = 0.2 * max(u.shape) ** 0.5
            # the direction's own error: 2^-20 of its terms, which may cancel in u, carried on at 3.45 a step
            direction = 2.0 ** -20 * (m.norm() + g.norm()).item() / max(u.norm().item(), 1e-30)
            got, new = cut(A.flat, i), w * (1 - lr * wd) - lr * s * want
            assert (got - new).norm() <= lr * s * (err + 3.45 ** 5 * direction) + 4e-7 * w.norm(), (n, i)
            # ... and the matrix did move: by far more than that bound
            assert (got - w * (1 - lr * wd)).norm() >= 0.9 * lr * s * want.norm() and want.norm() > 0.3, (n, i)
            count += 1
    return count


def test_captured_steps_follow_the_formula(build):
    """GraphedTrainer's replays: after each, every Muon matrix has moved from where it was by the update of THIS step's gradient and momentum, whatever the
    run-to-run noise of the gradients; the rate changes between replays."""
    import poet_amd
    r = build("tiny", 2, True, "fp32", dropout=0.0)
    r["model"].train()
    tr = poet_amd.GraphedTrainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.1, warm=1, muon=dict(momentum=0.9))
    A = tr.arena
    for k in range(5):
        A.set_lr((1e-3, 1e-3, 4e-4, 4e-4, 2e-3)[k])
        p0, m0 = A.flat.clone(), A.m.clone()
        tr.step(r["samples"], r["targets"])
        torch.cuda.synchronize()
        assert _formula(A, p0, m0, 0.9, 0.1, 0.1) >= 10, k
        assert torch.equal(A.flat_bf16, A.flat.to(torch.bfloat16))
    assert tr.ready


@pytest.mark.parametrize("max_norm", [0.0, 0.1])
def test_captured_arena_step_has_the_bits_of_the_eager_one(build, max_norm):
    """The optimiser step alone, captured, against the eager one on the same gradients: weights, moments and images bit for bit over five replays, with
    other gradients and rates in between and eager work on the device."""
    import poet_amd
    from poet_amd import ops
    arenas = []
    for _ in range(2):
        r = build("tiny", 2, True, "fp32", dropout=0.0)
        arenas.append(poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=max_norm, distributed=False, muon=dict(momentum=0.9)).arena)
    E, G = arenas
    assert torch.equal(E.flat, G.flat)
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda: 1e-2 * torch.randn(E.grad.shape, generator=gen, device="cuda")      # noqa: E731

    def step(A):
        ops.counter_add(A.step_word, 1)
        A.step(max_norm, step_dev=A.step_word)

    state = lambda A: (A.flat, A.m, A.v, A.flat_bf16, A.flat_bf16_lo)      # noqa: E731
    for A in arenas:
        A.grad.copy_(torch.full_like(A.grad, 1e-3))
        step(A)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(G)
    for k in range(5):
        g, lr = new(), 1e-3 / (k + 1)
        for A in arenas:
            A.grad.copy_(g)
            A.set_lr(lr)
        before = E.flat.clone()
        step(E)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(state(E), state(G))), k
        for n, p, o in E.entries:
            assert not torch.equal(E.flat[o:o + p.numel()], before[o:o + p.numel()]), (k, n)
