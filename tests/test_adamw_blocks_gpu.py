"""The AdamW step over a flat range: learning-rate words of any sign, and blocks of 64 elements that another optimiser owns."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from poet_amd import ops as _ops
    return _ops


def state(n, seed=0, off=0):
    """p, g, m, v, bf16 images hi, lo; off elements behind a 16-byte boundary."""
    g = torch.Generator().manual_seed(seed)
    vals = [torch.randn(n, generator=g), 0.01 * torch.randn(n, generator=g), 0.01 * torch.randn(n, generator=g), 1e-4 * torch.rand(n, generator=g),
            torch.full((n,), 3.0), torch.full((n,), 5.0)]
    out = []
    for i, t in enumerate(vals):
        buf = torch.zeros(n + 8, dtype=torch.float32 if i < 4 else torch.bfloat16, device="cuda")[off:off + n]
        buf.copy_(t)
        out.append(buf)
    return out


def step(ops, s, lr=1e-2, wd=0.1, **kw):
    p, g, m, v, hi, lo = s
    ops.adamw(p, g, m, v, p.numel(), lr, 0.9, 0.999, 1e-8, wd, 3, p_bf16=hi, p_bf16_lo=lo, **kw)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("n", [64, 257, 5003])
def test_learning_rate_words_of_any_sign(ops, n, off):
    """lr_scale multiplies lr, whatever its sign: a word of -0.5 at lr is a word of 0.5 at -lr, bit for bit; one of -0 is one of 0: the weights
    stay, their moments move on."""
    blocks = (n + 63) // 64
    a, b = state(n, off=off), state(n, off=off)
    words = 0.1 + torch.rand(blocks, generator=torch.Generator().manual_seed(1)).cuda()
    step(ops, a, lr_scale=-words)
    step(ops, b, lr=-1e-2, lr_scale=words)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c, before = state(n, off=off), state(n, off=off)
    step(ops, c, lr_scale=torch.full((blocks,), -0.0, device="cuda"))
    assert torch.equal(c[0], before[0]) and torch.equal(c[2], a[2]) and torch.equal(c[3], a[3]) and not torch.equal(c[2], before[2])
    assert torch.equal(c[4], before[0].bfloat16())
    # the formula in float64, a step up the gradient: relative roundings of a few 2^-24 in m, sqrt(v) and their quotient, one in p
    p, g, m, v = (t.cpu().double() for t in before[:4])
    lr = -1e-2 * words.cpu().double().repeat_interleave(64)[:n]
    m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
    move = (lr / (1 - 0.9 ** 3)) * m / (v.sqrt() / (1 - 0.999 ** 3) ** 0.5 + 1e-8)
    # (1 - 0.999^3 in fp32: 2^-24 absolute of 3e-3, so 2e-5 relative, half of it under the root; 1 - b1, 1 - b2 and m's cancellation the rest)
    assert ((a[0].cpu().double() - (p * (1 - lr * 0.1) - move)).abs() <= 4e-5 * move.abs() + 4 * 2.0 ** -24 * p.abs() + 1e-8).all()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("n", [64, 257, 5003])
def test_blocks_of_another_optimiser(ops, n, off):
    """A marked block keeps weights, moments and images; every other one has the bits of a step without marks."""
    blocks = (n + 63) // 64
    words = 0.1 + torch.rand(blocks, generator=torch.Generator().manual_seed(2)).cuda()
    for marks in (torch.arange(blocks) % 2, torch.arange(blocks) % 3 == 2, torch.ones(blocks), torch.zeros(blocks)):
        skip = marks.to(torch.uint8).cuda()
        a, b, before = state(n, off=off), state(n, off=off), state(n, off=off)
        step(ops, a, lr_scale=words, skip=skip)
        step(ops, b, lr_scale=words)
        owned = skip.bool().repeat_interleave(64)[:n]
        for x, y, z in zip(a, b, before):
            assert torch.equal(x[owned], z[owned]) and torch.equal(x[~owned], y[~owned])
    c, d = state(n, off=off), state(n, off=off)
    step(ops, c, skip=torch.zeros(blocks, dtype=torch.uint8, device="cuda"))
    step(ops, d)
    assert all(torch.equal(x, y) for x, y in zip(c, d))


def test_arena_with_a_negative_rate(ops):
    """Without Muon a negative rate steps up the gradient; with it, where the matrices' rates count by their magnitude, it is refused."""
    import poet_amd
    from tests.product_runner import build_product
    r = build_product("tiny", 2, True, "fp32", dropout=0.0)
    A = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.0, max_norm=0.0, distributed=False).arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w0 = A.flat.clone()
    A.set_lr(-1e-3)
    A.step(0.0)
    for n, p, o in A.entries:
        k = slice(o, o + p.numel())
        assert ((A.flat[k] - w0[k]) * A.grad[k] >= 0).all() and not torch.equal(A.flat[k], w0[k]), n
    q = build_product("tiny", 2, True, "fp32", dropout=0.0)
    M = poet_amd.Trainer(q["model"], q["crit"], lr=1e-3, max_norm=0.0, distributed=False, muon=True).arena
    keep = M.lr_scale.clone()
    for bad in (-1e-3, float("nan")):
        with pytest.raises(ValueError):
            M.set_lr(bad)
    assert torch.equal(M.lr_scale, keep) and M.lr == 1e-3
