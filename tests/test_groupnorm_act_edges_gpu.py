"""Edges of GroupNorm + activation: constant groups far from zero, squares beyond fp32, on both the one-launch and the chunked path."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.test_groupnorm_act_gpu import DTYPES, fn, make, ops, ref, check  # noqa: E402,F401


# (rows, channels a group): n = rows x channels, most of them with n fl(1 / n) != 1; 41 .. 700 rows take one launch, the others chunks (20011 x 1100: a
# group in pieces of channels)
CONSTANT = [(41, 8), (47, 8), (55, 1), (61, 12), (83, 12), (300, 8), (700, 3), (4700, 8), (5003, 3), (20011, 12), (1031, 1100)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("HW,cpg", CONSTANT)
def test_constant_groups_are_exactly_beta(ops, HW, cpg, dtype):
    """x = c over a group: the mean is c (a first mean is some ulps off; the n equal deviations from it, their sum and its quotient by n are right to
    2^-20 of those ulps, so the corrected mean rounds to c), the variance 0, h = 0 and z = beta, whatever 1 / sqrt(eps) = 316 would make of a mean one ulp off.  The stored statistics say the same."""
    dt, G = DTYPES[dtype], 4
    C = G * cpg
    for k, v in enumerate((1000.0, 0.3, -77.77)):
        x, w, b, dy = make(2, HW, C, dt, seed=HW + k)
        x[1, :, cpg:2 * cpg] = v
        c = x[1, 0, cpg].float()
        y, stats = torch.empty_like(x), torch.empty(2, G, 2, device="cuda")
        ops.groupnorm_act_fwd(x, w, b, y, G, "none", stats=stats)
        assert torch.equal(y[1, :, cpg:2 * cpg], b[cpg:2 * cpg].to(dt).expand(HW, cpg)), v
        assert stats[1, 1, 0] == c, (v, float(stats[1, 1, 0] - c))
        r = ref(x, w, b, G, "none", 1e-5)
        check(y, r["y"], r["tol_y"], f"the other groups, {v}")
        # backward of the same group: h = 0, so dgamma gets nothing from it and dx is rstd (p - mean p)
        dx, dw, db = torch.empty_like(x), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        ops.groupnorm_act_bwd(dy[1:], x[1:], stats[1:], w, b, G, "none", dx=dx[1:], dgamma=dw, dbeta=db)
        assert (dw[cpg:2 * cpg] == 0).all()


def test_a_far_mean_with_a_small_spread(ops):
    """Two values, c and c + 2^-8, half the rows each: mean c + 2^-9 and variance 2^-18 (both fp32 numbers), so h = +- 2^-9 / sqrt(2^-18 + eps)."""
    for HW, cpg in ((82, 8), (610, 4), (9402, 8)):
        x = torch.full((1, HW, 4 * cpg), 1000.0, device="cuda")
        x[:, ::2] += 2.0 ** -8
        w, b = torch.ones(4 * cpg, device="cuda"), torch.zeros(4 * cpg, device="cuda")
        y, stats = torch.empty_like(x), torch.empty(1, 4, 2, device="cuda")
        ops.groupnorm_act_fwd(x, w, b, y, 4, "none", stats=stats)
        assert (stats[..., 0] == 1000.0 + 2.0 ** -9).all()
        want = 2.0 ** -9 / (2.0 ** -18 + 1e-5) ** 0.5
        # (rstd: the variance's sums of n equal squares, eps and the root, a few roundings of 2^-24; the deviation itself is exact)
        assert (y.double().abs() - want).abs().max() <= 16 * 2.0 ** -24 * want


@pytest.mark.parametrize("HW", [40, 900, 20000])
@pytest.mark.parametrize("size", [1e20, 1e25, 1e37])
def test_squares_beyond_fp32_are_not_finite(ops, HW, size):
    """Deviations whose squares leave fp32: the variance is not representable, so the group comes out NaN, never finite and wrong; the other groups
    and images are untouched.  Deviations of 1e15 (sums of squares to 1e36) stay in range."""
    x, w, b, _ = make(2, HW, 64, torch.float32, seed=HW)
    clean, big = torch.empty_like(x), x.clone()
    ops.groupnorm_act_fwd(x, w, b, clean, 8, "silu")
    big[1, :, 8:16] *= size
    y, stats = torch.empty_like(x), torch.empty(2, 8, 2, device="cuda")
    ops.groupnorm_act_fwd(big, w, b, y, 8, "silu", stats=stats)
    assert torch.isnan(y[1, :, 8:16]).all() and torch.isnan(stats[1, 1, 1])
    keep = torch.ones(2, 1, 64, dtype=torch.bool, device="cuda").expand(2, HW, 64).clone()
    keep[1, :, 8:16] = False
    assert torch.equal(y[keep], clean[keep])
    big[1, :, 8:16] = x[1, :, 8:16] * 1e15
    ops.groupnorm_act_fwd(big, w, b, y, 8, "silu")
    r = ref(big, w, b, 8, "silu", 1e-5)
    check(y, r["y"], r["tol_y"], "deviations of 1e15")


def test_overlapping_parameter_gradients_are_refused(ops):
    """dgamma / dbeta on each other, or on gamma / beta, which other workgroups read meanwhile: refused, nothing written."""
    x, w, b, dy = make(2, 50, 64, torch.float32)
    stats = torch.empty(2, 8, 2, device="cuda")
    ops.groupnorm_act_fwd(x, w, b, torch.empty_like(x), 8, "silu", stats=stats)
    buf = torch.full((200,), 7.0, device="cuda")
    w0, b0 = w.clone(), b.clone()
    for dw, db in ((buf[:64], buf[:64]), (buf[:64], buf[63:127]), (w, buf[:64]), (buf[:64], w), (b, buf[:64]), (buf[:64], b)):
        with pytest.raises(ValueError):
            ops.groupnorm_act_bwd(dy, x, stats, w, b, 8, "silu", dgamma=dw, dbeta=db)
    assert (buf == 7).all() and torch.equal(w, w0) and torch.equal(b, b0)
    ops.groupnorm_act_bwd(dy, x, stats, w, b, 8, "silu", dgamma=buf[:64], dbeta=buf[64:128])
    assert (buf[128:] == 7).all() and (buf[:128] != 7).all()
