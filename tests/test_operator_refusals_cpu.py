"""What the GroupNorm + activation and orthogonalisation operators refuse before they look at a device."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [True, False])
def test_group_norm_act_refuses_forward_mode_tangents(which, grad):
    """A tangent on x, weight or bias is refused (with gradients on and off: no_grad does not switch forward mode off); inside a dual level, tensors
    without one go on to the ordinary checks."""
    from poet_amd import GroupNormAct, PoetHipError, functional
    args = [torch.randn(2, 5, 8), torch.ones(8), torch.zeros(8)]
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = list(args)
        dual[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            functional.group_norm_act(*dual, 2, act="silu")
        with pytest.raises(PoetHipError):                   # (no GPU path for CPU tensors)
            functional.group_norm_act(*args, 2, act="silu")
    if which == 0:
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            GroupNormAct(2, 8)(fwd.make_dual(args[0], args[0]))


def test_orthogonalize_refuses_what_asks_for_a_gradient():
    """requires_grad under enabled gradients, or a tangent, alone and in a list; detached, or under no_grad, the ordinary checks are next."""
    from poet_amd import PoetHipError, ops
    g, p = torch.randn(4, 6), torch.nn.Parameter(torch.randn(4, 6))
    for arg in (p, [g, p], p * 2, torch.stack([p, p])):
        with pytest.raises(NotImplementedError, match="no gradient"):
            ops.orthogonalize(arg)
    with fwd.dual_level():
        d = fwd.make_dual(g, g)
        for arg in (d, [g, d]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.orthogonalize(arg)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                ops.orthogonalize(arg)
    for arg in (g, p.detach(), [g, p.detach()]):
        with pytest.raises(PoetHipError):                   # (no GPU path for CPU tensors)
            ops.orthogonalize(arg)
    with torch.no_grad(), pytest.raises(PoetHipError):
        ops.orthogonalize(p)


def arena(**kw):
    """A parameter arena over one encoder-like Linear, on the CPU (where Muon is refused, after its options have been looked at)."""
    from poet_amd import ParamArena
    m = torch.nn.Module()
    m.transformer = torch.nn.Module()
    m.transformer.encoder = torch.nn.Linear(8, 4)
    return ParamArena(m, **kw)


def test_an_empty_dict_of_muon_options_means_the_defaults():
    for off in (None, False):
        a = arena(muon=off)
        assert a.muon is None and a.muon_names == [] and a.muon_blocks is None
    for on in (True, {}, dict(momentum=0.9)):
        with pytest.raises(ValueError, match="GPU"):
            arena(muon=on)


def test_muon_options_are_checked_when_the_arena_is_built():
    """Unknown names and values that the first step would refuse, before a parameter is moved; a refusal further on is of the device only."""
    for bad in (dict(beta=0.9), dict(momentun=0.9), dict(momentum=1.0), dict(momentum=-0.1), dict(momentum=float("nan")), dict(steps=0), dict(steps=17),
                dict(eps=-1.0), dict(coeffs=(1.0, 2.0)), dict(steps=3, coeffs=[(3.0, -3.2, 1.2)] * 2), dict(scale="max"), dict(self=1)):
        with pytest.raises(ValueError) as e:
            arena(muon=bad)
        assert "GPU" not in str(e.value), bad
    for good in (dict(momentum=0.0, nesterov=False, steps=3, coeffs=[(3.0, -3.2, 1.2)] * 3, eps=0.0, scale="spectral"), dict(lr=0.02, weight_decay=0.0)):
        with pytest.raises(ValueError, match="GPU"):
            arena(muon=good)


def test_more_narrow_matrices_than_a_launch_has_workgroups_are_refused():
    """2^23 workgroups of 512 threads are 2^32: refused with the workspace, before another group of the list has been updated."""
    from poet_amd import _lib
    lib, n = _lib.load(), 1 << 23
    dims = (ctypes.c_int * (n + 1))(*[2] * (n + 1))
    assert lib.poet_muon_workspace(dims, dims, n - 1) > 0
    assert lib.poet_muon_workspace(dims, dims, n) < 0 and b"too many matrices" in lib.poet_hip_last_error()
    dims[n] = 300
    assert lib.poet_muon_workspace(dims, dims, n + 1) < 0


def test_parameter_gradients_apart_from_each_other_and_from_the_parameters():
    from poet_amd.ops import _params_apart
    assert _params_apart(0, 256, 512, 768, 256) and _params_apart(768, 512, 0, 0, 256)
    for a in ((0, 0, 512, 768), (0, 252, 512, 768), (0, 256, 512 - 4, 768), (512, 0, 512, 768), (0, 768 + 4, 512, 768), (600, 0, 4096, 380)):
        assert not _params_apart(*a, 256), a
    assert _params_apart(0, 0, 0, 0, 0)                     # (no channels)


def test_a_negative_rate_is_refused_with_muon():
    for lr in (-1e-3, float("nan")):
        with pytest.raises(ValueError, match="negative"):
            arena(lr=lr, muon=True)
    assert arena(lr=-1e-3).lr == -1e-3
