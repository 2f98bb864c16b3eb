"""Refusals of the GroupNorm + activation and orthogonalisation entry points, checked without a GPU: the C ABI turns bad arguments into
error codes before anything is launched, the tensor-level wrappers raise."""
import ctypes
import os

import pytest
import torch

FAKE = ctypes.c_void_p(0x1000)


@pytest.fixture(scope="module")
def lib():
    from poet_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from poet_amd.build import build_library
        build_library(verbose=False)
    return _lib.load()


def gn_fwd(lib, x=FAKE, N=1, HW=10, C=64, G=8, act=0, xd=0, yd=0, ws=FAKE, nws=None):
    need = lib.poet_groupnorm_act_workspace(N, HW, C, G)
    return lib.poet_groupnorm_act_fwd(x, HW * C, C, FAKE, FAKE, FAKE, HW * C, C, FAKE, N, HW, C, G, 1e-5, act, xd, yd, ws, need if nws is None else nws, None)


def test_groupnorm_act_refuses_bad_arguments(lib):
    for kw in (dict(x=None), dict(G=7), dict(G=0), dict(N=0), dict(HW=-1), dict(act=4), dict(act=-1), dict(ws=None), dict(nws=8),
               dict(ws=ctypes.c_void_p(0x1001)), dict(xd=7), dict(xd=2, yd=0), dict(xd=1, yd=2)):
        assert gn_fwd(lib, **kw) < 0, kw
        assert b"groupnorm_act" in lib.poet_hip_last_error(), kw
    assert lib.poet_groupnorm_act_workspace(1, 10, 64, 7) < 0
    assert lib.poet_groupnorm_act_workspace(1, 10, 1 << 21, 1) < 0
    rc = lib.poet_groupnorm_act_bwd(FAKE, 640, 64, FAKE, 640, 64, FAKE, FAKE, FAKE, None, 0, 0, None, None, 0, 1, 10, 64, 8, 0, 0, 0, FAKE, 1 << 20, None)
    assert rc < 0 and b"something must be asked for" in lib.poet_hip_last_error()


def test_groupnorm_act_workspace_covers_every_layout(lib):
    """The workspace grows with nothing but N, C and the row chunks, and stays small against the tensor."""
    for N, HW, C, G in ((1, 1, 8, 1), (16, 4800, 256, 32), (8, 19200, 256, 32), (2, 33, 4096, 2), (1, 40, 5000, 1250), (1, 50, 2100, 1), (100000, 1, 8, 8)):
        need = lib.poet_groupnorm_act_workspace(N, HW, C, G)
        assert 0 < need and need % 8 == 0


def test_rows3_refuses_what_a_kernel_could_not_address():
    from poet_amd.ops import _rows3
    x = torch.empty(2, 5, 8)
    assert _rows3(x, "x", 2, 5, 8) == (40, 8)
    assert _rows3(x.transpose(0, 1), "x", 5, 2, 8, out=True) == (8, 40)          # images interleaved row by row: no element twice
    with pytest.raises(ValueError):
        _rows3(x.transpose(1, 2), "x", 2, 8, 5)
    with pytest.raises(ValueError):
        _rows3(x, "x", 2, 5, 4)
    with pytest.raises(ValueError):
        _rows3(x[:1].expand(2, 5, 8), "y", 2, 5, 8, out=True)
    assert _rows3(x[:1].expand(2, 5, 8), "x", 2, 5, 8) == (0, 8)                 # an input may repeat


def test_cpu_tensors_are_refused():
    from poet_amd import PoetHipError, functional
    x, w = torch.zeros(1, 4, 8), torch.ones(8)
    with pytest.raises(PoetHipError):
        functional.group_norm_act(x, w, w, 2)
