"""Refusals of the GroupNorm + activation and orthogonalisation entry points, checked without a GPU: the C ABI turns bad arguments into
error codes before anything is launched, the tensor-level wrappers raise."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

FAKE = ctypes.c_void_p(0x1000)
REFUSED = (-1, -2)                       # POET_ERR_ARG, POET_ERR_UNSUPPORTED: nothing was launched (a launch without a GPU is -3)


@pytest.fixture(scope="module")
def lib():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: a call that is not refused must find no GPU to run on")
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
        assert gn_fwd(lib, **kw) in REFUSED, kw
        assert b"groupnorm_act" in lib.poet_hip_last_error(), kw
    assert lib.poet_groupnorm_act_workspace(1, 10, 64, 7) < 0
    assert lib.poet_groupnorm_act_workspace(1, 10, 1 << 21, 1) < 0
    rc = lib.poet_groupnorm_act_bwd(FAKE, 640, 64, FAKE, 640, 64, FAKE, FAKE, FAKE, None, 0, 0, None, None, 0, 1, 10, 64, 8, 0, 0, 0, FAKE, 1 << 20, None)
    assert rc in REFUSED and b"something must be asked for" in lib.poet_hip_last_error()


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


def orth(lib, rows=(8,), cols=(16,), n=None, gd=0, od=0, steps=5, coeffs=None, eps=1e-7, ws=FAKE, nws=None, ptr=0x1000, ld=None):
    n = len(rows) if n is None else n
    r, c = (ctypes.c_int * len(rows))(*rows), (ctypes.c_int * len(cols))(*cols)
    need = lib.poet_muon_workspace(r, c, n)
    ptrs = (ctypes.c_void_p * len(rows))(*[ptr] * len(rows))
    lds = (ctypes.c_int64 * len(rows))(*(ld or cols))
    cf = (ctypes.c_double * (3 * max(steps, 1)))(*(coeffs or (3.4445, -4.7750, 2.0315)) * max(steps, 1))
    return lib.poet_orthogonalize(ptrs, lds, ptrs, lds, r, c, n, gd, od, steps, cf, eps, ws, need if nws is None else nws, None)


def test_orthogonalize_refuses_bad_arguments(lib):
    for kw in (dict(n=0), dict(rows=(0,)), dict(rows=(1 << 21,)), dict(cols=(-3,)), dict(gd=3), dict(od=-1), dict(steps=0), dict(steps=17),
               dict(coeffs=(50.0, 0.0, 0.0)), dict(coeffs=(float("nan"), 0.0, 0.0)), dict(coeffs=(float("inf"), 0.0, 0.0)), dict(eps=-1.0), dict(eps=float("nan")),
               dict(ws=None), dict(ws=ctypes.c_void_p(0x1008)), dict(nws=255), dict(rows=(300,), cols=(400,), nws=1 << 20), dict(ptr=None), dict(ld=(15,))):
        assert orth(lib, **kw) in REFUSED, kw
        assert b"orthogonalize" in lib.poet_hip_last_error() or b"muon" in lib.poet_hip_last_error(), kw


def test_muon_step_refuses_bad_arguments(lib):
    r, c = (ctypes.c_int * 1)(8), (ctypes.c_int * 1)(16)
    need = lib.poet_muon_workspace(r, c, 1)
    ptrs, cf = (ctypes.c_void_p * 1)(0x1000), (ctypes.c_double * 15)(*(3.4445, -4.7750, 2.0315) * 5)

    def step(p=ptrs, g=ptrs, m=ptrs, hi=None, lo=None, mu=0.95, n=1, nws=need):
        return lib.poet_muon_step(p, g, m, hi, lo, None, None, r, c, n, 0.02, mu, 1, 0.0, 5, cf, 1e-7, None, 0.0, 1.0, FAKE, nws, None)

    for kw in (dict(p=None), dict(g=None), dict(m=None), dict(lo=ptrs), dict(mu=1.0), dict(mu=-0.1), dict(mu=float("nan")), dict(n=0), dict(nws=0)):
        assert step(**kw) in REFUSED, kw
        assert b"muon_step" in lib.poet_hip_last_error(), kw


def test_muon_workspace_counts_every_plane(lib):
    """Two X buffers and the two square matrices, as fp16 pairs on whole tiles, and nothing that grows with the list beyond them."""
    one = lib.poet_muon_workspace((ctypes.c_int * 1)(256), (ctypes.c_int * 1)(256), 1)
    assert one >= 4 * 4 * 256 * 256
    five = lib.poet_muon_workspace((ctypes.c_int * 5)(*[256] * 5), (ctypes.c_int * 5)(*[256] * 5), 5)
    assert five <= 5 * one
    big = (ctypes.c_int * 9)(*[1 << 20] * 9)
    assert lib.poet_muon_workspace(big, big, 1) >= 16 << 40               # (64-bit sizes)
    assert lib.poet_muon_workspace(big, big, 9) < 0                       # more tiles than a launch can have


def test_overlap_of_written_matrices():
    """items: (start, rows, row stride, row width, written, index).  Whatever shares a byte is a clash (the other way round, columns that
    meet only below one's last row count as one)."""
    from poet_amd.ops import _clash
    assert not _clash([(0, 4, 64, 64, True, 0), (256, 4, 64, 64, True, 1)])
    assert _clash([(0, 4, 64, 64, True, 0), (252, 4, 64, 64, True, 1)])
    assert not _clash([(0, 4, 64, 64, False, 0), (0, 4, 64, 64, False, 1)])          # two inputs
    assert not _clash([(0, 4, 64, 64, False, 0), (0, 4, 64, 64, True, 0)])           # an output on its own input
    assert _clash([(0, 4, 64, 64, False, 0), (0, 4, 64, 64, True, 1)])
    assert not _clash([(0, 9, 64, 32, True, 0), (32, 9, 64, 32, True, 1)])           # halves of the same rows
    assert _clash([(0, 9, 64, 32, True, 0), (28, 9, 64, 32, True, 1)])
    assert _clash([(0, 9, 64, 36, True, 0), (32, 9, 64, 32, True, 1)])
    assert _clash([(0, 100, 8, 8, True, 0), (8, 1, 8, 8, False, 1), (400, 2, 8, 8, False, 2)])
    g = torch.Generator().manual_seed(3)
    n = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))                 # noqa: E731
    for _ in range(300):
        ld = n(4, 12)
        items = [(n(0, 60), n(1, 6), ld, n(1, ld + 1), bool(n(0, 2)), i // 2) for i in range(4)]
        bytes_of = [{s + r * ld + c for r in range(rows) for c in range(w)} for s, rows, ld, w, _, _ in items]
        want = any(bytes_of[i] & bytes_of[j] and (items[i][4] or items[j][4]) and items[i][5] != items[j][5] for i in range(4) for j in range(i))
        assert _clash(items) or not want, items


def test_groupnorm_output_apart_from_its_input():
    from poet_amd.ops import _apart, _rows3
    buf = torch.zeros(2, 12, 16)

    def apart(a, b):
        N, HW, C = a.shape
        _apart(a, *_rows3(a, "a", N, HW, C), b, *_rows3(b, "b", N, HW, C), N, HW, C, "y")

    apart(buf, buf)
    apart(buf, buf.clone())
    apart(buf[:, :6], buf[:, 6:])                         # other rows of the same images, either way round
    apart(buf[:, 6:], buf[:, :6])
    apart(buf[:, :, :8], buf[:, :, 8:])                   # other columns
    apart(buf[:1, 2:5], buf[:1, 5:8])
    for a, b in ((buf[:, :7], buf[:, 5:]), (buf[:, :6], buf[:, 1:7]), (buf[:, :, :8], buf[:, :, 4:12]), (buf[:, ::2], buf[:, :6]), (buf[0:1].expand(2, 12, 16), buf),
                 (buf, buf.view(torch.int32)), (buf.view(-1)[:192].view(1, 12, 16), buf.view(torch.bfloat16).view(-1)[:192].view(1, 12, 16))):
        with pytest.raises(ValueError):
            apart(a, b)


def test_sizes_beyond_a_launch_are_refused(lib):
    need = lib.poet_groupnorm_act_workspace(1 << 24, 1, 64, 64)
    assert need > 0 and gn_fwd(lib, N=1 << 24, HW=1, C=64, G=64, nws=need) in REFUSED and b"threads" in lib.poet_hip_last_error()
    for cf in ((3.0, float("nan"), 0.0), (3.0, 0.0, float("nan")), (3.0, float("-inf"), 0.0)):
        assert orth(lib, coeffs=cf) in REFUSED and b"range" in lib.poet_hip_last_error()


def test_m0_is_only_written_by_the_dma(tmp_path):
    """The tiles' LDS-DMA sets M0 by hand in inline assembly (hipcc takes no "m0" clobber): safe only while nothing else in that source uses it."""
    from poet_amd.build import CSRC, FLAGS, _hipcc
    if not (os.path.exists(_hipcc()) or shutil.which(_hipcc())):
        pytest.skip("no hipcc")
    out = str(tmp_path / "muon.s")
    subprocess.check_call([_hipcc(), *FLAGS, "-S", "--cuda-device-only", os.path.join(CSRC, "muon.hip"), "-o", out], stderr=subprocess.DEVNULL)
    text = open(out).read()
    lines = [l.strip() for l in text.splitlines() if re.search(r"\bm0\b", l) and not l.lstrip().startswith((";", "//"))]
    assert lines and all(re.fullmatch(r"s_mov_b32 m0, s\d+", l) for l in lines), [l for l in lines if not re.fullmatch(r"s_mov_b32 m0, s\d+", l)][:5]
    assert not re.search(r"v_movrel|s_set_gpr_idx", text)
