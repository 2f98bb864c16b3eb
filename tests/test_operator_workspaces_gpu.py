"""What a workspace holds before a call (here 0xFF bytes: NaN as fp16, fp32 and fp64, -1 as an integer) does not reach a result, and nothing is written behind
its end.  The calls get exactly the bytes they ask for, inside a larger buffer of a known pattern."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.test_muon_gpu import check, matrix, ops  # noqa: E402,F401

GUARD = 1 << 16


class Dirty:
    """Stands in for ops._muon_ws: every workspace is 0xFF bytes from end to end, with a guard behind it."""

    def __init__(self):
        self.given = []

    def __call__(self, lib, rows, cols, n, device):
        need = lib.poet_muon_workspace(rows, cols, n)
        assert need > 0
        buf = torch.full((need + GUARD,), 0xFF, dtype=torch.uint8, device=device)
        buf[need:] = 0x5A
        self.given.append((buf, need))
        return buf[:need]

    def intact(self):
        assert self.given
        ok = all((buf[need:] == 0x5A).all().item() for buf, need in self.given)
        self.given.clear()
        return ok


# every kind of group (one workgroup, slabs, chains of small and of large tiles), either tile edge in both products, sizes that end inside a tile
LISTS = [[(1, 1)], [(66, 256)], [(33, 896)], [(96, 288), (90, 17)], [(20, 2000)], [(60, 1500)] * 3, [(31, 4097), (64, 700)],
         [(200, 200)] * 3, [(200, 200)] * 10, [(200, 200)] * 14, [(200, 400)] * 8, [(131, 257)], [(97, 97), (250, 1000)],
         [(257, 131), (300, 300)], [(300, 300)] * 4, [(513, 513)], [(321, 700), (450, 450)], [(1100, 1030)] * 2, [(1100, 1030)] * 6,
         [(400, 2600), (2500, 500), (600, 600), (520, 300)], [(20, 100), (7, 33), (90, 64), (50, 60), (1, 1)] * 8,
         [(256, 256)] * 9 + [(900, 256)] * 4 + [(200, 410)] * 3 + [(700, 300), (260, 1500), (300, 300), (3, 50), (40, 900)]]


@pytest.mark.parametrize("shapes", LISTS, ids=lambda s: f"{len(s)}x{s[0][0]}x{s[0][1]}")
def test_orthogonalize_on_a_workspace_of_nan(ops, monkeypatch, shapes):
    gs = [matrix(m, n, seed=i).cuda() for i, (m, n) in enumerate(shapes)]
    clean = ops.orthogonalize(gs)
    dirty = Dirty()
    monkeypatch.setattr(ops, "_muon_ws", dirty)
    outs = ops.orthogonalize(gs)
    assert dirty.intact()
    for i, (g, o, c) in enumerate(zip(gs, outs, clean)):
        assert torch.isfinite(o).all() and torch.equal(o, c), (i, shapes[i])
    for i in sorted({shapes.index(s) for s in shapes})[:4]:
        check(outs[i], gs[i], f"{shapes[i]}")
        assert torch.equal(outs[i], ops.orthogonalize(gs[i])), shapes[i]              # (alone: other tiles, other places in the workspace)
    assert dirty.intact()


@pytest.mark.parametrize("shapes", LISTS, ids=lambda s: f"{len(s)}x{s[0][0]}x{s[0][1]}")
def test_muon_step_on_a_workspace_of_nan(ops, monkeypatch, shapes):
    def lists():
        return [[matrix(m, n, seed=k + 3 * i).cuda() for i, (m, n) in enumerate(shapes)] for k in range(3)]
    a, b = lists(), lists()
    ops.muon_step(*a, lr=0.02, weight_decay=0.1)
    dirty = Dirty()
    monkeypatch.setattr(ops, "_muon_ws", dirty)
    ops.muon_step(*b, lr=0.02, weight_decay=0.1)
    assert dirty.intact()
    for x, y in zip(a[0] + a[2], b[0] + b[2]):
        assert torch.isfinite(y).all() and torch.equal(x, y)


SHAPES = [(1, 1, 8, 1), (3, 121, 96, 8), (2, 1000, 66, 33), (1, 50, 2100, 1), (2, 33, 4096, 2), (1, 40, 5000, 1250), (16, 1200, 256, 32), (2, 5000, 64, 2), (3, 4001, 36, 3),
          (1, 20011, 256, 256), (5, 17, 40, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,HW,C,G", SHAPES)
def test_groupnorm_act_on_a_workspace_of_nan(ops, N, HW, C, G, dtype):
    """The C entry points on a workspace of exactly their size, against the ordinary calls: the same bits."""
    from poet_amd import _lib
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(HW)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")      # noqa: E731
    x, dy, w, b = r(N, HW, C).to(dtype), r(N, HW, C).to(dtype), r(C), r(C)
    y, stats, dx, dw, db = torch.empty_like(x), torch.empty(N, G, 2, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ops.groupnorm_act_fwd(x, w, b, y, G, "gelu", stats=stats)
    ops.groupnorm_act_bwd(dy, x, stats, w, b, G, "gelu", dx=dx, dgamma=dw, dbeta=db)
    need, dt = lib.poet_groupnorm_act_workspace(N, HW, C, G), ops.dcode(x)
    buf = torch.full((need + GUARD,), 0xFF, dtype=torch.uint8, device="cuda")
    buf[need:] = 0x5A
    got = [torch.empty_like(t) for t in (y, stats, dx, dw, db)]
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.poet_groupnorm_act_fwd(p(x), HW * C, C, p(w), p(b), p(got[0]), HW * C, C, p(got[1]), N, HW, C, G, 1e-5, 2, dt, dt, p(buf), need, s) == 0
    buf[:need] = 0xFF
    assert lib.poet_groupnorm_act_bwd(p(dy), HW * C, C, p(x), HW * C, C, p(stats), p(w), p(b), p(got[2]), HW * C, C, p(got[3]), p(got[4]), 0, N, HW, C, G, 2, dt, dt,
                                      p(buf), need, s) == 0
    assert all(torch.equal(u, v) for u, v in zip((y, stats, dx, dw, db), got)) and (buf[need:] == 0x5A).all()
