"""The workspace that the GroupNorm + activation entry points ask for is enough for every layout they may choose, and bounded by the tensor."""
import ctypes

import pytest

from tests.test_operators_cpu import FAKE, lib  # noqa: F401  (the fixture skips where a GPU exists: made-up addresses)

SHAPES = [(1, 1, 8, 1), (16, 4800, 256, 32), (8, 19200, 256, 32), (2, 33, 4096, 2), (1, 40, 5000, 1250), (1, 50, 2100, 1), (100000, 1, 8, 8),
          (1, 20011, 36, 3), (3, 70001, 256, 256), (1, 2047, 1028, 1), (2, 513, 4112, 2), (1, 9, 3, 3), (5, 100, 1 << 14, 1 << 14), (1, 5000, 1 << 20, 1)]
TYPES = [(0, 0), (1, 1), (2, 2), (1, 0), (0, 1)]
LAUNCHED = -3                            # POET_ERR_LAUNCH: every check has passed, and there is no GPU to run on


@pytest.mark.parametrize("N,HW,C,G", SHAPES)
def test_workspace_is_enough_for_every_type_and_alignment(lib, N, HW, C, G):
    """Both directions at the returned size, aligned (vectors) and not (single elements), contiguous and strided rows: none is refused."""
    need = lib.poet_groupnorm_act_workspace(N, HW, C, G)
    # 8 bytes x (N G (T P + 1) + N T C) with G P <= C and T <= HW / 8 + 1 chunks of rows
    assert 0 < need <= 2 * N * HW * C + 24 * N * C and need % 8 == 0
    for xd, yd in TYPES:
        for base in (0x1000, 0x1000 + (4 if xd == 0 or yd == 0 else 2)):
            for row in (C, C + 8, C + 1):
                t = ctypes.c_void_p(base)
                img = HW * row
                rc = lib.poet_groupnorm_act_fwd(t, img, row, FAKE, FAKE, t, img, row, None, N, HW, C, G, 1e-5, 3, xd, yd, FAKE, need, None)
                assert rc == LAUNCHED, (xd, yd, base, row, rc, lib.poet_hip_last_error())
                for dx, dw in ((t, FAKE), (t, None), (None, FAKE)):
                    rc = lib.poet_groupnorm_act_bwd(t, img, row, t, img, row, FAKE, FAKE, FAKE, dx, img, row, dw, dw, 0, N, HW, C, G, 2, xd, yd, FAKE, need, None)
                    assert rc == LAUNCHED, (xd, yd, base, row, rc, lib.poet_hip_last_error())
