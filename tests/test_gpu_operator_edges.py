"""The token-mixer operators where their inner workings could give way: rows that land while others are read.

The bounds are those of test_gpu_operators.py.  2^-25 is half of fp16's smallest number.
"""

import pytest
import torch

from test_gpu_operators import F, UNIT, close, norm64, norm_inputs  # noqa: F401

pytestmark = pytest.mark.gpu

HALF_FLOOR = 2.0 ** -25


RINGS = [
    # rows enough for every team to fill each of its stages again; one to sixteen warps a row, with and without sums
    (torch.float32, (5453, 2048), None, True, True, True),
    (torch.float32, (2, 9000, 384), (2, 9000, 384), True, True, True),
    (torch.float32, (20000, 1024), None, False, False, False),
    (torch.float32, (3000, 8192), None, True, False, True),
    (torch.bfloat16, (4, 10000, 512), (4, 1, 512), True, True, True),
    (torch.float16, (6000, 4096), None, False, True, False),
]


@pytest.mark.parametrize("case", RINGS, ids=str)
def test_rows_keep_their_values_while_the_next_ones_land(F, case):  # noqa: F811
    """Stages of the rings are filled again only when they have been read: the same bits time after time, and the formula's values."""
    x, y, wp, wn, gate, s, gu, gn = norm_inputs(case)
    first = None
    for _ in range(25):
        got = []
        for save in ("full", "int8"):
            u, n, saved = F.gated_residual_norm(x, y, post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s, save=save)
            got += [u, n, *F.gated_residual_norm_backward(gu, None if wn is None else gn, saved)]
        if first is None:
            first = got
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(first, got))
    u, n = first[:2]
    e, e32 = UNIT[x.dtype], (x.shape[-1] + 16) * UNIT[torch.float32]
    exp, maj = norm64(x, y, wp, wn, gate, s, 1e-6)["u"]
    floor = HALF_FLOOR if x.dtype == torch.float16 else 0.0
    close(u, exp, e * exp.abs() + 2 * e32 * maj + floor, "u")
    if wn is not None:
        U = u.double()
        N = wn.double() * U / torch.sqrt((U * U).mean(-1, keepdim=True) + 1e-6)
        close(n, N, (e + e32) * N.abs() + floor + 1e-30, "n")
    F.check_operators()
