"""Sines near half a turn, where an angle's rounding shows: a pair (1, 0) comes out as (cos, sin).

The angle is |position| 1e-16 turns off at most for a frequency of a radian, here up to 4.2 times that; a sine 2 ulp of itself; what is added for the part of the angle that fp32 leaves, 9.4e-8 radians at most, is off
by 2^-22 of itself and its square: 1e-13 in all."""
import numpy as np
import pytest
import torch

import helpers
from test_gpu_rope import call

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


@pytest.mark.parametrize("layout", [capi.ROPE_HALVES, capi.ROPE_PAIRS])
@pytest.mark.parametrize("dims", [64, 50])
def test_sines_near_half_a_turn(cuda, layout, dims):
    rng = np.random.default_rng(dims)
    n = dims // 2
    turns = 0.5 + rng.choice([-1, 1], n) * 10.0 ** rng.uniform(-7, -1, n)
    r = capi.Rope(dims, layout, 1.0)
    r.turns[:n] = turns.tolist()
    pos = np.array([[1, 3, -1, 1001, -77777, 2 ** 20 + 1]])
    x = torch.zeros(1, pos.size, 2, 64, device="cuda")
    x[..., :n] = 1.0
    if layout == capi.ROPE_PAIRS:
        x.zero_()
        x[..., :dims:2] = 1.0
    y = torch.empty_like(x)
    for inverse in (0, 1):
        assert call(cuda, r, x, y, torch.from_numpy(pos.astype(np.int32)).cuda(), inverse) == 0
        torch.cuda.synchronize()
        got = (y[0, :, :, 1:dims:2] if layout == capi.ROPE_PAIRS else y[0, :, :, n:dims]).double().cpu().numpy()
        # the whole part of the turns first, in integers of 2^-53 turns: nothing of the product is lost
        units = np.array([[int(p) * int(t * 2.0 ** 53) for t in turns] for p in pos[0]], dtype=object)
        left = np.array([[((u + 2 ** 52) % 2 ** 53) - 2 ** 52 for u in row] for row in units], dtype=np.float64) * 2.0 ** -53
        want = np.sin(2 * np.pi * left)[:, None] * (-1 if inverse else 1)
        bound = 2.0 ** -22 * np.abs(want) + 2 * np.pi * 1e-16 * np.abs(pos[0])[:, None, None] * 4.2 + 1e-13
        assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()
