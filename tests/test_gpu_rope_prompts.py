"""Rotation of so many tokens that a CTA has several, up to as many as it takes: rows that begin and end inside a CTA, a last CTA with fewer.
Bounds: those of test_gpu_rope.py."""
import numpy as np
import pytest
import torch

import helpers
from test_gpu_rope import BF16, F32, HALF, KIND, PARTS, call, make_plan, turned
from test_rope_shares import rope_launch

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


@pytest.fixture(scope="module")
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def within(got, want, bound, dt):
    return np.abs(got.double().cpu().numpy() - want) <= bound + HALF[dt] * np.abs(want) * (1 + 2.0 ** -7) + 1e-37


# layout, heads, head dim, dims, tokens a CTA (of fp32; of bf16), rows
ROTATIONS = [(0, 3, 64, 64, (32, 32), 3), (0, 5, 64, 32, (25, 32), 1), (1, 3, 64, 64, (32, 32), 7), (1, 2, 72, 24, (32, 32), 5), (1, 7, 80, 50, (14, 28), 2), (0, 40, 128, 128, (1, 3), 4),
             (0, 4, 128, 50, (16, 16), 3), (0, 9, 128, 50, (7, 14), 1), (0, 3, 128, 6, (16, 16), 600), (0, 12, 64, 36, (10, 16), 2), (0, 2, 16, 12, (16, 16), 9),
             (0, 2, 256, 250, (15, 16), 3), (0, 4, 256, 250, (8, 15), 2), (0, 70, 256, 242, (1, 1), 2)]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("case", ROTATIONS)
def test_rotation(cuda, sms, dt, case):
    layout, H, hd, dims, most, rows = case
    most = most[dt == BF16]
    T = (4 * sms * most + 17) // rows + 1
    per, _, _ = rope_launch(layout == capi.ROPE_HALVES, dims, hd, H, rows * T, 4 if dt == F32 else 2, sms)
    assert per == most and (rows * T % per or per == 1 or rows > 1)
    rng = np.random.default_rng(dims + H)
    r = make_plan(cuda, dims, layout, **PARTS)
    x = torch.from_numpy(rng.standard_normal((rows, T, H + 1, hd)).astype(np.float32)).to(dt).cuda()[:, :, :H]
    pos = rng.integers(0, 100000, (rows, T))
    dpos, x64 = torch.from_numpy(pos.astype(np.int32)).cuda(), x.double().cpu().numpy()
    for inverse in (0, 1):
        whole = torch.full((rows, T, H + 1, hd), 7.0, dtype=dt, device="cuda")
        y = whole[:, :, :H]
        assert call(cuda, r, x, y, dpos, inverse) == 0
        want, bound = turned(x64, pos, r, inverse)
        assert within(y, want, bound, dt).all() and (whole[:, :, H] == 7).all()
        z = x.clone()                                           # in place: only the dims that turn are moved
        assert call(cuda, r, z, z, dpos, inverse) == 0
        assert torch.equal(z, y)
        head_major = torch.full((rows, H, T, hd), float("nan"), dtype=dt, device="cuda")
        assert call(cuda, r, x, head_major.transpose(1, 2), dpos, inverse) == 0
        assert torch.equal(head_major.transpose(1, 2), y)
    want, bound = turned(x64, np.broadcast_to(np.arange(T), (rows, T)), r)
    assert call(cuda, r, x, y, None) == 0
    assert within(y, want, bound, dt).all()
