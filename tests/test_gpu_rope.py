"""Rotary positions by a plan (ncmb_rope) against the formula in 64 bits.

Bound. The angle's fraction of a turn, doubled, is at most 1 and rounded to fp32: 2^-25, times pi: 1.6 * 2^-24 radians. p * turns is off by 2^-53
of itself, and a frequency of the oracle's by another 2^-51: 2 pi |p turns| 2^-50 radians at most. Cosine and sine are within 2 ulp of at most
1 (2 * 2^-24 each), the magnitude's product and its own rounding add 2 * 2^-24, the two products and their sum 2 * 2^-24: with
|x1| + |x2| = a, an element is within magnitude * a * (8 * 2^-24 + 2 pi |p turns| 2^-50), and half a unit of its type."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16
KIND = {F32: capi.F32, BF16: capi.BF16}
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
PARTS = dict(scaling=capi.ROPE_PARTS, factor=4.0, trained=8192.0, low=1.0, high=4.0, magnitude=1.1386)


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def make_plan(lib, dims, layout, theta=10000.0, scaling=0, factor=1.0, trained=1.0, low=0.0, high=1.0, magnitude=1.0):
    r = capi.Rope()
    assert lib.ncmb_rope_plan(r, dims, layout, theta, scaling, factor, trained, low, high, magnitude) == 0
    return r


def turned(x, pos, r, inverse=False):
    """x float64 [...][heads][hd], pos [...] int64 -> the rotation and its bound, float64"""
    n, m = r.dims, float(np.float32(r.magnitude))
    t = pos[..., None].astype(np.float64) * np.array(r.turns[:n // 2])
    a = 2 * np.pi * (t - np.rint(t))
    c, s = (m * np.cos(a))[..., None, :], (m * np.sin(-a if inverse else a))[..., None, :]
    i = np.arange(n // 2)
    p, q = (2 * i, 2 * i + 1) if r.layout == capi.ROPE_PAIRS else (i, i + n // 2)
    y, bound = x.copy(), np.zeros_like(x)
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., q] * c + x[..., p] * s
    size = abs(m) * (np.abs(x[..., p]) + np.abs(x[..., q])) * (8 * 2.0 ** -24 + 2 * np.pi * np.abs(t)[..., None, :] * 2.0 ** -50)
    bound[..., p] = bound[..., q] = size
    return y, bound


def check(got, want, bound, dt):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound + HALF[dt] * np.abs(want) * (1 + 2.0 ** -7) + 1e-37).all(), np.abs(got - want).max()


def call(lib, r, x, y, pos, inverse=0):
    rows, T, H, hd = x.shape
    return lib.ncmb_rope(r, x.data_ptr(), capi.strides(x, 3), y.data_ptr(), capi.strides(y, 3), KIND[x.dtype], rows, T, H, hd, pos.data_ptr() if pos is not None else None, inverse)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("layout", [capi.ROPE_HALVES, capi.ROPE_PAIRS])
@pytest.mark.parametrize("rows,T,H,hd,dims", [(1, 1, 1, 8, 2), (5, 1, 18, 64, 64), (2, 37, 3, 64, 32), (1, 300, 5, 128, 128), (3, 11, 2, 128, 50), (2, 9, 7, 72, 24), (1, 5, 40, 128, 6),
                                              (1, 3, 2, 256, 256), (2, 130, 1, 80, 72), (70, 3, 9, 16, 12), (1, 2, 700, 64, 64), (4, 257, 12, 64, 36)])
def test_sizes(cuda, dt, layout, rows, T, H, hd, dims):
    rng = np.random.default_rng(rows * 1000 + T + dims)
    r = make_plan(cuda, dims, layout, **(PARTS if dims % 8 == 0 else {}))
    x = torch.from_numpy(rng.standard_normal((rows, T, H + 2, hd)).astype(np.float32)).to(dt).cuda()[:, :, 1:H + 1]     # heads among others
    pos = torch.from_numpy(rng.integers(0, 100000, (rows, T)).astype(np.int32)).cuda()
    x64 = x.double().cpu().numpy()
    for inverse in (0, 1):
        want, bound = turned(x64, pos.cpu().numpy().astype(np.int64), r, inverse)
        y = torch.full((rows, T, H, hd), float("nan"), dtype=dt, device="cuda")
        assert call(cuda, r, x, y, pos, inverse) == 0
        check(y, want, bound, dt)
        head_major = torch.full((rows, H, T, hd), float("nan"), dtype=dt, device="cuda")
        assert call(cuda, r, x, head_major.transpose(1, 2), pos, inverse) == 0
        assert torch.equal(head_major.transpose(1, 2), y)
    z = x.clone()                                                       # (contiguous) in place
    whole = torch.full((rows, T, H + 1, hd), 7.0, dtype=dt, device="cuda")
    whole[:, :, :H] = x
    assert call(cuda, r, whole[:, :, :H], whole[:, :, :H], pos, 1) == 0
    assert torch.equal(whole[:, :, :H], y) and (whole[:, :, H] == 7).all()
    want, bound = turned(x64, np.broadcast_to(np.arange(T), (rows, T)), r)
    assert call(cuda, r, z, z, None) == 0
    check(z, want, bound, dt)


@pytest.mark.parametrize("scaling", [dict(), dict(scaling=capi.ROPE_LINEAR, factor=8.0), dict(scaling=capi.ROPE_BASE, factor=8.0), PARTS])
def test_far_positions(cuda, scaling):
    """Up to both ends of 32 bits; the bound's last term says what 64-bit products leave."""
    pos = np.array([[0, 1, 4095, 131071, 1000000, 16777217, 2 ** 31 - 1, -1, -131072, -2 ** 31]])
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((1, pos.size, 4, 64)).astype(np.float32)).cuda()
    for layout in (capi.ROPE_HALVES, capi.ROPE_PAIRS):
        r = make_plan(cuda, 64, layout, theta=1000000.0, **scaling)
        y = torch.empty_like(x)
        assert call(cuda, r, x, y, torch.from_numpy(pos.astype(np.int32)).cuda()) == 0
        want, bound = turned(x.double().cpu().numpy(), pos, r)
        check(y, want, bound, F32)


@pytest.mark.parametrize("layout", [capi.ROPE_HALVES, capi.ROPE_PAIRS])
def test_gradient(cuda, layout):
    """inverse is the transpose: <g, J d> = <J^T g, d>, and J d is a difference of two calls."""
    rng = np.random.default_rng(9)
    r = make_plan(cuda, 48, layout, **PARTS)
    x, d, g = (torch.from_numpy(rng.standard_normal((2, 33, 5, 64)).astype(np.float32)).cuda() for _ in range(3))
    pos = torch.from_numpy(rng.integers(0, 5000, (2, 33)).astype(np.int32)).cuda()
    f = lambda v, inv=0: (lambda y: (call(cuda, r, v, y, pos, inv), y)[1])(torch.empty_like(v)).double()
    jd, gx = f(x + d) - f(x), f(g, 1)
    a, b = (g.double() * jd).sum().item(), (gx * d.double()).sum().item()
    size = (g.double().abs() * 4 * (x.double().abs() + d.double().abs())).sum().item()
    assert abs(a - b) <= 40 * 2.0 ** -24 * size
    # and by autograd of the formula
    want, bound = turned(g.double().cpu().numpy(), pos.cpu().numpy().astype(np.int64), r, True)
    check(f(g, 1), want, bound, F32)


def test_as_rope_apply(cuda):
    """The plan's halves are what rope_apply does with tables of the same angles."""
    T, H, hd = 29, 6, 64
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((1, H, T, hd)).astype(np.float32)).cuda()
    r = make_plan(cuda, hd, capi.ROPE_HALVES)
    a = 2 * np.pi * np.arange(T)[:, None] * np.array(r.turns[:hd // 2])
    cs, sn = (torch.from_numpy(np.tile(f(a), 2).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    y, z = torch.empty_like(x), x.clone()
    assert call(cuda, r, x.transpose(1, 2), y.transpose(1, 2), None) == 0
    cuda.rope_apply(z.data_ptr(), None, cs.data_ptr(), sn.data_ptr(), 1, H, T, hd)
    torch.cuda.synchronize()
    assert (y - z).abs().max().item() <= 8 * 2.0 ** -24 * 2 * x.abs().max().item()


def test_not_finite(cuda):
    """An infinity or NaN spoils its own pair alone."""
    r = make_plan(cuda, 32, capi.ROPE_PAIRS)
    x = torch.randn(1, 8, 3, 64, device="cuda")
    clean, y = torch.empty_like(x), torch.empty_like(x)
    assert call(cuda, r, x, clean, None) == 0
    x[0, 5, 1, 10], x[0, 2, 0, 40] = float("nan"), float("inf")
    assert call(cuda, r, x, y, None) == 0
    torch.cuda.synchronize()
    bad = ~torch.isfinite(y)
    assert bad.sum() == 3 and bad[0, 5, 1, 10:12].all() and bad[0, 2, 0, 40]
    assert torch.equal(y[~bad], clean[~bad])
