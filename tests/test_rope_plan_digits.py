"""A plan's turns, and the products with positions that the kernels form in 64 bits, against 50 digits.

A frequency is theta^-x, x = 2 i / dims. x is off by 2^-53 of itself, so the power by x ln(theta) 2^-53; theta's scaling, the power, the division by 2 pi
and the product with a position add 5 roundings of 2^-53. So a product is off by (5 + y) e^-y 2^-53 |position| / 2 pi with y = x ln(theta), which is
largest at y = 0: 8.9e-17 |position|. The header says 1e-16."""
from decimal import Decimal, getcontext

import pytest

import helpers

capi = helpers.capi
getcontext().prec = 50
PI = Decimal("3.14159265358979323846264338327950288419716939937510582")


@pytest.fixture(scope="module")
def lib():
    return capi.NcmLib(helpers.CUDA_LIB)


def turns(dims, theta, scaling, factor, trained, low, high):
    theta, factor = Decimal(theta), Decimal(factor)
    if scaling == capi.ROPE_BASE and dims > 2:
        theta *= (factor.ln() * dims / (dims - 2)).exp()
    for i in range(dims // 2):
        f = (theta.ln() * -2 * i / dims).exp() / (2 * PI)
        if scaling == capi.ROPE_LINEAR:
            f /= factor
        if scaling == capi.ROPE_PARTS:
            g = min(Decimal(1), max(Decimal(0), (Decimal(trained) * f - Decimal(low)) / (Decimal(high) - Decimal(low))))
            f *= g + (1 - g) / factor
        yield f


@pytest.mark.parametrize("scaling", [capi.ROPE_PLAIN, capi.ROPE_LINEAR, capi.ROPE_BASE])
@pytest.mark.parametrize("dims,theta", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (256, 1000000.0), (50, 1000000.0)])
def test_products(lib, scaling, dims, theta):
    r = capi.Rope()
    assert lib.ncmb_rope_plan(r, dims, 0, theta, scaling, 8.0, 0.0, 0.0, 0.0, 1.0) == 0
    for i, f in enumerate(turns(dims, theta, scaling, 8.0, 0.0, 0.0, 0.0)):
        for pos in (1, 4095, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31):
            assert abs(Decimal(float(pos) * r.turns[i]) - pos * f) <= abs(pos) * Decimal("1e-16")


def test_parts(lib):
    """The ramp adds to a frequency's relative error a few roundings of turns in the trained context, at most `high` of them: 2^-50 of the frequency."""
    r = capi.Rope()
    assert lib.ncmb_rope_plan(r, 128, 1, 10000.0, capi.ROPE_PARTS, 4.0, 8192.0, 1.0, 4.0, 1.1386) == 0
    for i, f in enumerate(turns(128, 10000.0, capi.ROPE_PARTS, 4.0, 8192.0, 1.0, 4.0)):
        assert abs(Decimal(r.turns[i]) - f) <= Decimal("1e-16")
