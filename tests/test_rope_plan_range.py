"""Plans whose magnitude or frequencies the library cannot hold are refused; a plan that is refused stays as it was."""
import math

import pytest

import helpers

capi = helpers.capi


@pytest.fixture(scope="module")
def lib():
    return capi.NcmLib(helpers.CUDA_LIB)


def plan(lib, r, dims=64, theta=10000.0, scaling=capi.ROPE_PLAIN, factor=1.0, magnitude=1.0):
    return lib.ncmb_rope_plan(r, dims, capi.ROPE_HALVES, theta, scaling, factor, 0.0, 0.0, 0.0, magnitude)


@pytest.mark.parametrize("bad", [dict(magnitude=1e39), dict(magnitude=-3.5e38), dict(scaling=capi.ROPE_LINEAR, factor=1e-309, theta=1e-10), dict(theta=5e-324, scaling=capi.ROPE_LINEAR, factor=1e-10),
                                 dict(dims=63), dict(magnitude=math.nan)])
def test_refused(lib, bad):
    r = capi.Rope()
    assert plan(lib, r) == 0
    before = bytes(r)
    assert plan(lib, r, **bad) == -1 and bytes(r) == before


def test_the_ends_are_taken(lib):
    for kw in (dict(magnitude=3.4e38), dict(magnitude=-3.4e38), dict(magnitude=0.0), dict(theta=1e-300, dims=256), dict(theta=1e300, scaling=capi.ROPE_BASE, factor=1e300)):
        r = capi.Rope()
        assert plan(lib, r, **kw) == 0 and all(math.isfinite(t) for t in r.turns) and math.isfinite(r.magnitude)
