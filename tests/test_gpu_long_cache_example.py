"""examples/long_cache.py: trees give the text that single steps give, in no more steps; the budget is held."""
import importlib.util
import os

import pytest

import helpers

pytestmark = pytest.mark.gpu


def test_four_ways_to_decode():
    spec = importlib.util.spec_from_file_location("long_cache", os.path.join(helpers.ROOT, "examples", "long_cache.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    got = ex.run(prompt=1500, new=24)
    ref, steps, held = got["one_by_one"]
    assert len(ref) == 24 and held == 1524
    assert got["trees"][0] == ref and got["trees"][1] <= steps
    assert len(got["budget"][0]) == 24 and got["budget"][2] == ex.BUDGET
    assert len(got["blocks"][0]) == 24
    small = ex.run(prompt=700, new=8)               # as many blocks as the row has, so block attention is attention
    assert small["blocks"][0] == small["one_by_one"][0]
