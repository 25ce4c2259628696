"""Arrays of a selection or reordering that share memory in a way in which one group's, or one row's, results would be another's inputs are refused."""
import pytest

import helpers
from test_paged_refusals import P, cache, reorder, select

capi = helpers.capi


@pytest.fixture(scope="module")
def lib():
    return capi.NcmLib(helpers.CUDA_LIB)


# (4 rows, 8 entries a row, 100 pages)
@pytest.mark.parametrize("bad", [dict(len_dst=P), dict(len_dst=P + 12), dict(table_dst=P - 124), dict(refs=P - 396), dict(refs=3 * P + 124), dict(refs=4 * P), dict(len_dst=3 * P + 64),
                                 dict(table_dst=4 * P - 124), dict(len_dst=5 * P + 124), dict(refs=5 * P - 396), dict(refs=6 * P + 12)])
def test_reorder(lib, bad):
    assert reorder(lib, **bad) == -1


# (2 groups of 4 beams, 8 continuations, 1000 words)
@pytest.mark.parametrize("bad", [dict(scores_out=2 * P), dict(scores_out=2 * P + 28), dict(scores_out=2 * P - 60), dict(parents=2 * P), dict(tokens=2 * P), dict(done_out=2 * P),
                                 dict(n_out=4, scores_out=2 * P + 4), dict(n_out=4, parents=2 * P), dict(done=7 * P, eos=3, done_out=7 * P), dict(done=7 * P, eos=3, n_out=4, done_out=7 * P + 4),
                                 dict(done=7 * P, eos=3, scores_out=7 * P), dict(parents=3 * P + 60), dict(tokens=4 * P), dict(done_out=5 * P), dict(scores_out=P), dict(tokens=P + 31996)])
def test_select(lib, bad):
    assert select(lib, **bad) == -1
