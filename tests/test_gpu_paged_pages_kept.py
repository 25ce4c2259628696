"""What becomes of pages when rows go on as others (ncmb_paged_reorder), counted, apart from any statement of the tables: pages of rows' own are
all held again as long as the tables have room for the longest row's full pages and a row's own; what has no room falls off a table's end, and `refs` tells."""
import collections

import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def rows_of(rng, groups, group, page, full, own, width):
    """Tables of rows of unequal lengths, some without a sequence: `full` full pages at most, the same for a group as far as they go, and `own` of a row's own."""
    n_full = rng.integers(0, full + 1, (groups, group))
    lens = n_full * page + rng.integers(0, page, (groups, group))
    none = rng.random((groups, group)) < 0.2
    n_full[none], lens[none] = 0, -1
    pages = iter(rng.permutation(groups * (full + group * own)))
    table = np.full((groups, group, width), -1)
    mine = np.empty((groups, group, own), int)
    for g in range(groups):
        shared = [next(pages) for _ in range(full)]
        for j in range(group):
            mine[g, j] = [next(pages) for _ in range(own)]
            table[g, j, :n_full[g, j]] = shared[:n_full[g, j]]
            table[g, j, n_full[g, j]:n_full[g, j] + own] = mine[g, j][:width - n_full[g, j]]
    return table, lens, mine


def reordered(cuda, rng, table, lens, parents, page, n_pages):
    groups, group, width = table.shape
    rows = groups * group
    k = torch.randn(n_pages, 1, page, 8, device="cuda")
    v = torch.randn_like(k)
    t, n = torch.from_numpy(table.reshape(rows, width).astype(np.int32)).cuda(), torch.from_numpy(lens.reshape(rows).astype(np.int32)).cuda()
    c = capi.PagedCache.of(k, v, t, n)
    count = collections.Counter(table[table >= 0].tolist())
    refs = torch.tensor([count[p] for p in range(n_pages)], dtype=torch.int32, device="cuda")
    t2, n2, p = torch.empty_like(t), torch.empty_like(n), torch.from_numpy(parents.reshape(rows).astype(np.int32)).cuda()
    assert cuda.ncmb_paged_reorder(c, group, p.data_ptr(), 1, 0, t2.data_ptr(), n2.data_ptr(), refs.data_ptr()) == 0
    torch.cuda.synchronize()
    after = t2.cpu().numpy().reshape(table.shape)
    held = collections.Counter(after[after >= 0].tolist())
    assert refs.tolist() == [held[p] for p in range(n_pages)]
    return after


@pytest.mark.parametrize("groups,group,page,full,own", [(1, 1, 8, 3, 2), (4, 5, 16, 4, 3), (2, 33, 8, 6, 2), (1, 256, 8, 3, 4), (30, 4, 64, 0, 2)])
def test_with_room_none_of_its_own_is_lost(cuda, groups, group, page, full, own):
    rng = np.random.default_rng(group + own)
    for seed in range(5):
        table, lens, mine = rows_of(rng, groups, group, page, full, own, full + own)
        parents = rng.integers(0, group, (groups, group))
        parents[rng.random(parents.shape) < 0.1] = -1
        after = reordered(cuda, rng, table, lens, parents, page, groups * (full + group * own))
        for g in range(groups):
            held = collections.Counter(after[g][after[g] >= 0].tolist())
            assert all(held[p] == 1 for p in mine[g].ravel())
            # full pages go on with the rows that have them
            for j in range(group):
                p = parents[g, j]
                n = lens[g, p] // page if p >= 0 and lens[g, p] > 0 else 0
                assert after[g, j, :n].tolist() == table[g, p, :n].tolist()


def test_without_room_they_fall_off_the_end(cuda):
    """A table of four entries: row 1, which had no sequence and four pages, goes on as row 0 behind two full pages, with two of its four."""
    table = np.array([[[0, 1, 2, -1], [4, 5, 6, 7]]])
    after = reordered(cuda, None, table, np.array([[16, -1]]), np.array([[0, 0]]), 8, 8)
    assert after.tolist() == [[[0, 1, 2, -1], [0, 1, 4, 5]]]
