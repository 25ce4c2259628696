"""ncmb_cache_evict with one array for `known` (or `seen`) and the new lengths, as a loop that evicts again and again has it."""
import pytest
import torch

import helpers
import test_gpu_cache_operators as ops

capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def evict_loop(cuda, shared, lens, budget, recent, steps, nkv, grow):
    """Rows that grow by `grow` tokens between evictions; what is held after each. `shared`: which input is the array of the lengths."""
    B, hd, cap = len(lens), 16, max(lens) + grow * steps + 3
    g = torch.Generator(device="cuda").manual_seed(B + budget)
    k, v = (torch.randn(B, nkv, cap, hd, device="cuda", generator=g) for _ in range(2))
    w = torch.rand(B, nkv, cap, device="cuda", generator=g)
    pos = torch.full((B, nkv, cap), -1, dtype=torch.int32, device="cuda")
    length, seen = (torch.tensor(lens, dtype=torch.int32, device="cuda") for _ in range(2))
    known = torch.zeros(B, dtype=torch.int32, device="cuda")
    c, got = capi.KVCache.of(k, v, length), []
    for step in range(steps):
        use_known, use_seen = known.clone(), seen.clone()
        to = {"known": use_known, "seen": use_seen, None: torch.empty_like(known)}[shared]
        assert cuda.ncmb_cache_evict(c, c, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr(), use_known.data_ptr(), use_seen.data_ptr(), budget, recent,
                                     0, to.data_ptr()) == 0
        known = to.clone()
        got.append((known, pos.clone(), w.clone(), k.clone(), v.clone()))
        length.copy_(known + grow)
        seen += grow
    torch.cuda.synchronize()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("shared", ["known", "seen"])
@pytest.mark.parametrize("lens,budget,recent,nkv,grow", [
    ([300, 90, 20] * 20, 100, 16, 8, 1), ([1500, 1400], 1505, 32, 4, 1), ([30000, 12], 2000, 100, 2, 5), ([9000] * 4, 4000, 64, 8, 200)])
def test_one_array(cuda, shared, lens, budget, recent, nkv, grow):
    a, b = (evict_loop(cuda, x, lens, budget, recent, 4, nkv, grow) for x in (None, shared))
    for one, two in zip(a, b):
        for x, y in zip(one, two):
            assert torch.equal(x, y)


def test_lengths_that_share_memory_with_the_old_ones_are_refused(cuda):
    p = 1 << 22
    for at in (-4, 0, 4):
        src, dst = ops.fake_cache(), ops.fake_cache(k=1 << 23, v=1 << 24)
        assert cuda.ncmb_cache_evict(src, dst, p, 2 * p, 3 * p, 4 * p, None, 5 * p, 10, 2, 0, (1 << 19) + at) == -1
