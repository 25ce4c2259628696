"""ncmb_cache_evict where more tokens are `recent` than the budget holds: the latest ones in the text stay."""
import numpy as np
import pytest
import torch

import helpers
import test_gpu_cache_operators as ops

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens,budget,recent,known", [
    ([1000, 900, 300, 2], 300, 5000, 0), ([1000, 900, 301], 300, 301, 300), ([65, 64, 1], 64, 65, 64), ([2049, 2056], 2048, 2 ** 31 - 1, 2048),
    ([20000, 70], 3000, 4000, 0), ([20000, 9999], 3000, 20000, 1500), ([70001], 512, 600, 0)])
def test_places_by_the_definition(cuda, monkeypatch, lens, budget, recent, known, inplace):
    """The latest min(recent, budget) places, then weights: the reference's order with the window cut to the budget."""
    ref = ops.evict_ref
    monkeypatch.setattr(ops, "evict_ref", lambda n, b, r, *rest: ref(n, b, min(r, b), *rest))
    ops.run_evict(cuda, budget, lens, budget, recent, known, 2, 16, BF16, "token", inplace, "heavy")


@pytest.mark.parametrize("budget,prompt", [(64, 200), (64, 65), (1000, 9000)])
def test_a_sliding_window(cuda, budget, prompt):
    """A prompt is cut, then one token comes and one goes: the last `budget` places are held, the new one among them."""
    nkv, hd, cap = 2, 16, prompt + 8
    g = torch.Generator(device="cuda").manual_seed(budget)
    k = torch.randn(1, nkv, cap, hd, device="cuda", generator=g)
    v = torch.randn(1, nkv, cap, hd, device="cuda", generator=g)
    w = torch.rand(1, nkv, cap, device="cuda", generator=g)
    pos = torch.full((1, nkv, cap), -1, dtype=torch.int32, device="cuda")
    n, known, seen = prompt, 0, prompt
    for step in range(6):
        length, dk, ds = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (n, known, seen))
        left = torch.zeros(1, dtype=torch.int32, device="cuda")
        c = capi.KVCache.of(k, v, length)
        assert cuda.ncmb_cache_evict(c, c, w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr(), dk.data_ptr(), ds.data_ptr(), budget, 10 * budget, n,
                                     left.data_ptr()) == 0
        torch.cuda.synchronize()
        assert left.item() == budget
        for h in range(nkv):
            assert sorted(pos[0, h, :budget].tolist()) == list(range(seen - budget, seen))
        n, known, seen = budget + 1, budget, seen + 1
