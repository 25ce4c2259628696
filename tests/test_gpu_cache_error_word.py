"""ncmb_cache_attention on wide tiles when the word of the bounded waits is set: the call ends, the word is reported, nothing is read from
what earlier calls left in the scratch memory, and the next call is right."""
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
    lib = capi.NcmLib(helpers.CUDA_LIB)
    yield lib
    lib.ncmb_set_cache_variant(0)
    lib.ncmb_gemm_tc_check()


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("lens,T,H,nkv", [([3000, 17], 40, 14, 2), ([9001], 64, 4, 1)])
def test_a_call_that_finds_it_set(cuda, kt, qt, weights, lens, T, H, nkv):
    hd, B = 64, len(lens)
    cuda.ncmb_set_cache_variant(1)                      # scratch: scores and partial results where the wide call's ranges will stand
    ops.run_attention(cuda, 1, [5000, 3000], 33, 14, 2, 64, BF16, F32, "token", True, True)
    ops.run_attention(cuda, 2, [12000], 40, 14, 2, 64, BF16, F32, "token", False, False)
    cuda.ncmb_set_cache_variant(2)
    rng = np.random.default_rng(T)
    k, v = ops.make_cache(rng, lens, max(lens) + T, nkv, hd, kt, "token", T)
    q = torch.from_numpy(rng.standard_normal((B, T, H, hd)).astype(np.float32)).to(qt).cuda()
    out = torch.full_like(q, 5.0)
    w = torch.full((B, nkv, max(lens) + T), 5.0, device="cuda") if weights else None
    c = capi.KVCache.of(k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert cuda.ncmb_gemm_tc_check() == 0
    cuda.ncmb_gemm_tc_raise(47)
    assert cuda.ncmb_cache_attention(c, q.data_ptr(), H * hd, out.data_ptr(), H * hd, ops.KIND[qt], H, T, None, 0.0, 0, w.data_ptr() if weights else None) == 0
    torch.cuda.synchronize()
    assert (out == 5.0).all() and (w is None or (w == 5.0).all())
    assert cuda.ncmb_gemm_tc_check() == 47
    ops.run_attention(cuda, 3, lens, T, H, nkv, hd, kt, qt, "token", True, weights)
    assert cuda.ncmb_gemm_tc_check() == 0
