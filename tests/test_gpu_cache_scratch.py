"""ncmb_cache_attention's scratch memory holds what CTAs share, not something for every tile of queries: a call of many rows and new
tokens on a stream that has made none takes some MB, and its results are right."""
import numpy as np
import pytest
import torch

import helpers
import test_gpu_cache_operators as ops
import test_gpu_cache_streams as streams

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    lib = capi.NcmLib(helpers.CUDA_LIB)
    yield lib
    torch.cuda.synchronize()
    lib.ncmb_set_stream(None)
    lib.ncmb_set_cache_variant(0)


@pytest.mark.parametrize("variant", [1, 2])
def test_many_query_tiles(cuda, variant):
    B, T, H, nkv, hd, n = 64, 256, 32, 8, 64, 50
    rng = np.random.default_rng(variant)
    k, v = ops.make_cache(rng, [n - b % 3 for b in range(B)], n + T, nkv, hd, torch.bfloat16, "head", T)
    q = torch.randn(B, T, H, hd, device="cuda")
    out = torch.empty_like(q)
    lens = torch.tensor([n - b % 3 for b in range(B)], dtype=torch.int32, device="cuda")
    c = capi.KVCache.of(k, v, lens)
    cuda.ncmb_set_cache_variant(variant)
    call = lambda rows: cuda.ncmb_cache_attention(rows, q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, T, None, 0.0, 0, None)
    few = capi.KVCache.of(k[:1], v[:1], lens[:1])
    assert call(few) == 0                               # what the first launch of a kernel takes is taken
    s = torch.cuda.Stream(priority=-1)
    with streams.on(cuda, s):
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        assert call(c) == 0
        torch.cuda.synchronize()
        assert free - torch.cuda.mem_get_info()[0] <= 40 << 20
    G = H // nkv
    for b, h in ((0, 0), (37, 5), (63, 7)):
        m = n - b % 3
        want, _, rel = ops.attend64(q[b, :, h * G:(h + 1) * G], k[b, h, :m + T], v[b, h, :m + T], ops.visible(m, T, None), hd ** -0.5)
        ops.check(out[b, :, h * G:(h + 1) * G], want, (rel * float(v[b, h, :m + T].float().abs().max()))[:, :, None], torch.float32)
