"""ncmb_cache_attention where a call takes several launches (the scores that weights are formed from would pass 2 GB), and over caches whose offsets
pass 32 bits, with either kind of tiles. Bounds are test_gpu_cache_operators.py's."""
import numpy as np
import pytest
import torch

import helpers
import test_gpu_cache_operators as ops

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module", params=[1, 2])
def cuda(request):
    lib = capi.NcmLib(helpers.CUDA_LIB)
    lib.ncmb_set_cache_variant(request.param)
    yield lib
    lib.ncmb_set_cache_variant(0)
    assert lib.ncmb_gemm_tc_check() == 0


@pytest.mark.parametrize("qt", [torch.float32, torch.bfloat16])
def test_several_launches(cuda, qt):
    """205 MB of scores a row: 10 rows a launch, the last one not full."""
    lens = [300, 0, 57, 128, 700, 1, 90, 400, 15, 16, 333, 260, 0, 77]
    ops.run_attention(cuda, 3, lens, 64, 4, 1, 8, torch.bfloat16, qt, "head", True, True, cap=200000, max_len=700)


@pytest.mark.parametrize("T,H", [(1, 4), (10, 14), (24, 14)])
@pytest.mark.parametrize("apart", ["rows", "tokens", "heads"])
def test_offsets_beyond_32_bits(cuda, T, H, apart):
    nkv, hd, n, cap = 2, 64, 160, 200
    far = (1 << 31) + 4096
    rows, strides = {"rows": (2, (far, hd, 2 * nkv * hd, 1)), "tokens": (1, (0, hd, 1 << 24, 1)), "heads": (1, (0, far, 2 * hd, 1))}[apart]
    if rows == 1:
        strides = (cap * 2 * nkv * hd,) + strides[1:]
    last = sum(s * (x - 1) for s, x in zip(strides, (rows, nkv, cap, hd)))
    at_v = nkv * hd if apart != "heads" else hd
    rng = np.random.default_rng(T)
    buf = torch.empty(last + at_v + 8, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.as_strided(buf, (rows, nkv, cap, hd), strides, at) for at in (0, at_v))
    for x in (k, v):
        x.copy_(torch.from_numpy(rng.standard_normal((rows, nkv, cap, hd)).astype(np.float32)))
    q = torch.from_numpy(rng.standard_normal((rows, T, H, hd)).astype(np.float32)).cuda()
    out, lens = torch.empty_like(q), [n, n + 9][:rows]
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, T, None, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    G = H // nkv
    for b, m in enumerate(lens):
        for h in range(nkv):
            want, _, rel = ops.attend64(q[b, :, h * G:(h + 1) * G], k[b, h, :m + T], v[b, h, :m + T], ops.visible(m, T, None), hd ** -0.5)
            ops.check(out[b, :, h * G:(h + 1) * G], want, (rel * float(v[b, h, :m + T].float().abs().max()))[:, :, None], torch.float32)
