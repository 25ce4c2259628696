"""ncmb_cache_attention: a place of the tree that holds no token has a zero result and no share of the weights, whatever the cached
tokens hold that it does not look at."""
import numpy as np
import pytest
import torch

import helpers
import test_gpu_cache_operators as ops

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module", params=[0, 1, 2])
def cuda(request):
    lib = capi.NcmLib(helpers.CUDA_LIB)
    lib.ncmb_set_cache_variant(request.param)
    yield lib
    lib.ncmb_set_cache_variant(0)
    assert lib.ncmb_gemm_tc_check() == 0


SHAPES = [(3, 2, 2, 64), (5, 14, 2, 64), (40, 14, 2, 64), (33, 8, 2, 128), (30, 5, 1, 40)]
ODD = [float("nan"), float("inf"), float("-inf")]


def attend(cuda, k, v, lens, q, par, w):
    B, T, H, hd = q.shape
    out = torch.full_like(q, 7.0)
    dl, dp = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(par, dtype=torch.int32, device="cuda")
    assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, ops.KIND[q.dtype], H, T, dp.data_ptr(), 0.0, 0,
                                     w.data_ptr() if w is not None else None) == 0
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", SHAPES)
@pytest.mark.parametrize("n", [61, 700, 9000])
def test_zero_beside_cached_infinities(cuda, kt, qt, T, H, nkv, hd, n):
    rng = np.random.default_rng(T + n)
    k, v = ops.make_cache(rng, [n, n // 2], n + T, nkv, hd, kt, "token", T)
    k[:, :, 3], v[:, :, 5], v[:, :, n // 2 - 2] = ODD[n % 3], ODD[T % 3], ODD[(n + T) % 3]
    par = [[-1] + [(t - 1 if t % 3 else -2) for t in range(1, T)] for _ in range(2)]
    q = torch.from_numpy(rng.standard_normal((2, T, H, hd)).astype(np.float32)).to(qt).cuda()
    for w in (None, torch.zeros(2, nkv, n + T, device="cuda")):
        out = attend(cuda, k, v, [n, n // 2], q, par, w)
        for b in range(2):
            for t in range(T):
                if par[b][t] == -2:
                    assert (out[b, t] == 0).all(), (b, t)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", SHAPES)
@pytest.mark.parametrize("n", [61, 9000])
def test_a_row_without_tokens_leaves_its_weights(cuda, kt, qt, T, H, nkv, hd, n):
    rng = np.random.default_rng(T + n)
    k, v = ops.make_cache(rng, [n], n + T, nkv, hd, kt, "head", T)
    for i in range(3):
        k[:, :, 7 * i], v[:, :, 7 * i + 1] = ODD[i], ODD[i]
    q = torch.from_numpy(rng.standard_normal((1, T, H, hd)).astype(np.float32)).to(qt).cuda()
    w = torch.rand(1, nkv, n + T, device="cuda")
    was = w.clone()
    out = attend(cuda, k, v, [n], q, [[-2] * T], w)
    assert (out == 0).all()
    assert torch.equal(w[:, :, :n], was[:, :, :n]) and (w[:, :, n:] == 0).all()


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", SHAPES)
def test_weights_beside_an_infinite_value(cuda, kt, qt, T, H, nkv, hd):
    """Values have no part in the weights; places without a token neither."""
    n = 300
    rng = np.random.default_rng(T)
    k, v = ops.make_cache(rng, [n], n + T, nkv, hd, kt, "token", T)
    v[:, :, 40] = float("inf")
    par = [[-1] + [(t - 1 if t % 3 else -2) for t in range(1, T)]]
    q = torch.from_numpy(rng.standard_normal((1, T, H, hd)).astype(np.float32)).to(qt).cuda()
    w = torch.zeros(1, nkv, n + T, device="cuda")
    attend(cuda, k, v, [n], q, par, w)
    G, ok = H // nkv, ops.visible(n, T, par[0])
    for h in range(nkv):
        _, p, rel = ops.attend64(q[0, :, h * G:(h + 1) * G], k[0, h], torch.zeros_like(k[0, h]), ok, hd ** -0.5)
        want = p.sum((0, 1))
        assert (np.abs(w[0, h].double().cpu().numpy() - want) <= (p * rel[:, :, None]).sum((0, 1)) + 2.0 ** -22 * want + 1e-30).all()
