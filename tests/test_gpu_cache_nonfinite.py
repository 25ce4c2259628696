"""Infinities, NaN and the type's extremes in keys and values that a token does not see must not reach its result
(ncmb_cache_attention, ncmb_block_attention): places without a token, siblings in a tree, tokens to come."""
import math

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


JUNK = [float("nan"), float("inf"), float("-inf"), 3.3e38, -3.3e38]


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", [(3, 2, 2, 64), (4, 12, 3, 128), (12, 14, 2, 64), (40, 14, 2, 64), (33, 8, 2, 128), (30, 5, 1, 40)])
@pytest.mark.parametrize("n", [0, 61, 700])
def test_unseen_tokens(cuda, kt, qt, T, H, nkv, hd, n):
    rng = np.random.default_rng(T + n)
    G = H // nkv
    k, v = ops.make_cache(rng, [n], n + T, nkv, hd, kt, "token", T)
    # node 0 and a chain from it; the odd ones of the rest are leaves full of junk, some places hold no token at all
    par = [-1] + [t - 2 if t % 2 == 0 else 0 for t in range(1, T)]
    for t in range(5, T, 6):
        par[t] = -3
    bad = [t for t in range(T) if t % 2 == 1]
    for i, t in enumerate(bad):
        k[0, :, n + t], v[0, :, n + t] = JUNK[i % 5], JUNK[(i + 1) % 5]
    q = torch.from_numpy(rng.standard_normal((1, T, H, hd)).astype(np.float32)).to(qt).cuda()
    out = torch.empty_like(q)
    dl, dp = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([par], dtype=torch.int32, device="cuda")
    assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, ops.KIND[qt], H, T, dp.data_ptr(), 0.0, 0, None) == 0
    torch.cuda.synchronize()
    ok = ops.visible(n, T, par)
    good = [t for t in range(T) if t not in bad]
    keep = np.array([j for j in range(n + T) if j < n or j - n not in bad])
    for h in range(nkv):
        kk, vv = k[0, h][torch.from_numpy(keep).cuda()], v[0, h][torch.from_numpy(keep).cuda()]
        want, _, rel = ops.attend64(q[0, good, h * G:(h + 1) * G], kk, vv, ok[good][:, keep], 1 / math.sqrt(hd))
        ops.check(out[0, good, h * G:(h + 1) * G], want, (rel * float(vv.float().abs().max()))[:, :, None], qt)
    for t in range(T):                                  # places without a token give zero whatever stands there
        if par[t] == -3:
            assert (out[0, t] == 0).all()


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", [(3, 2, 2, 64), (20, 14, 2, 64), (33, 8, 2, 128)])
def test_tokens_to_come(cuda, kt, qt, T, H, nkv, hd):
    """A run of tokens whose last one is junk: the ones before it are as without it."""
    rng = np.random.default_rng(T)
    G, n = H // nkv, 130
    k, v = ops.make_cache(rng, [n], n + T, nkv, hd, kt, "head", T)
    k[0, :, n + T - 1], v[0, :, n + T - 1] = float("nan"), float("inf")
    q = torch.from_numpy(rng.standard_normal((1, T, H, hd)).astype(np.float32)).to(qt).cuda()
    a, b = torch.empty_like(q), torch.empty_like(q)
    c = capi.KVCache.of(k, v, torch.tensor([n], dtype=torch.int32, device="cuda"))
    nb = -(-(n + T) // 16)
    codes, scales = torch.zeros(1, nkv, nb, hd, dtype=torch.int8, device="cuda"), torch.zeros(1, nkv, nb, device="cuda")
    assert cuda.ncmb_cache_attention(c, q.data_ptr(), H * hd, a.data_ptr(), H * hd, ops.KIND[qt], H, T, None, 0.0, 0, None) == 0
    assert cuda.ncmb_block_attention(c, q.data_ptr(), H * hd, b.data_ptr(), H * hd, ops.KIND[qt], H, T, 16, codes.data_ptr(), scales.data_ptr(), nb, 0, 1, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    ok = ops.visible(n, T, None)[:T - 1, :n + T - 1]
    for h in range(nkv):
        kk, vv = k[0, h, :n + T - 1], v[0, h, :n + T - 1]
        want, _, rel = ops.attend64(q[0, :T - 1, h * G:(h + 1) * G], kk, vv, ok, 1 / math.sqrt(hd))
        for out in (a, b):
            ops.check(out[0, :T - 1, h * G:(h + 1) * G], want, (rel * float(vv.float().abs().max()))[:, :, None], qt)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
def test_weights_of_unseen_tokens(cuda, kt, qt):
    """A NaN key that nobody sees leaves the weights of the others alone and has a weight of zero."""
    rng = np.random.default_rng(7)
    for T, H, nkv in ((3, 2, 2), (40, 14, 2)):
        n, hd, G = 90, 64, H // nkv
        k, v = ops.make_cache(rng, [n], n + T, nkv, hd, kt, "token", T)
        par = [-1, -2] + list(range(1, T - 1))
        par[2] = 0
        k[0, :, n + 1], v[0, :, n + 1] = float("nan"), float("nan")
        q = torch.from_numpy(rng.standard_normal((1, T, H, hd)).astype(np.float32)).to(qt).cuda()
        out, w = torch.empty_like(q), torch.zeros(1, nkv, n + T, device="cuda")
        dl, dp = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([par], dtype=torch.int32, device="cuda")
        assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, ops.KIND[qt], H, T, dp.data_ptr(), 0.0, 0, w.data_ptr()) == 0
        torch.cuda.synchronize()
        keep = [j for j in range(n + T) if j != n + 1]
        ok = ops.visible(n, T, par)[:, keep]
        for h in range(nkv):
            _, p, rel = ops.attend64(q[0, :, h * G:(h + 1) * G], k[0, h, keep], v[0, h, keep], ok, 1 / 8)
            got = w[0, h].double().cpu().numpy()
            assert got[n + 1] == 0
            assert (np.abs(got[keep] - p.sum((0, 1))) <= (p * rel[:, :, None]).sum((0, 1)) + 2.0 ** -22 * p.sum((0, 1)) + 1e-30).all()
