"""What attention to an fp32 cache loses of a value: a query that sees one key alone gets that key's value, which the kernels hold as two TF32 terms.

The terms are within 2^-23 of the value; the tensor core adds them up and keeps 24 bits of the sum, cut off: another 2^-23 at most."""
import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32 = torch.float32


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def values(rng, *shape):
    """Significands of all kinds, a few powers of two apart"""
    return torch.from_numpy(np.ldexp(rng.uniform(1, 2, shape), rng.integers(-3, 4, shape)).astype(np.float32) * rng.choice([-1, 1], shape).astype(np.float32)).cuda()


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("H,nkv,hd", [(4, 4, 64), (8, 1, 128), (32, 2, 64), (16, 1, 128)])          # tiles of 8 rows, of 16
def test_a_value_comes_back_in_22_bits(cuda, paged, H, nkv, hd):
    rng = np.random.default_rng(H + hd)
    rows = 60
    k, v, q = values(rng, rows, nkv, 16, hd), values(rng, rows, nkv, 16, hd), values(rng, rows, H, hd)
    out = torch.empty_like(q)
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    if paged:
        c = capi.PagedCache.of(k, v, torch.arange(rows, dtype=torch.int32, device="cuda")[:, None], lens)
        assert cuda.ncmb_paged_attention(c, q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, 1, None, 0.0, 0) == 0
    else:
        assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, lens), q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, 1, None, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    want = v[:, :, 0].double().repeat_interleave(H // nkv, 1)
    assert ((out.double() - want).abs() <= 2.0 ** -22 * want.abs()).all(), ((out.double() - want).abs() / want.abs()).max().log2()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "payload", "negative"])
def test_what_is_not_a_number_is_not_lost(cuda, bad):
    """A NaN of any bits among a key, a value or a query that is seen gives a NaN; an infinite value something that is not finite."""
    rng = np.random.default_rng(3)
    hd, n = 64, 40
    word = {"payload": 0x7f800001, "negative": -1}.get(bad)
    bad = np.array([word], np.int64).astype(np.int32).view(np.float32)[0] if word is not None else np.float32(bad)
    for H in (4, 12):                                           # tiles of 8 rows, of 16
        for where in ("key", "value", "query"):
            k, v, q = values(rng, 4, 1, 16, hd), values(rng, 4, 1, 16, hd), values(rng, 1, H, hd)
            {"key": k[1, 0, 3], "value": v[1, 0, 3], "query": q[0, 2]}[where][17] = torch.from_numpy(np.array([bad]))[0].cuda()
            if np.isinf(bad) and where != "value":
                continue                                        # a score of infinity: what comes of it is open
            out = torch.zeros_like(q)
            c = capi.PagedCache.of(k, v, torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda"))
            assert cuda.ncmb_paged_attention(c, q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, 1, None, 0.0, 0) == 0
            torch.cuda.synchronize()
            hit = torch.zeros_like(out, dtype=torch.bool)
            if where == "value":
                hit[..., 17] = True
            elif where == "key":
                hit[:] = True
            else:
                hit[0, 2] = True
            if np.isnan(bad):
                assert torch.isnan(out[hit]).all()
            else:
                assert not torch.isfinite(out[hit]).any()


@pytest.mark.parametrize("H", [4, 16])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_are_not_short(cuda, H, hd):
    """A score whose products are all positive, read off the probability of a key of zeros beside it: exp(-score). The tensor core cuts its accumulator off
    after each product of eight dims, on the average by half a last place, 2^-24 of what it holds at most; two accumulators take turns, so each is cut n =
    hd / 16 times, at 1 / n, 2 / n ... of what it comes to: together short by (n + 1) / 2 2^-24 of the score on the average. Everything else (pairs 2^-23,
    the scaled score 2^-24, an exponential 2^-22 of itself, a fortieth of that of the score) goes either way: 1e-8 of the score for 256 means or more."""
    rng = np.random.default_rng(hd + H)
    rows, scale = 64, 40.0 / hd
    k, v = torch.zeros(rows, 1, 16, hd, device="cuda"), torch.zeros(rows, 1, 16, hd, device="cuda")
    k[:, 0, 1] = torch.from_numpy(rng.uniform(0.5, 1.5, (rows, hd)).astype(np.float32)).cuda()
    v[:, 0, 0] = 1.0
    q = torch.from_numpy(rng.uniform(0.5, 1.5, (rows, H, hd)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    c = capi.PagedCache.of(k, v, torch.arange(rows, dtype=torch.int32, device="cuda")[:, None], torch.ones(rows, dtype=torch.int32, device="cuda"))
    assert cuda.ncmb_paged_attention(c, q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, 1, None, scale, 0) == 0
    torch.cuda.synchronize()
    c2 = float(np.float32(scale) * np.float32(1.44269504))
    score = (q.double() * k[:, 0, 1].double()[:, None]).sum(-1) * c2
    short = ((torch.log2(out[..., 0].double()) + torch.log2(1 + torch.exp2(-score)) + score) / score).mean().item()
    assert -1e-8 <= short <= (hd / 16 + 1) / 2 * 2.0 ** -24 + 1e-8, short / 2.0 ** -24
