"""Sums of exponentials of ncmb_beam_select where roundings do not average: logits that are nearly all equal, and maxima that rise from tile to tile.

Bound of log sum exp, in units of 2^-22: an exponential by the GPU 1; its argument, a rounded difference times a rounded log2 e, each to half a unit of fp32, d
(2 + 1/4) 2^-24 of itself where d, the distance below the maximum in bits, is on a weighted average of the V terms log2(V) at most: 0.6 log2(V); 32 terms
added in fp32 by 10 additions of 2^-24: 2.5; the sum scaled by a maximum that rises, once a tile of 8192 at most, 1 each time, and three times where
threads, warps and parts meet. In all (V / 8192 + 1 + 0.6 log2(V) + 7); 64-bit scores are then rounded to fp32, here near 0."""
import math

import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def bound(V):
    return (V / 8192 + 1 + 0.6 * math.log2(V) + 7) * 2.0 ** -22


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("V", [300, 50257, 151936, 1 << 20])
def test_log_sum_exp(cuda, dt, V):
    i = torch.arange(V, device="cuda")
    tops = [2.0, 5.5, 8.3, 11.1, 12.7, 14.0]
    rows = [torch.where(i == V // 2, t, 0.0) for t in tops] + [torch.zeros(V, device="cuda"), i // 8192 * 0.7, i // 8192 * 0.0703125 + (i % 8192 == 77) * 3, -(i // 8192) * 0.7, (i * 7919 % 1000) * 0.01]
    x = torch.stack([r.float() for r in rows]).to(dt)
    n = x.shape[0]
    m = x.double().amax(1, keepdim=True)
    lse = m[:, 0] + (x.double() - m).exp().sum(1).log()
    scores = (lse - m[:, 0]).float()                            # so that the best score is near 0
    out, par, tok = torch.empty(n, device="cuda"), *(torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    for groups, beams in ((n, 1), (1, n)):                      # rows in few and in many parts
        k = 1 if beams == 1 else n
        assert cuda.ncmb_beam_select(x.data_ptr(), V, capi.F32 if dt == F32 else capi.BF16, groups, beams, V, scores.data_ptr(), None, -1, k, out.data_ptr(), par.data_ptr(), tok.data_ptr(),
                                     None) == 0
        torch.cuda.synchronize()
        row = torch.arange(n, device="cuda") if beams == 1 else par.long()
        want = scores.double()[row] + (x.double()[row, tok.long()] - lse[row])
        err = (out.double() - want).abs()
        assert (err <= bound(V) + 2.0 ** -24 * want.abs()).all(), err.max()
