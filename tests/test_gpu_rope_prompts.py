"""Rotation and append of so many tokens that a CTA has several, up to as many as it takes: rows that begin and end inside a CTA, a last CTA with fewer,
tokens that are nobody's. Bounds: those of test_gpu_rope.py."""
import numpy as np
import pytest
import torch

import helpers
from test_gpu_paged_cache import Pool
from test_gpu_rope import BF16, F32, HALF, KIND, PARTS, call, make_plan, turned
from test_rope_shares import append_per, rope_launch

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


@pytest.fixture(scope="module")
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def within(got, want, bound, dt):
    return np.abs(got.double().cpu().numpy() - want) <= bound + HALF[dt] * np.abs(want) * (1 + 2.0 ** -7) + 1e-37


# layout, heads, head dim, dims, tokens a CTA (of fp32; of bf16), rows
ROTATIONS = [(0, 3, 64, 64, (32, 32), 3), (0, 5, 64, 32, (25, 32), 1), (1, 3, 64, 64, (32, 32), 7), (1, 2, 72, 24, (32, 32), 5), (1, 7, 80, 50, (14, 28), 2), (0, 40, 128, 128, (1, 3), 4),
             (0, 4, 128, 50, (16, 16), 3), (0, 9, 128, 50, (7, 14), 1), (0, 3, 128, 6, (16, 16), 600), (0, 12, 64, 36, (10, 16), 2), (0, 2, 16, 12, (16, 16), 9),
             (0, 2, 256, 250, (15, 16), 3), (0, 4, 256, 250, (8, 15), 2), (0, 70, 256, 242, (1, 1), 2)]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("case", ROTATIONS)
def test_rotation(cuda, sms, dt, case):
    layout, H, hd, dims, most, rows = case
    most = most[dt == BF16]
    T = (4 * sms * most + 17) // rows + 1
    per, _, _ = rope_launch(layout == capi.ROPE_HALVES, dims, hd, H, rows * T, 4 if dt == F32 else 2, sms)
    assert per == most and (rows * T % per or per == 1 or rows > 1)
    rng = np.random.default_rng(dims + H)
    r = make_plan(cuda, dims, layout, **PARTS)
    x = torch.from_numpy(rng.standard_normal((rows, T, H + 1, hd)).astype(np.float32)).to(dt).cuda()[:, :, :H]
    pos = rng.integers(0, 100000, (rows, T))
    dpos, x64 = torch.from_numpy(pos.astype(np.int32)).cuda(), x.double().cpu().numpy()
    for inverse in (0, 1):
        whole = torch.full((rows, T, H + 1, hd), 7.0, dtype=dt, device="cuda")
        y = whole[:, :, :H]
        assert call(cuda, r, x, y, dpos, inverse) == 0
        want, bound = turned(x64, pos, r, inverse)
        assert within(y, want, bound, dt).all() and (whole[:, :, H] == 7).all()
        z = x.clone()                                           # in place: only the dims that turn are moved
        assert call(cuda, r, z, z, dpos, inverse) == 0
        assert torch.equal(z, y)
        head_major = torch.full((rows, H, T, hd), float("nan"), dtype=dt, device="cuda")
        assert call(cuda, r, x, head_major.transpose(1, 2), dpos, inverse) == 0
        assert torch.equal(head_major.transpose(1, 2), y)
    want, bound = turned(x64, np.broadcast_to(np.arange(T), (rows, T)), r)
    assert call(cuda, r, x, y, None) == 0
    assert within(y, want, bound, dt).all()


# query heads, kv heads, head dim, dims (0: none), layout, tokens a CTA (of fp32; of bf16), rows, page
APPENDS = [(2, 1, 64, 64, 0, (32, 32), 11, 16), (2, 1, 64, 64, 1, (32, 32), 3, 64), (2, 1, 64, 0, 0, (32, 32), 40, 8), (14, 2, 64, 32, 0, (7, 14), 5, 32), (8, 2, 128, 128, 1, (5, 10), 30, 64),
           (4, 4, 64, 50, 0, (9, 9), 6, 16), (2, 1, 72, 24, 0, (28, 32), 4, 8), (2, 1, 128, 50, 0, (20, 20), 1300, 8), (3, 1, 64, 64, 0, (25, 32), 1100, 8)]


@pytest.mark.parametrize("kt,qt", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("case", APPENDS)
def test_append(cuda, sms, kt, qt, case):
    H, nkv, hd, dims, layout, most, rows, page = case
    most = most[qt == BF16]
    rng = np.random.default_rng(rows + dims)
    lead, trail = 5, 9                                          # tokens of no row, at both ends of CTAs
    share = (4 * sms * most + 100) // rows + 1
    news = [int(n) for n in share // 2 + rng.integers(0, share + 1, rows)]
    if rows > 3:
        news[2] = 0
    news[0] += max(0, 4 * sms * most - sum(news))
    lens = [int(n) for n in rng.integers(0, 3 * page, rows)]
    lens[1 % rows] = -1                                         # no sequence: its tokens go nowhere
    total = lead + sum(news) + trail
    assert append_per(layout == capi.ROPE_HALVES, dims, hd, H + 2 * nkv, total, 4 if qt == F32 else 2, sms) == most
    width = max((max(0, n) + t) // page + 1 for n, t in zip(lens, news))
    pool = Pool(rng, rows, width, page, nkv, hd, kt, ["token", "head", "gap"][rows % 3])
    pool.k.zero_(), pool.v.zero_()
    pool.len.copy_(torch.tensor(lens))
    table = pool.table.clone()
    full = rows - 1                                             # the last row's second half of pages is not there
    table[full, width // 2:] = -1
    r = make_plan(cuda, dims, layout, **PARTS) if dims else None
    x = torch.from_numpy(rng.standard_normal((total, H + 2 * nkv, hd)).astype(np.float32)).to(qt).cuda()
    start = lead + np.concatenate([[0], np.cumsum(news)])
    row = np.repeat(np.arange(rows), news)
    i = lead + np.arange(len(row))
    at = np.array(lens)[row] + i - start[row]
    here = np.array(lens)[row] >= 0
    stored = here & ~((row == full) & (at // page >= width // 2))
    for pos in (None, rng.integers(-1000, 300000, total)):
        x64 = x[lead:lead + len(row)].double().cpu().numpy()
        places = at if pos is None else pos[i]
        want, bound = turned(x64[:, :H + nkv], places, r) if dims else (x64[:, :H + nkv], np.zeros_like(x64[:, :H + nkv]))
        q_out = torch.full((total, H, hd), 5.0, dtype=qt, device="cuda")
        dstart = torch.from_numpy(start.astype(np.int32)).cuda()
        dpos = torch.from_numpy(pos.astype(np.int32)).cuda() if pos is not None else None
        es, base, ld = x.element_size(), x.data_ptr(), (H + 2 * nkv) * hd
        assert cuda.ncmb_paged_append(pool.handle(table), r, base, ld, q_out.data_ptr(), H * hd, H, base + H * hd * es, ld, base + (H + nkv) * hd * es, ld, KIND[qt], total, dstart.data_ptr(),
                                      dpos.data_ptr() if pos is not None else None) == 0
        torch.cuda.synchronize()
        q = q_out[lead:lead + len(row)]
        assert within(q, want[:, :H], bound[:, :H], qt)[here].all() and (q[torch.from_numpy(~here).cuda()] == 5).all()
        assert (q_out[:lead] == 5).all() and (q_out[lead + len(row):] == 5).all()
        p, s = (torch.from_numpy(t[stored]).cuda() for t in (pool.pages[row, at // page], at % page))
        k, v = pool.k[0][p, :, s], pool.v[0][p, :, s]
        assert within(k, want[stored, H:], bound[stored, H:], kt).all()
        assert torch.equal(v, x[lead:lead + len(row), H + nkv:][torch.from_numpy(stored).cuda()].to(kt))
        for t in (pool.k[0], pool.v[0]):                        # and nothing else was written
            t[p, :, s] = 0
            assert not t.any()


def test_many_tokens_without_starts(cuda, sms):
    """As many new tokens of every row, several a CTA: the same bits as with starts, and as a token a row at a time."""
    H, nkv, hd, page, rows = 2, 1, 64, 64, 5
    T = 4 * sms * 32 // rows + 3
    rng = np.random.default_rng(1)
    pool = Pool(rng, rows, T // page + 3, page, nkv, hd, BF16, "token")
    x = torch.randn(rows, T, H + 2 * nkv, hd, device="cuda")
    r = make_plan(cuda, hd, capi.ROPE_HALVES)
    got = []
    for kind in ("plain", "starts", "pieces"):
        pool.k.zero_(), pool.v.zero_()
        q = torch.empty(rows, T, H, hd, device="cuda")
        ld, n = (H + 2 * nkv) * hd, 3 if kind == "pieces" else 1
        for j in range(n):
            a, b = j * T // n, (j + 1) * T // n
            pool.len.fill_(70 + a)
            y, z = x[:, a:b].contiguous(), torch.empty(rows, b - a, H, hd, device="cuda")
            starts = torch.arange(0, rows * T + 1, T, dtype=torch.int32, device="cuda") if kind == "starts" else None
            p = y.data_ptr()
            assert cuda.ncmb_paged_append(pool.handle(), r, p, ld, z.data_ptr(), H * hd, H, p + H * hd * 4, ld, p + (H + nkv) * hd * 4, ld, capi.F32, rows * (b - a),
                                          starts.data_ptr() if starts is not None else None, None) == 0
            q[:, a:b] = z
        torch.cuda.synchronize()
        got.append((q, pool.k.clone(), pool.v.clone()))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
