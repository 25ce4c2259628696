"""Operators on long key/value caches (include/ncm_b200.h): attention of new and drafted tokens with its weights, eviction,
block summaries, block attention. Against plain implementations in 64 bits on the CPU; whole numbers and moved data exactly.

Bounds. A score is a sum of hd products; products are exact to 2^-21 of their size and each of at most 3 hd / 8 partial sums is
rounded or truncated at 2^-23, so |error of a score| <= E = (2^-21 + 3 hd / 8 * 2^-23) * scale * max_j sum_d |q_d k_jd|.
A probability is then off by at most (2 E + 2^-20) of itself (exponential, sum, division), a result by that share of the
largest |v|, plus half a unit in the last place of its type. Worst cases add up where real errors do not, so the 2-norm of
the errors is also held to 5e-6 of the results' (fp32), or 2^-8 (bf16)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import helpers

capi = helpers.capi
NEW = 256


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


F32, BF16 = torch.float32, torch.bfloat16
KIND = {F32: capi.F32, BF16: capi.BF16}
HALF_ULP = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def make_cache(rng, lens, cap, nkv, hd, dt, layout, extra, dev="cuda"):
    """k, v as [rows][n_kv][cap][hd] views; slots from lens[b] + extra on hold NaN, infinities and the type's extremes."""
    B = len(lens)
    full = rng.standard_normal((2, B, nkv, cap, hd)).astype(np.float32)
    junk = np.array([np.nan, np.inf, -np.inf, 3.3e38, -3.3e38], np.float32)
    for b, n in enumerate(lens):
        full[:, b, :, n + extra:] = junk[rng.integers(0, 5, (2, nkv, max(0, cap - n - extra), hd))]
    x = torch.from_numpy(full).to(dt)
    if layout == "token":
        buf = torch.empty(B, cap, 2, nkv, hd, dtype=dt, device=dev)
        k, v = (buf[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
    elif layout == "gap":               # rows, heads and tokens apart, each by a multiple of 16 bytes
        buf = torch.empty(2, B, nkv + 1, cap + 3, hd + 8, dtype=dt, device=dev)
        k, v = (buf[i, :, :nkv, :cap, :hd] for i in (0, 1))
    else:
        k, v = (torch.empty(B, nkv, cap, hd, dtype=dt, device=dev) for _ in range(2))
    k.copy_(x[0]); v.copy_(x[1])
    return k, v


def make_parents(rng, B, T):
    rows = []
    for b in range(B):
        row = []
        for t in range(T):
            x = rng.random()
            if x < 0.12:
                row.append(int(rng.choice([-2, -7, t, t + 5, 2 ** 30])))       # no token stands here
            elif x < 0.25 or t == 0:
                row.append(-1)
            else:
                row.append(int(rng.integers(max(0, t - 6), t)))
        rows.append(row)
    return rows


def visible(n, T, par):
    """[T][n + T] booleans"""
    ok = np.zeros((T, n + T), bool)
    used = [par is None or -1 <= par[t] < t for t in range(T)]
    for t in range(T):
        if not used[t]:
            continue
        ok[t, :n] = True
        at = t
        while at >= 0 and used[at]:
            ok[t, n + at] = True
            at = at - 1 if par is None else par[at]
    return ok


def attend64(q, k, v, ok, scale):
    """q [T][G][hd], k / v [m][hd], ok [T][m] -> out [T][G][hd], p [T][G][m], bound of |error| per (T, G)"""
    q, k, v = (x.double().cpu().numpy() for x in (q, k, v))
    s = np.einsum("tgd,md->tgm", q, k) * scale
    size = np.einsum("tgd,md->tgm", np.abs(q), np.abs(k)) * abs(scale)
    s = np.where(ok[:, None], s, -np.inf)
    m = s.max(-1, keepdims=True)
    e = np.where(ok[:, None], np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
    z = e.sum(-1, keepdims=True)
    p = np.divide(e, z, out=np.zeros_like(e), where=z > 0)
    hd = q.shape[-1]
    E = (2.0 ** -21 + 3 * hd / 8 * 2.0 ** -23) * np.where(ok[:, None], size, 0).max(-1)
    return np.einsum("tgm,md->tgd", p, v), p, 2 * E + 2.0 ** -20


def check(got, want, bound, dt):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    worst = bound + HALF_ULP[dt] * np.abs(want) + 1e-30
    assert (np.abs(got - want) <= worst).all(), float((np.abs(got - want) / worst).max())
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= {F32: 5e-6, BF16: 2.0 ** -8}[dt] * norm + 1e-30


def run_attention(cuda, seed, lens, T, H, nkv, hd, kt, qt, layout, tree, weights, cap=None, max_len=0, scale=0.0):
    rng = np.random.default_rng(seed)
    B, G = len(lens), H // nkv
    cap = cap or max(lens) + T + 7
    k, v = make_cache(rng, lens, cap, nkv, hd, kt, layout, T)
    ld = H * hd + 16
    q = torch.from_numpy(rng.standard_normal((B, T, ld)).astype(np.float32) * 2).to(qt).cuda()
    out = torch.full((B, T, ld), 77.0, dtype=qt, device="cuda")
    par = make_parents(rng, B, T) if tree else None
    dpar = torch.tensor(par, dtype=torch.int32, device="cuda") if tree else None
    w0 = torch.from_numpy(rng.random((B, nkv, cap)).astype(np.float32))
    w = w0.cuda() if weights else None
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cache = capi.KVCache.of(k, v, dl)
    rc = cuda.ncmb_cache_attention(cache, q.data_ptr(), ld, out.data_ptr(), ld, KIND[qt], H, T, dpar.data_ptr() if tree else None, scale, max_len,
                                   w.data_ptr() if weights else None)
    assert rc == 0
    torch.cuda.synchronize()
    assert (out[:, :, H * hd:] == 77.0).all()           # beyond the heads nothing is written
    o = out[:, :, :H * hd].view(B, T, H, hd)
    qv = q[:, :, :H * hd].view(B, T, nkv, G, hd)
    sc = scale or 1 / math.sqrt(hd)
    for b, n in enumerate(lens):
        ok = visible(n, T, par[b] if tree else None)
        for h in range(nkv):
            want, p, rel = attend64(qv[b, :, h], k[b, h, :n + T], v[b, h, :n + T], ok, sc)
            check(o[b, :, h * G:(h + 1) * G], want, (rel * float(v[b, h, :n + T].float().abs().max()))[:, :, None], qt)
            if not weights:
                continue
            shares = p.sum((0, 1))
            exp = w0[b, h].double().numpy().copy()
            exp[:n] += shares[:n]
            exp[n:n + T] = shares[n:]
            got = w[b, h].double().cpu().numpy()
            tol = (p * rel[:, :, None]).sum((0, 1)) + 2.0 ** -22 * exp[:n + T] + 1e-30
            assert (np.abs(got[:n + T] - exp[:n + T]) <= tol).all()
            assert (got[n + T:] == exp[n + T:]).all()   # beyond the tokens nothing is written
    return o


TYPES = [(F32, F32), (BF16, F32), (BF16, BF16)]


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("hd,H,nkv", [(64, 14, 2), (128, 8, 2), (64, 3, 3), (40, 10, 2), (8, 4, 1), (72, 5, 1), (128, 48, 3), (96, 1, 1)])
@pytest.mark.parametrize("T,tree", [(1, False), (1, True), (5, True), (19, True), (33, False)])
def test_attention(cuda, kt, qt, hd, H, nkv, T, tree):
    run_attention(cuda, 3 * hd + T, [0, 1, 40, 333], T, H, nkv, hd, kt, qt, ["token", "head", "gap"][(hd + T) % 3], tree, T % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("n", [0, 1, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
def test_attention_at_tile_ends(cuda, kt, qt, n):
    run_attention(cuda, n, [n, max(0, n - 1)], 3, 4, 2, 64, kt, qt, "token", True, True, cap=n + 3)
    run_attention(cuda, n, [n], 1, 4, 2, 128, kt, qt, "head", False, True, cap=n + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("T,tree", [(64, True), (100, True), (256, True), (256, False)])
def test_attention_of_large_trees(cuda, kt, qt, T, tree):
    run_attention(cuda, T, [100, 0, 517], T, 14, 2, 64, kt, qt, "token", tree, True)


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", [(1, 14, 2, 64), (1, 12, 12, 64), (24, 14, 2, 64), (16, 32, 8, 128), (1, 4, 4, 128)])
def test_attention_over_long_rows(cuda, kt, qt, T, H, nkv, hd):
    run_attention(cuda, T, [9001], T, H, nkv, hd, kt, qt, "token", T > 1, True)
    run_attention(cuda, T, [5000, 3, 12000], T, H, nkv, hd, kt, qt, "head", T > 1, False, max_len=700)    # the bound is too low


@pytest.mark.gpu
def test_attention_of_far_apart_scores(cuda):
    """Scores of hundreds: all weight on one token, others underflow."""
    for kt, qt in TYPES:
        run_attention(cuda, 5, [300, 70], 4, 6, 2, 64, kt, qt, "token", True, True, scale=4.0)
        run_attention(cuda, 6, [300, 70], 1, 6, 2, 64, kt, qt, "token", False, True, scale=-0.25)


@pytest.mark.gpu
def test_attention_beyond_32_bit_offsets(cuda):
    B, nkv, hd, n, T, H = 2, 2, 64, 70, 2, 4
    stride = (1 << 31) + 4096
    rng = np.random.default_rng(1)
    buf = torch.empty(stride + 2 * 200 * nkv * hd, dtype=BF16, device="cuda")
    k = torch.as_strided(buf, (B, nkv, 200, hd), (stride, hd, 2 * nkv * hd, 1))
    v = torch.as_strided(buf, (B, nkv, 200, hd), (stride, hd, 2 * nkv * hd, 1), nkv * hd)
    for x in (k, v):
        x.copy_(torch.from_numpy(rng.standard_normal((B, nkv, 200, hd)).astype(np.float32)))
    q = torch.from_numpy(rng.standard_normal((B, T, H, hd)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    dl = torch.tensor([n, n + 9], dtype=torch.int32, device="cuda")
    assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, capi.F32, H, T, None, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    for b, m in enumerate([n, n + 9]):
        for h in range(nkv):
            want, _, rel = attend64(q[b, :, 2 * h:2 * h + 2], k[b, h, :m + T], v[b, h, :m + T], visible(m, T, None), 1 / 8)
            check(out[b, :, 2 * h:2 * h + 2], want, (rel * 6)[:, :, None], F32)


@pytest.mark.gpu
def test_lengths_that_do_not_fit_count_as_the_nearest(cuda):
    rng = np.random.default_rng(2)
    k, v = make_cache(rng, [50, 50, 50], 50, 1, 64, F32, "token", 0)
    q = torch.from_numpy(rng.standard_normal((3, 2, 1, 64)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    dl = torch.tensor([-5, 1000, 48], dtype=torch.int32, device="cuda")
    assert cuda.ncmb_cache_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), 64, out.data_ptr(), 64, capi.F32, 1, 2, None, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    for b, n in enumerate([0, 48, 48]):
        want, _, rel = attend64(q[b], k[b, 0, :n + 2], v[b, 0, :n + 2], visible(n, 2, None), 1 / 8)
        check(out[b], want, (rel * 6)[:, :, None], F32)


@pytest.mark.gpu
def test_attention_gives_the_same_bits_again(cuda):
    a = run_attention(cuda, 11, [3000, 17], 9, 14, 2, 64, BF16, F32, "token", True, True)
    b = run_attention(cuda, 11, [3000, 17], 9, 14, 2, 64, BF16, F32, "token", True, True)
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------- eviction

def evict_ref(n, budget, recent, known, seen, w, pos):
    """(from slot of each kept slot, places) of one row and head"""
    place = [int(pos[s]) if s < known else seen - n + s for s in range(n)]
    n2 = min(n, budget)
    if n == 0:
        return [], []
    last = max(place)
    # latest tokens, weights, tokens without one that can be compared
    rank = lambda s: (0, 0.0, s) if place[s] > last - recent else (2, 0.0, s) if math.isnan(w[s]) else (1, -float(w[s]), s)
    kept = set(sorted(range(n), key=rank)[:n2])
    movers = iter([s for s in range(n2, n) if s in kept])
    src = [s if s in kept else next(movers) for s in range(n2)]
    return src, [place[s] for s in src]


def run_evict(cuda, seed, lens, budget, recent, known, nkv, hd, kt, layout, inplace, kind="heavy", max_len=0):
    rng = np.random.default_rng(seed)
    B, cap = len(lens), max(max(lens), 1) + 9
    k, v = make_cache(rng, lens, cap, nkv, hd, kt, layout, 0)
    w = np.exp(2 * rng.standard_normal((B, nkv, cap))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, (B, nkv, cap)).astype(np.float32)
        w[w == 1] = -0.0
    elif kind == "same":
        w[:] = 0.25
    elif kind == "odd":
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.1] = 1e-42
    far = 5 * cap
    pos = np.stack([rng.permutation(far)[:cap] for _ in range(B * nkv)]).reshape(B, nkv, cap).astype(np.int32)
    kn = [min(known, n) for n in lens]
    seen = [far + n for n in lens]
    cap2 = cap if inplace else min(budget, cap) + 2
    dw, dp = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    dl, dk, ds = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, kn, seen))
    l2 = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    k0, v0 = k.clone(), v.clone()
    if inplace:
        k2, v2, w2, p2 = k, v, dw, dp
    else:
        k2, v2 = (torch.full((B, nkv, cap2, hd), 5.0, dtype=kt, device="cuda") for _ in range(2))
        w2, p2 = torch.full((B, nkv, cap2), 5.0, device="cuda"), torch.full((B, nkv, cap2), 5, dtype=torch.int32, device="cuda")
    b2 = (w2.clone(), p2.clone(), k2.clone(), v2.clone())
    src = capi.KVCache.of(k, v, dl)
    dst = src if inplace else capi.KVCache.of(k2, v2, dl)
    assert cuda.ncmb_cache_evict(src, dst, dw.data_ptr(), w2.data_ptr(), dp.data_ptr(), p2.data_ptr(), dk.data_ptr() if known else None, ds.data_ptr(),
                                 budget, recent, max_len, l2.data_ptr()) == 0
    torch.cuda.synchronize()
    assert l2.tolist() == [min(n, budget) for n in lens]
    bits = lambda t: t.contiguous().view(torch.int32 if t.dtype != BF16 else torch.int16).cpu().numpy()
    for b, n in enumerate(lens):
        for h in range(nkv):
            at, place = evict_ref(n, budget, recent, kn[b] if known else 0, seen[b], w[b, h], pos[b, h])
            n2 = len(at)
            assert p2[b, h, :n2].tolist() == place
            assert (bits(w2[b, h, :n2]) == bits(torch.from_numpy(w[b, h][at]))).all()
            assert (bits(k2[b, h, :n2]) == bits(k0[b, h][at])).all()
            assert (bits(v2[b, h, :n2]) == bits(v0[b, h][at])).all()
            for x, was in zip((w2, p2, k2, v2), b2):            # beyond the kept nothing is written
                assert (bits(x[b, h, n2:]) == bits(was[b, h, n2:])).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["heavy", "ties", "same", "odd"])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens,budget,recent,known", [
    ([0, 1, 5, 64], 4, 2, 0), ([65, 64, 63, 1], 64, 0, 64), ([300, 0, 257, 999], 256, 256, 256), ([300, 20, 257, 999], 100, 7, 50),
    ([2050, 2049], 2048, 64, 2048), ([4097, 2], 1, 1, 0), ([4097, 900], 5000, 3, 0), ([1000, 900], 300, 5000, 0)])
def test_eviction(cuda, kind, inplace, lens, budget, recent, known):
    run_evict(cuda, budget, lens, budget, recent, known, 3, 64, BF16 if budget % 2 else F32, ["token", "head", "gap"][budget % 3], inplace, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kt", [(8, F32), (8, BF16), (40, BF16), (72, F32), (128, F32), (128, BF16)])
def test_eviction_of_widths(cuda, hd, kt):
    run_evict(cuda, hd, [130, 77], 60, 10, 20, 2, hd, kt, "token", False)
    run_evict(cuda, hd, [130, 77], 60, 10, 20, 2, hd, kt, "gap", True)


@pytest.mark.gpu
@pytest.mark.parametrize("n,budget,kind", [(20000, 3000, "heavy"), (20000, 9999, "ties"), (70001, 512, "same"), (70001, 40000, "odd"), (260000, 1000, "heavy")])
def test_eviction_of_long_rows(cuda, n, budget, kind):
    """Several CTAs share a row; the longest do not fit their shared memory."""
    run_evict(cuda, 1, [n], budget, 100, 0, 1, 8, BF16, "head", False, kind)
    run_evict(cuda, 2, [n, 500], budget, 100, n // 2, 1, 8, F32, "head", True, kind, max_len=300)      # the bound is too low


# ------------------------------------------------------------------------------------------- blocks

def summaries_ref(k, n, block):
    """codes [nb][hd], scales [nb] of one row and head in numpy's fp32, which rounds as the definition states"""
    nb = -(-n // block)
    x = np.zeros((nb * block, k.shape[1]), np.float32)
    x[:n] = k[:n]
    x = x.reshape(nb, block, -1)
    while x.shape[1] > 1:
        x = x[:, :x.shape[1] // 2] + x[:, x.shape[1] // 2:]
    cnt = np.minimum(block, n - np.arange(nb) * block).astype(np.float32)
    mean = x[:, 0] / cnt[:, None]
    scale = np.abs(mean).max(1) / np.float32(127)
    code = np.rint(np.divide(mean, scale[:, None], out=np.zeros_like(mean), where=scale[:, None] > 0))
    return code.astype(np.int8), scale


@pytest.mark.gpu
@pytest.mark.parametrize("kt", [F32, BF16])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [8, 40, 64, 128])
def test_summaries(cuda, kt, block, hd):
    rng = np.random.default_rng(block + hd)
    lens, nkv, new = [0, 1, 200, 517, 640], 2, 3
    cap = 700
    k, v = make_cache(rng, lens, cap, nkv, hd, kt, ["token", "head", "gap"][hd % 3], new)
    k[2, 1, :190] = 0                                   # blocks of zeros: scale 0, codes 0
    nb = -(-cap // block)
    for first in (None, [0, 0, 150, 517, 640]):
        codes = torch.full((len(lens), nkv, nb, hd), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((len(lens), nkv, nb), 99.0, device="cuda")
        dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        df = torch.tensor(first, dtype=torch.int32, device="cuda") if first else None
        assert cuda.ncmb_block_summaries(capi.KVCache.of(k, v, dl), new, df.data_ptr() if first else None, block, 0, codes.data_ptr(), scales.data_ptr()) == 0
        torch.cuda.synchronize()
        for b, n in enumerate(lens):
            for h in range(nkv):
                c, s = summaries_ref(k[b, h].float().cpu().numpy(), n + new, block)
                lo = (first[b] if first else 0) // block
                got_c, got_s = codes[b, h].cpu().numpy(), scales[b, h].cpu().numpy()
                assert (got_c[lo:len(s)] == c[lo:]).all() and (got_s[lo:len(s)] == s[lo:]).all()
                assert (got_c[:lo] == 99).all() and (got_c[len(s):] == 99).all() and (got_s[:lo] == 99).all() and (got_s[len(s):] == 99).all()


def picks_ref(q, codes, scales, cur, n_sel, n_first, n_last):
    """q [G][hd] fp32, codes [nb][hd], scales [nb]: picked blocks of 0 ... cur, ascending"""
    top = np.abs(q).max(1).astype(np.float32) / np.float32(127)
    q8 = np.rint(np.divide(q, top[:, None], out=np.zeros_like(q), where=top[:, None] > 0)).astype(np.int64)
    score = ((q8 @ codes[:cur + 1].astype(np.int64).T).astype(np.float32) * top[:, None]).max(0) * scales[:cur + 1]
    rank = sorted(range(cur + 1), key=lambda i: (0 if i < n_first or i > cur - n_last else 1, 0.0 if i < n_first or i > cur - n_last else -score[i], i))
    return sorted(rank[:n_sel])


def run_blocks(cuda, seed, lens, T, H, nkv, hd, kt, qt, layout, block, n_sel, n_first, n_last, with_picks=True, same=False, max_len=0):
    rng = np.random.default_rng(seed)
    B, G = len(lens), H // nkv
    cap = max(lens) + T + 3
    k, v = make_cache(rng, lens, cap, nkv, hd, kt, layout, T)
    nb = -(-cap // block)
    codes = rng.integers(-127, 128, (B, nkv, nb, hd)).astype(np.int8)
    scales = (rng.random((B, nkv, nb)) * 0.01).astype(np.float32)
    if same:                                            # scores that tie
        codes[:] = codes[:, :, :1]
        scales[:] = 0.01
    dc, ds = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    q = torch.from_numpy(rng.standard_normal((B, T, H, hd)).astype(np.float32) * 2).to(qt).cuda()
    if T > 1:
        q[0, 1] = 0                                     # a query of zeros
    out = torch.full_like(q, 9.0)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    picks = torch.full((B, T, nkv, n_sel), -9, dtype=torch.int32, device="cuda")
    assert cuda.ncmb_block_attention(capi.KVCache.of(k, v, dl), q.data_ptr(), H * hd, out.data_ptr(), H * hd, KIND[qt], H, T, block, dc.data_ptr(),
                                     ds.data_ptr(), n_sel, n_first, n_last, 0.0, max_len, picks.data_ptr() if with_picks else None) == 0
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        for t in range(T):
            for h in range(nkv):
                qh = q[b, t, h * G:(h + 1) * G]
                p = picks_ref(qh.float().cpu().numpy(), codes[b, h], scales[b, h], (n + t) // block, n_sel, n_first, n_last)
                if with_picks:
                    assert picks[b, t, h].tolist() == p + [-1] * (n_sel - len(p))
                tok = np.concatenate([np.arange(i * block, (i + 1) * block) for i in p])
                tok = torch.from_numpy(tok[tok <= n + t]).cuda()
                want, _, rel = attend64(qh[None], k[b, h][tok], v[b, h][tok], np.ones((1, tok.numel()), bool), 1 / math.sqrt(hd))
                check(out[b, t, h * G:(h + 1) * G][None], want, (rel * float(v[b, h][tok].float().abs().max()))[:, :, None], qt)


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,H,nkv", [(64, 14, 2), (128, 8, 2), (40, 3, 3), (8, 20, 1)])
def test_block_attention(cuda, kt, qt, block, hd, H, nkv):
    run_blocks(cuda, hd + block, [0, block - 1, 5 * block, 1500], 3, H, nkv, hd, kt, qt, ["token", "head", "gap"][hd % 3], block, 6, 1, 2)
    run_blocks(cuda, hd + block, [1999], 1, H, nkv, hd, kt, qt, "token", block, 1, 0, 1, with_picks=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kt,qt", TYPES)
def test_block_attention_over_long_rows(cuda, kt, qt):
    run_blocks(cuda, 1, [40000, 100], 1, 14, 2, 64, kt, qt, "token", 64, 33, 1, 2)
    run_blocks(cuda, 2, [40000, 100], 2, 4, 1, 128, kt, qt, "head", 16, 100, 4, 8, max_len=50)      # the bound is too low
    run_blocks(cuda, 3, [20000, 7000], 1, 4, 1, 64, kt, qt, "token", 32, 1000, 0, 1)
    run_blocks(cuda, 4, [6000, 64], 2, 4, 2, 64, kt, qt, "token", 16, 20, 0, 1, same=True)


@pytest.mark.gpu
def test_block_attention_with_more_blocks_than_shared_memory_holds(cuda):
    run_blocks(cuda, 5, [300000], 1, 4, 1, 8, BF16, F32, "head", 16, 30, 1, 1)


@pytest.mark.gpu
def test_block_attention_over_all_blocks_is_attention(cuda):
    rng = np.random.default_rng(4)
    B, nkv, hd, n, T, H = 2, 2, 64, 500, 4, 6
    k, v = make_cache(rng, [n, n - 77], n + T, nkv, hd, F32, "token", T)
    q = torch.from_numpy(rng.standard_normal((B, T, H, hd)).astype(np.float32)).cuda()
    a, b = torch.empty_like(q), torch.empty_like(q)
    c = capi.KVCache.of(k, v, torch.tensor([n, n - 77], dtype=torch.int32, device="cuda"))
    nb = -(-(n + T) // 32)
    codes, scales = torch.zeros(B, nkv, nb, hd, dtype=torch.int8, device="cuda"), torch.zeros(B, nkv, nb, device="cuda")
    assert cuda.ncmb_block_summaries(c, T, None, 32, 0, codes.data_ptr(), scales.data_ptr()) == 0
    assert cuda.ncmb_block_attention(c, q.data_ptr(), H * hd, a.data_ptr(), H * hd, capi.F32, H, T, 32, codes.data_ptr(), scales.data_ptr(), nb, 0, 1, 0.0, 0, None) == 0
    assert cuda.ncmb_cache_attention(c, q.data_ptr(), H * hd, b.data_ptr(), H * hd, capi.F32, H, T, None, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    assert float((a - b).norm() / b.norm()) < 5e-6


# ------------------------------------------------------------------------------------------- streams, refusals

@pytest.mark.gpu
def test_calls_run_on_the_stream_that_was_set(cuda):
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    cuda.ncmb_set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            run_attention(cuda, 21, [600, 40], 6, 14, 2, 64, BF16, F32, "token", True, True)
            run_evict(cuda, 22, [600, 40], 128, 16, 0, 2, 64, BF16, "token", False)
            run_blocks(cuda, 23, [1600, 40], 2, 14, 2, 64, BF16, F32, "token", 32, 8, 1, 1)
    finally:
        torch.cuda.synchronize()
        cuda.ncmb_set_stream(None)


def fake_cache(**kw):
    a = dict(k=1 << 20, v=1 << 21, type=capi.F32, rows=2, n_kv=2, hd=64, capacity=100, row_stride=100 * 256, head_stride=64, token_stride=256, len=1 << 19)
    a.update(kw)
    return capi.KVCache(*(a[f] for f, _ in capi.KVCache._fields_))


BAD_CACHE = [dict(type=2), dict(hd=12), dict(hd=136), dict(hd=0), dict(k=None), dict(v=(1 << 21) + 4), dict(len=None), dict(rows=-1), dict(n_kv=0),
             dict(capacity=0), dict(token_stride=32), dict(token_stride=257), dict(row_stride=-4), dict(head_stride=8)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_a_cache_that_does_not_fit_is_refused(cuda, bad, capfd):
    c, good, p = fake_cache(**bad), fake_cache(), 1 << 22
    assert cuda.ncmb_cache_attention(c, p, 256, p, 256, capi.F32, 4, 1, None, 0.0, 0, None) == -1
    assert cuda.ncmb_cache_evict(c, good, p, 2 * p, p, 2 * p, None, p, 10, 2, 0, p) == -1
    assert cuda.ncmb_cache_evict(good, c, p, 2 * p, p, 2 * p, None, p, 10, 2, 0, p) == -1
    assert cuda.ncmb_block_summaries(c, 0, None, 64, 0, p, p) == -1
    assert cuda.ncmb_block_attention(c, p, 256, p, 256, capi.F32, 4, 1, 64, p, p, 8, 1, 1, 0.0, 0, None) == -1
    assert len(capfd.readouterr().err.strip().splitlines()) == 5


def test_arguments_that_do_not_fit_are_refused(cuda):
    c, p = fake_cache(), 1 << 22
    def attend(q=p, ldq=256, out=p, ldo=256, act=capi.F32, H=4, T=1, scale=0.0):
        return cuda.ncmb_cache_attention(c, q, ldq, out, ldo, act, H, T, None, scale, 0, None)
    for bad in (dict(q=None), dict(out=None), dict(q=p + 4), dict(ldq=255), dict(ldq=252), dict(ldo=258), dict(act=capi.BF16), dict(act=5), dict(H=3), dict(H=0),
                dict(T=0), dict(T=257), dict(T=101), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attend(**bad) == -1, bad
    d = fake_cache(k=1 << 23, v=1 << 24)
    def evict(src=c, dst=d, w=p, w2=2 * p, pos=3 * p, pos2=4 * p, seen=p, budget=10, recent=2, l2=p):
        return cuda.ncmb_cache_evict(src, dst, w, w2, pos, pos2, None, seen, budget, recent, 0, l2)
    for bad in (dict(w=None), dict(w2=None), dict(pos=None), dict(pos2=None), dict(seen=None), dict(l2=None), dict(l2=1 << 19), dict(budget=0), dict(recent=-1),
                dict(w2=p), dict(pos2=3 * p), dict(dst=c), dict(dst=fake_cache(k=1 << 20)), dict(dst=fake_cache(k=1 << 23, v=1 << 24, capacity=9)),
                dict(dst=fake_cache(k=1 << 23, v=1 << 24, hd=32)), dict(dst=fake_cache(k=1 << 23, v=1 << 24, type=capi.BF16)),
                dict(dst=fake_cache(k=(1 << 20) + 1024, v=1 << 24)), dict(dst=fake_cache(token_stride=512), w2=p, pos2=3 * p)):
        assert evict(**bad) == -1, bad
    assert cuda.ncmb_cache_evict(fake_cache(capacity=400000), d, p, 2 * p, p, 2 * p, None, p, 10, 2, 0, p) == -1
    for block, new, codes, scales in ((0, 0, p, p), (48, 0, p, p), (256, 0, p, p), (64, -1, p, p), (64, 101, p, p), (64, 0, None, p), (64, 0, p, None), (64, 0, p + 8, p)):
        assert cuda.ncmb_block_summaries(c, new, None, block, 0, codes, scales) == -1
    def blocks(q=p, ldq=256, act=capi.F32, H=4, T=1, block=32, codes=p, scales=p, sel=8, first=1, last=1, scale=0.0):
        return cuda.ncmb_block_attention(c, q, ldq, p, 256, act, H, T, block, codes, scales, sel, first, last, scale, 0, None)
    for bad in (dict(q=None), dict(ldq=250), dict(act=capi.BF16), dict(H=5), dict(T=0), dict(T=300), dict(block=24), dict(codes=None), dict(codes=p + 4), dict(scales=None),
                dict(sel=1), dict(sel=1025), dict(first=-1), dict(last=0), dict(first=2 ** 31 - 1), dict(scale=float("nan"))):
        assert blocks(**bad) == -1, bad


def test_empty_batches_are_nothing_to_do(cuda):
    c, d, p = fake_cache(rows=0), fake_cache(rows=0, k=1 << 23, v=1 << 24), 1 << 22
    assert cuda.ncmb_cache_attention(c, p, 256, p, 256, capi.F32, 4, 1, None, 0.0, 0, None) == 0
    assert cuda.ncmb_cache_evict(c, d, p, 2 * p, p, 2 * p, None, p, 10, 2, 0, p) == 0
    assert cuda.ncmb_block_summaries(c, 0, None, 64, 0, p, p) == 0
    assert cuda.ncmb_block_attention(c, p, 256, p, 256, capi.F32, 4, 1, 64, p, p, 8, 1, 1, 0.0, 0, None) == 0


def test_a_view_of_a_cache_states_its_strides():
    buf = torch.zeros(3, 20, 2, 4, 16, dtype=BF16)
    n = torch.zeros(3, dtype=torch.int32)
    k, v = (buf[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
    c = capi.KVCache.of(k, v, n)
    assert (c.k, c.v, c.type, c.rows, c.n_kv, c.hd, c.capacity) == (buf.data_ptr(), buf.data_ptr() + 128, capi.BF16, 3, 4, 16, 20)
    assert (c.row_stride, c.head_stride, c.token_stride, c.len) == (20 * 128, 16, 128, n.data_ptr())
    for bad in ((k, v[:, :, :5]), (k, v.contiguous()), (k, v.float()), (k.transpose(2, 3), v.transpose(2, 3))):
        with pytest.raises(ValueError):
            capi.KVCache.of(*bad, n)
    assert C.sizeof(capi.KVCache) == 72
