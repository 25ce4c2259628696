"""The best continuations of groups of beams (ncmb_beam_select) against a plain selection in 64 bits.

Bound of a score: an exponential is within 2^-22 of itself and its argument's rounding within 2^-23 (x 2^-d d <= 0.54 for the term's weight), 32 of them
are added in fp32 (10 * 2^-24), the sum is scaled by the maximum's changes, each within 2^-22, at most one a tile after a part's first (18 here)
and three where threads, warps and parts meet: log sum exp within 25 * 2^-22 = 6e-6, and half a unit of fp32. Two continuations of
different beams that are nearer than twice that may change places (equal beams, whose sums are equal, may not)."""
import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16
FMAX = np.finfo(np.float32).max
LSE = 25 * 2.0 ** -22


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


def plain(x, scores, done, eos, n):
    """x float32 [groups][beams][V] -> scores (64 bits), parents, tokens, done of the n best, and score and log sum exp of each group's candidates"""
    out, every = [], []
    for g in range(x.shape[0]):
        cands, seen = [], {}
        for k in range(x.shape[1]):
            r = x[g, k].astype(np.float64)
            r = np.where(np.isnan(r), -np.inf, np.minimum(r, FMAX))
            if done is not None and done[g, k]:
                r = np.full_like(r, -np.inf)
                r[eos] = 0.0
            key = r.tobytes()
            if key not in seen:                                 # equal rows, equal sums
                m = r.max()
                seen[key] = (m + np.log(np.exp(r - m).sum()) if m > -np.inf else 0.0, np.lexsort((np.arange(len(r)), -r))[:n + 1])
            lse, order = seen[key]
            if done is not None and done[g, k]:
                lse = 0.0
            s = float(scores[g, k])
            s = -np.inf if np.isnan(s) else s
            for i, w in enumerate(order):
                cands.append((-np.inf if r[w] == -np.inf else s + (r[w] - lse), -k, -i, w, lse))
        cands.sort(key=lambda c: c[:3], reverse=True)
        out.append(cands[:n])
        every.append(cands)
    sc = np.array([[c[0] for c in o[:n]] for o in out])
    par = np.array([[-c[1] for c in o[:n]] for o in out])
    tok = np.array([[c[3] for c in o[:n]] for o in out])
    dn = (tok == eos) | (np.take_along_axis(done, par, 1) != 0 if done is not None else False)
    known = [{(-c[1], c[3]): (c[0], c[4]) for c in o} for o in every]
    return sc, par, tok, dn.astype(np.int32), known


def run(cuda, x, scores, n, done=None, eos=-1, dt=F32, ld=None, offset=0, in_place=False):
    """x: float32 [groups][beams][V] whose values dt holds"""
    G, K, V = x.shape
    ld = ld or V
    buf = torch.full((offset + G * K * ld,), float("nan"), dtype=dt, device="cuda")
    rows = buf[offset:].view(G * K, ld)
    rows[:, :V] = torch.from_numpy(x.reshape(G * K, V)).to(dt)
    sc = torch.from_numpy(np.asarray(scores, np.float32)).cuda()
    dn = torch.from_numpy(done.astype(np.int32)).cuda() if done is not None else None
    so, po, to, do = sc if in_place else torch.empty(G, n, device="cuda"), *(torch.full((G, n), -9, dtype=torch.int32, device="cuda") for _ in range(3))
    if in_place and dn is not None:
        do = dn
    want = plain(rows[:, :V].float().cpu().numpy().reshape(G, K, V), np.asarray(scores, np.float32), done, eos, n)
    assert cuda.ncmb_beam_select(rows.data_ptr(), ld, capi.F32 if dt == F32 else capi.BF16, G, K, V, sc.data_ptr(), dn.data_ptr() if dn is not None else None, eos, n, so.data_ptr(),
                                 po.data_ptr(), to.data_ptr(), do.data_ptr()) == 0
    torch.cuda.synchronize()
    got = [t.cpu().numpy() for t in (so, po, to, do)]
    for g, i in zip(*np.nonzero((got[1] != want[1]) | (got[2] != want[2]))):
        mine, best = want[4][g][got[1][g, i], got[2][g, i]], want[4][g][want[1][g, i], want[2][g, i]]
        assert got[1][g, i] != want[1][g, i] and mine[1] != best[1] and abs(mine[0] - best[0]) <= 2 * LSE, (g, i, mine, best)
    for g in range(G):
        picks = list(zip(got[1][g], got[2][g]))
        assert len(set(picks)) == n and [d for d in got[3][g]] == [int(w == eos or (done is not None and done[g, k] != 0)) for k, w in picks]
    a, b = got[0].astype(np.float64), want[0]
    fine = np.isfinite(b)
    assert np.array_equal(a[~fine], b[~fine])
    assert (np.abs(a - b)[fine] <= LSE + 2.0 ** -24 * np.abs(b[fine]) * (1 + 2.0 ** -20)).all()
    return got


def logits(rng, G, K, V, dt=F32):
    x = 2 * rng.standard_normal((G, K, V)) + 6 * np.maximum(0, rng.standard_normal((G, K, V)) - 2.5)
    return torch.from_numpy(x.astype(np.float32)).to(dt).float().numpy()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("G,K,V,n", [(1, 1, 1, 1), (1, 4, 50257, 8), (3, 5, 1000, 5), (2, 3, 4096, 6), (2, 8, 4097, 16), (1, 128, 300, 128), (40, 2, 777, 3), (1, 2, 3, 6), (2, 1, 200, 128),
                                     (1, 32, 8192, 64), (300, 1, 129, 1), (1, 1, 16384, 33), (2, 4, 151936, 9)])
def test_sizes(cuda, dt, G, K, V, n):
    rng = np.random.default_rng(G * 7 + K * 3 + V + n)
    x = logits(rng, G, K, V, dt)
    scores = (-30 * rng.random((G, K))).astype(np.float32)
    got = run(cuda, x, scores, n, dt=dt)
    es = 4 if dt == F32 else 2
    ld = V + 16 // es - V % (16 // es) + 16 // es                        # rows of whole 16 bytes, and rows that begin anywhere
    for other in (run(cuda, x, scores, n, dt=dt, ld=ld), run(cuda, x, scores, n, dt=dt, ld=ld + 1, offset=3)):
        assert np.array_equal(got[1], other[1]) and np.array_equal(got[2], other[2])


@pytest.mark.parametrize("n", [1, 7, 32, 100])
def test_orders_of_values(cuda, n):
    """Rising, falling, constant, few values, large ones a stride apart: however they lie, what reaches a bound fits the list."""
    V = 30011
    i = np.arange(V)
    rows = [i * 1e-3, -i * 1e-3, np.zeros(V), (i * 7919 % 5).astype(float), np.where(i % 256 == 3, 5 + i * 1e-4, 0), np.where(i % 1024 < 4, 5 - i * 1e-4, -1), np.where(i // 16 % 256 == 9, 3.0, 0),
            np.where(i >= V - 300, i - V + 301.0, 0), np.where(i < 300, i * 0.01, -50.0)]
    x = np.stack(rows).astype(np.float32)[:, None]
    run(cuda, x, np.zeros((len(rows), 1)), n)
    run(cuda, x, np.zeros((len(rows), 1)), n, ld=30012)


@pytest.mark.parametrize("V", [50, 9001])
def test_masked_and_not_finite(cuda, V):
    """NaN, infinities, rows of nothing, the type's lowest value, -0 against 0, beams that are not there."""
    rng = np.random.default_rng(V)
    x = logits(rng, 6, 4, V)
    x[0, 1] = -np.inf
    x[0, 2] = np.nan
    x[1, :, 10:] = -np.inf
    x[2, 0, rng.random(V) < 0.3] = np.nan
    x[2, 1, 5], x[2, 1, 7] = np.inf, np.inf
    x[2, 2, 3:] = -FMAX
    x[3] = -FMAX
    x[4, 0] = np.where(np.arange(V) % 2, 0.0, -0.0)
    x[5] = -np.inf
    scores = np.array([[-1, -2, -3, -4.0], [-1, -np.inf, -3, np.nan], [-5, -9, -30, -50], [0, -100, -200, -300], [-1, -FMAX, -500, -501], [-1, -2, -3, -4]], np.float32)
    for n in (1, 4, 25, 40):
        run(cuda, x, scores, n)
        run(cuda, x, scores, n, ld=V + 3 & ~3)


def test_equal_beams(cuda):
    """The first step, when all beams are the same: of equal scores the lower beam is first; rows are split alike whatever their number."""
    rng = np.random.default_rng(8)
    for G, K, V in ((1, 4, 50257), (3, 8, 151936), (2, 128, 5000)):
        x = np.repeat(logits(rng, G, 1, V), K, 1)
        run(cuda, x, np.full((G, K), -2.5), min(2 * K, 128))
        first = np.full((G, K), -np.inf)
        first[:, 0] = 0
        got = run(cuda, x, first, min(2 * K, 128))
        assert (got[1] == 0).all()
        first[:, 1:] = -FMAX
        run(cuda, x, first, min(2 * K, 128))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_ended_beams(cuda, dt):
    rng = np.random.default_rng(12)
    for V, eos in ((7, 0), (7, 6), (2000, 2), (50257, 50256)):
        x = logits(rng, 5, 4, V, dt)
        scores = (-3 * rng.random((5, 4))).astype(np.float32)
        done = np.zeros((5, 4), np.int64)
        done[1, 2], done[2, :3], done[3] = 1, -1, 5
        x[4, :, eos] = 20.0                                      # ends now
        x = torch.from_numpy(x).to(dt).float().numpy()
        for n in (1, 4, 20):
            run(cuda, x, scores, n, done, eos, dt)
        run(cuda, x, scores, 4, done, eos, dt, in_place=True)
    run(cuda, logits(rng, 5, 4, 100), scores, 4, None, 3, in_place=True)


def test_again_and_captured(cuda):
    """The same bits call after call, also from a graph, with other calls' sizes in between."""
    rng = np.random.default_rng(4)
    x = logits(rng, 4, 6, 20000)
    scores = (-9 * rng.random((4, 6))).astype(np.float32)
    first = run(cuda, x, scores, 12)
    run(cuda, logits(rng, 1, 2, 60000), np.zeros((1, 2)), 30)
    for _ in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(first, run(cuda, x, scores, 12)))
    d, s = torch.from_numpy(x).cuda(), torch.from_numpy(scores).cuda()
    outs = [torch.zeros(4, 12, device="cuda")] + [torch.zeros(4, 12, dtype=torch.int32, device="cuda") for _ in range(3)]
    stream = torch.cuda.Stream()
    call = lambda: cuda.ncmb_beam_select(d.data_ptr(), 20000, capi.F32, 4, 6, 20000, s.data_ptr(), None, -1, 12, *(o.data_ptr() for o in outs))
    torch.cuda.synchronize()
    try:
        cuda.ncmb_set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            assert call() == 0
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                assert call() == 0
        for o in outs:
            o.zero_()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
    finally:
        cuda.ncmb_set_stream(None)
    assert all(np.array_equal(a, o.cpu().numpy()) for a, o in zip(first, outs))


@pytest.mark.parametrize("G,K,V", [(1, 1, 1 << 24), (2, 3, 3000001)])
def test_the_largest_vocabularies(cuda, G, K, V):
    """Against torch's sums and sorts in 64 bits; rows end inside a tile, and a row is split into as many parts as the GPU holds."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(G * K, V, device="cuda", generator=g)
    scores = -torch.rand(G, K, device="cuda", generator=g)
    n = 40
    out = torch.empty(G, n, device="cuda"), *(torch.empty(G, n, dtype=torch.int32, device="cuda") for _ in range(2))
    assert cuda.ncmb_beam_select(x.data_ptr(), V, capi.F32, G, K, V, scores.data_ptr(), None, -1, n, *(t.data_ptr() for t in out), None) == 0
    words = x.sort(dim=1, descending=True, stable=True).indices[:, :n]
    s = scores.double().view(-1, 1) + x.gather(1, words).double() - torch.logsumexp(x.double(), 1, keepdim=True)
    want, at = s.view(G, K * n).sort(dim=1, descending=True, stable=True)
    assert ((out[0].double() - want[:, :n]).abs() <= LSE * 20 + 2.0 ** -22).all()         # as many tiles a part as a row has, at most
    far = torch.ones(G, n, dtype=torch.bool, device="cuda")                               # from the next: those may not change places
    gap = (want[:, 1:n + 1] - want[:, :n]).abs() > 40 * LSE if K > 1 else torch.ones(G, n, dtype=torch.bool, device="cuda")
    if K > 1:
        far = gap & torch.cat([torch.ones_like(gap[:, :1]), gap[:, :-1]], 1)
    assert (out[1].long() == at[:, :n] // n)[far].all() and (out[2].long() == words.reshape(G, K * n).gather(1, at[:, :n]))[far].all()
