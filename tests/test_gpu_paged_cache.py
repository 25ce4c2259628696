"""Paged caches: append with rotation, attention through tables, reordering of groups. Against plain implementations in 64 bits; moved data
and whole numbers exactly. Bounds: test_gpu_rope.py's for what is rotated (and half a unit of the cache's type), test_gpu_cache_operators.py's
for attention."""
import numpy as np
import pytest
import torch

import helpers
import test_gpu_cache_operators as contiguous
from test_gpu_rope import HALF, KIND, PARTS, make_plan, turned

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


class Pool:
    """Pages in an order of their own; every slot holds junk until something is put there."""

    def __init__(self, rng, rows, width, page, nkv, hd, dt, layout, layers=1, spare=3):
        self.page, self.rows, self.width = page, rows, width
        n = rows * width + spare
        junk = np.array([np.nan, np.inf, -np.inf, 3.3e38, -3.3e38, 1.0], np.float32)
        full = torch.from_numpy(junk[rng.integers(0, 6, (2, layers, n, nkv, page, hd))]).to(dt).cuda()
        if layout == "token":
            self.buf = torch.empty(layers, n, page, 2, nkv, hd, dtype=dt, device="cuda")
            self.k, self.v = (self.buf[:, :, :, i].transpose(2, 3) for i in (0, 1))
        elif layout == "gap":
            self.buf = torch.empty(2, layers, n, nkv + 1, page + 1, hd + 8, dtype=dt, device="cuda")
            self.k, self.v = (self.buf[i, :, :, :nkv, :page, :hd] for i in (0, 1))
        else:
            self.buf = torch.empty(2, layers, n, nkv, page, hd, dtype=dt, device="cuda")
            self.k, self.v = self.buf[0], self.buf[1]
        self.k.copy_(full[0]); self.v.copy_(full[1])
        self.pages = rng.permutation(n)[:rows * width].reshape(rows, width)
        self.table = torch.from_numpy(self.pages.astype(np.int32)).cuda()
        self.len = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def handle(self, table=None):
        self.c = capi.PagedCache.of(self.k[0], self.v[0], self.table if table is None else table, self.len)
        return self.c

    def put(self, rng, lens):
        """Tokens 0 ... lens[b] - 1 of every row; their keys and values."""
        for b, n in enumerate(lens):
            if n <= 0:
                continue
            at = np.arange(n)
            p, s = torch.from_numpy(self.pages[b, at // self.page]).cuda(), torch.from_numpy(at % self.page).cuda()
            for x in (self.k, self.v):
                x[0][p, :, s] = torch.from_numpy(rng.standard_normal((n,) + (x.shape[2], x.shape[4])).astype(np.float32)).to(x.dtype).cuda()

    def row(self, b, n):
        at = np.arange(n)
        p, s = torch.from_numpy(self.pages[b, at // self.page]).cuda(), torch.from_numpy(at % self.page).cuda()
        return self.k[0][p, :, s], self.v[0][p, :, s]         # [n][nkv][hd]


# ------------------------------------------------------------------------------------------- append

APPENDS = [  # lens, new, H, nkv, hd, dims, page
    ([0], [1], 1, 1, 8, 8, 8), ([5, 0, 31], [1, 1, 1], 14, 2, 64, 64, 16), ([15, 16, 17, 0], [3, 0, 40, 1], 4, 4, 64, 32, 16), ([100, -1, 7], [9, 5, 130], 8, 2, 128, 128, 64),
    ([0, 3], [257, 1], 6, 2, 72, 24, 8), ([1000], [33], 12, 12, 64, 50, 32), ([0] * 40, [1 + b % 3 for b in range(40)], 2, 1, 16, 6, 1024)]


@pytest.mark.parametrize("kt,qt", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("pairs", [0, 1, None])
def test_append(cuda, kt, qt, layout, case, pairs):
    lens, news, H, nkv, hd, dims, page = case
    rng = np.random.default_rng(len(lens) * 100 + dims + hd)
    width = max((max(0, n) + t) // page + 1 for n, t in zip(lens, news))
    pool = Pool(rng, len(lens), width, page, nkv, hd, kt, layout)
    pool.len.copy_(torch.tensor(lens))
    r = None if pairs is None else make_plan(cuda, dims, pairs, **PARTS)
    lead, trail = 2, 3                                          # tokens that belong to no row
    start = lead + np.concatenate([[0], np.cumsum(news)])
    total = int(start[-1]) + trail
    x = torch.from_numpy(rng.standard_normal((total, H + 2 * nkv, hd)).astype(np.float32)).to(qt).cuda()
    pos = rng.integers(0, 300000, total) if page == 32 else None
    q_out = torch.full((total, H * hd + 8), 5.0, dtype=qt, device="cuda")
    want = {n: t.double().cpu().numpy().copy() for n, t in (("k", pool.k[0]), ("v", pool.v[0]))}
    bound = np.zeros_like(want["k"])
    q_want, q_bound = np.full((total, H, hd), 5.0), np.zeros((total, H, hd))
    x64 = x.double().cpu().numpy()
    for b, t in enumerate(news):
        if lens[b] < 0:
            continue
        i = start[b] + np.arange(t)
        at = lens[b] + np.arange(t)
        turn = (lambda y: (y, np.zeros_like(y))) if r is None else (lambda y: turned(y, pos[i] if pos is not None else at, r))
        q_want[i], q_bound[i] = turn(x64[i, :H])
        p, s = pool.pages[b, at // page], at % page
        want["k"][p, :, s], bound[p, :, s] = turn(x64[i, H:H + nkv])
        want["v"][p, :, s] = x64[i, H + nkv:]
    es, base, ld = x.element_size(), x.data_ptr(), (H + 2 * nkv) * hd
    dstart = torch.from_numpy(start.astype(np.int32)).cuda()
    dpos = torch.from_numpy(pos.astype(np.int32)).cuda() if pos is not None else None
    args = (base + H * hd * es, ld, base + (H + nkv) * hd * es, ld, KIND[qt], total, dstart.data_ptr(), dpos.data_ptr() if pos is not None else None)
    assert cuda.ncmb_paged_append(pool.handle(), r, base, ld, q_out.data_ptr(), H * hd + 8, H, *args) == 0
    torch.cuda.synchronize()
    near = lambda got, want, bound, dt: (np.isnan(want) & np.isnan(got)) | (got == want) | (np.abs(got - want) <= bound + HALF[dt] * np.abs(want) * (1 + 2.0 ** -7) + 1e-37)
    with np.errstate(invalid="ignore"):
        assert near(q_out[:, :H * hd].double().cpu().numpy().reshape(total, H, hd), q_want, q_bound, qt).all()
        assert near(pool.k[0].double().cpu().numpy(), want["k"], bound, kt).all()
        assert near(pool.v[0].double().cpu().numpy(), want["v"], 0, kt).all()
    assert (q_out[:, H * hd:] == 5).all()
    # queries in place, and keys and values alone, give the same bits
    k0, q0 = pool.k.clone(), q_out[:, :H * hd].clone()
    assert cuda.ncmb_paged_append(pool.handle(), r, base, ld, base, ld, H, *args) == 0
    used = torch.zeros(total, dtype=torch.bool)
    for b, t in enumerate(news):
        used[start[b]:start[b + 1]] = lens[b] >= 0
    assert torch.equal(x[:, :H].reshape(total, -1)[used.cuda()], q0[used.cuda()])
    assert cuda.ncmb_paged_append(pool.handle(), r, None, 0, None, 0, 0, *args) == 0
    torch.cuda.synchronize()
    assert torch.equal(pool.k.view(torch.int16 if kt == BF16 else torch.int32), k0.view(torch.int16 if kt == BF16 else torch.int32))


def test_append_a_step(cuda):
    """As many tokens of every row, without starts; many rows."""
    for rows, T in ((1100, 1), (3, 5)):
        rng = np.random.default_rng(rows)
        pool = Pool(rng, rows, 3, 8, 2, 64, BF16, "token")
        lens = rng.integers(0, 24 - T + 1, rows)
        pool.len.copy_(torch.from_numpy(lens.astype(np.int32)))
        x = torch.from_numpy(rng.standard_normal((rows * T, 4, 64)).astype(np.float32)).cuda()
        for starts in (None, torch.arange(0, rows * T + 1, T, dtype=torch.int32, device="cuda")):
            pool.k.zero_(); pool.v.zero_()
            assert cuda.ncmb_paged_append(pool.handle(), None, None, 0, None, 0, 0, x.data_ptr(), 256, x.data_ptr() + 512, 256, capi.F32, rows * T,
                                          starts.data_ptr() if starts is not None else None, None) == 0
            torch.cuda.synchronize()
            for b in list(range(0, rows, 37)) + [rows - 1]:
                k, v = pool.row(b, lens[b] + T)
                mine = x[b * T:(b + 1) * T].to(BF16)
                assert torch.equal(k[lens[b]:], mine[:, :2]) and torch.equal(v[lens[b]:], mine[:, 2:]) and not k[:lens[b]].any()


def test_append_without_pages(cuda):
    """Entries that are no page, rows that are full: nothing is stored and queries are rotated all the same."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, 4, 2, 8, 1, 16, F32, "head")
    pool.k.zero_(); pool.v.zero_()
    table = torch.tensor(pool.pages.astype(np.int32))
    table[0, 1], table[1, 0], table[2, 1] = -1, pool.k.shape[1], 2 ** 31 - 1
    pool.len.copy_(torch.tensor([7, 3, 8, 15]))
    d = table.cuda()
    r = make_plan(cuda, 16, 0)
    x = torch.randn(4 * 3, 3, 16, device="cuda")
    q = torch.zeros(12, 16, device="cuda")
    assert cuda.ncmb_paged_append(pool.handle(d), r, x.data_ptr(), 48, q.data_ptr(), 16, 1, x.data_ptr() + 64, 48, x.data_ptr() + 128, 48, capi.F32, 12, None, None) == 0
    torch.cuda.synchronize()
    want, bound = turned(x[:, :1].double().cpu().numpy(), (np.array([7, 3, 8, 15])[:, None] + np.arange(3)).reshape(-1), r)
    assert (np.abs(q.double().cpu().numpy()[:, None] - want) <= bound + 2.0 ** -24 * np.abs(want)).all()
    stored = pool.v[0, :, 0].abs().sum(-1) > 0
    assert stored.sum() == 2                                    # the first token of rows 0 and 3
    assert torch.equal(pool.v[0, pool.pages[0, 0], 0, 7], x[0, 2]) and torch.equal(pool.v[0, pool.pages[3, 1], 0, 7], x[9, 2])


# ------------------------------------------------------------------------------------------- attention

def run_attention(cuda, seed, lens, T, H, nkv, hd, kt, qt, layout, page, tree=False, max_len=0, scale=0.0, holes=()):
    rng = np.random.default_rng(seed)
    B, G = len(lens), H // nkv
    width = max((max(0, n) + T - 1) // page + 1 for n in lens) + 1
    pool = Pool(rng, B, width, page, nkv, hd, kt, layout)
    pool.put(rng, [n + T if n >= 0 else 0 for n in lens])
    pool.len.copy_(torch.tensor(lens))
    table = pool.table.clone()
    for b, i, bad in holes:
        table[b, i] = bad
    par = contiguous.make_parents(rng, B, T) if tree else None
    dpar = torch.tensor(par, dtype=torch.int32, device="cuda") if tree else None
    q = torch.from_numpy(1.5 * rng.standard_normal((B, T, H, hd)).astype(np.float32)).to(qt).cuda()
    out = torch.full((B, T, H * hd + 8), 5.0, dtype=qt, device="cuda")
    assert cuda.ncmb_paged_attention(pool.handle(table), q.data_ptr(), H * hd, out.data_ptr(), H * hd + 8, KIND[qt], H, T, dpar.data_ptr() if tree else None, scale, max_len) == 0
    torch.cuda.synchronize()
    assert (out[:, :, H * hd:] == 5).all()
    got = out[:, :, :H * hd].view(B, T, H, hd)
    for b, n in enumerate(lens):
        if n < 0:
            assert not got[b].any()
            continue
        ok = contiguous.visible(n, T, par[b] if tree else None)
        for bb, i, _ in holes:
            if bb == b:
                ok[:, i * page:(i + 1) * page] = False
        k, v = pool.row(b, n + T)
        k, v = (torch.nan_to_num(x.double(), 0, 0, 0) for x in (k, v))
        for h in range(nkv):
            want, _, rel = contiguous.attend64(q[b, :, h * G:(h + 1) * G], k[:, h], v[:, h], ok, scale or hd ** -0.5)
            bound = rel[..., None] * np.abs(v[:, h].cpu().numpy()).max()
            contiguous.check(got[b, :, h * G:(h + 1) * G], want, bound, qt)
    return got


TYPES = [(F32, F32), (BF16, F32), (BF16, BF16)]


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 1024])
@pytest.mark.parametrize("H,nkv,hd", [(12, 12, 64), (14, 2, 64), (4, 1, 128), (32, 2, 128), (3, 3, 72), (2, 1, 8)])
def test_one_token(cuda, kt, qt, page, H, nkv, hd):
    run_attention(cuda, page + H, [0, 1, page - 1, page, 33, 700], 1, H, nkv, hd, kt, qt, ["token", "head", "gap"][page % 7 % 3], page)


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("page,H,nkv,hd,T,tree", [(8, 14, 2, 64, 3, False), (16, 8, 8, 64, 9, True), (64, 8, 2, 128, 40, True), (16, 4, 4, 40, 256, False), (32, 28, 2, 64, 2, False)])
def test_several_tokens(cuda, kt, qt, page, H, nkv, hd, T, tree):
    run_attention(cuda, page + T, [0, 5, 300, 1111], T, H, nkv, hd, kt, qt, "token" if T % 2 else "head", page, tree)


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("B,n,page", [(1, 20000, 16), (30, 3000, 64), (130, 260, 8)])
def test_long_and_many(cuda, kt, qt, B, n, page):
    """Units cut over CTAs, joined in the kernel or by one of their own; a bound of lengths that is too low."""
    lens = [n] + [(b * 7919) % n for b in range(1, B)]
    for max_len in (0, 50):
        run_attention(cuda, B, lens, 1, 8, 2, 64, kt, qt, "head", page, max_len=max_len)


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_rows_and_entries_without_a_page(cuda, kt, qt, page):
    big = 2 ** 31 - 1
    run_attention(cuda, 1, [100, -1, 64, 0, 33, -2 ** 31], 1, 14, 2, 64, kt, qt, "token", page, holes=[(0, 1, -1), (0, 100 // page, big), (2, 0, 10 ** 6), (3, 0, -5)])
    run_attention(cuda, 2, [40, -7], 5, 4, 2, 128, kt, qt, "head", page, tree=True, holes=[(0, 0, -1), (0, 40 // page, -2)])


def test_lengths_beyond_the_pages(cuda):
    """A length above what the row's pages hold counts as the most that they hold beside the new tokens."""
    rng = np.random.default_rng(4)
    pool = Pool(rng, 2, 3, 16, 2, 64, BF16, "head")
    pool.put(rng, [48, 48])
    q = torch.randn(2, 1, 4, 64, device="cuda")
    outs = []
    for n in (47, 48, 1000, 2 ** 31 - 1):
        pool.len.fill_(n)
        out = torch.empty_like(q)
        assert cuda.ncmb_paged_attention(pool.handle(), q.data_ptr(), 256, out.data_ptr(), 256, capi.F32, 4, 1, None, 0.0, 0) == 0
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_shared_pages_and_far_offsets(cuda):
    """Rows that share pages see the same; pages whose offsets pass 32 bits."""
    nkv, hd, page = 2, 128, 64
    n_pages = 160000                                            # 160000 * 64 * 2 * 128 elements: 5.2 GB of keys
    k = torch.empty(n_pages, nkv, page, hd, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    far = torch.tensor([159999, 140001, 3, 150000], device="cuda")
    k[far], v[far] = (torch.randn(4, nkv, page, hd, device="cuda").to(BF16) for _ in range(2))
    table = torch.tensor([[159999, 140001, 3, -1], [159999, 140001, 3, 150000]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([190, 190], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 1, 4, hd, device="cuda").expand(2, 1, 4, hd).contiguous()
    out = torch.empty_like(q)
    c = capi.PagedCache.of(k, v, table, lens)
    x = torch.randn(2, 2 * nkv, hd, device="cuda")
    x[1] = x[0]
    lens.fill_(190)
    assert cuda.ncmb_paged_append(c, None, None, 0, None, 0, 0, x.data_ptr(), 2 * nkv * hd, x.data_ptr() + nkv * hd * 4, 2 * nkv * hd, capi.F32, 2, None, None) == 0
    assert cuda.ncmb_paged_attention(c, q.data_ptr(), 4 * hd, out.data_ptr(), 4 * hd, capi.F32, 4, 1, None, 0.0, 0) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1])
    assert torch.equal(k[3, :, 62], x[0, :nkv].to(BF16))
    kk, vv = (t[table[0, :3].long()].permute(1, 0, 2, 3).reshape(nkv, 192, hd)[:, :191] for t in (k, v))
    for h in range(nkv):
        want, _, rel = contiguous.attend64(q[0, :, 2 * h:2 * h + 2], kk[h], vv[h], np.ones((1, 191), bool), hd ** -0.5)
        contiguous.check(out[0, :, 2 * h:2 * h + 2], want, rel[..., None] * vv[h].abs().max().item(), F32)


# ------------------------------------------------------------------------------------------- reordering

def plain_reorder(table, lens, parents, group, page, n_pages, k, v, refs):
    """By the definition, row after row; k, v [layer][page][head][slot][hd] on the host are changed."""
    rows, width = table.shape
    table = np.where((table >= 0) & (table < n_pages), table, -1)
    t2, l2 = np.full_like(table, -1), np.empty(rows, np.int32)
    cap = width * page
    k0, v0 = k.clone(), v.clone()
    for g in range(0, rows, group):
        par = [int(p) if 0 <= p < group else -1 for p in parents[g:g + group]]
        free = [i for i in range(group) if i not in par]
        seen = set()
        for j, p in enumerate(par):
            first = p >= 0 and p not in seen
            seen.add(p)
            own = p if first else free.pop(0)
            n = min(max(lens[g + p], 0), cap) if p >= 0 else 0
            tp, to = n // page, min(max(lens[g + own], 0), cap) // page
            row = ([] if p < 0 else list(table[g + p, :tp])) + list(table[g + own, to:])
            row = (row + [-1] * width)[:width]
            t2[g + j], l2[g + j] = row, lens[g + p] if p >= 0 else -1
            src, dst = (table[g + p, tp] if p >= 0 and tp < width else -1), (table[g + own, to] if to < width else -1)
            if not first and src >= 0 and dst >= 0:
                k[:, dst, :, :n % page], v[:, dst, :, :n % page] = k0[:, src, :, :n % page], v0[:, src, :, :n % page]
    for x in table.ravel():
        if x >= 0: refs[x] -= 1
    for x in t2.ravel():
        if x >= 0: refs[x] += 1
    return t2, l2


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("layout", ["token", "head", "gap"])
@pytest.mark.parametrize("groups,group,page,layers,kind", [(1, 1, 8, 1, "random"), (3, 4, 16, 3, "random"), (2, 8, 64, 2, "one"), (2, 8, 32, 2, "same"), (5, 7, 16, 1, "bad"), (1, 256, 8, 2, "random"),
                                                           (4, 33, 8, 1, "bad"), (2, 5, 16, 2, "full")])
def test_reorder(cuda, dt, layout, groups, group, page, layers, kind):
    rng = np.random.default_rng(groups * 100 + group + page)
    rows, width, nkv, hd = groups * group, 6, 2, 24
    pool = Pool(rng, rows, width, page, nkv, hd, dt, layout, layers)
    lens = np.repeat(rng.integers(0, 3 * page, groups), group).astype(np.int32)
    if kind == "full":
        lens[:] = 2 * page                                      # nothing begun: pages change hands and nothing is copied
    table = pool.pages.astype(np.int32).copy()
    for g in range(groups):                                     # a common beginning
        table[g * group:(g + 1) * group, :lens[g * group] // page] = table[g * group, :lens[g * group] // page]
    table[:, 5] = -1
    parents = rng.integers(0, group, rows).astype(np.int32)
    if kind == "one":
        parents[:] = group - 1
    if kind == "same":
        parents = np.tile(np.arange(group)[::-1], groups).astype(np.int32)
    if kind == "bad":                                           # rows of other lengths, rows and entries that are empty, parents that are none
        lens = rng.integers(-1, width * page + 9, rows).astype(np.int32)
        lens[rng.random(rows) < 0.1] = 2 ** 31 - 1
        parents[rng.random(rows) < 0.2] = rng.choice([-1, group, 2 ** 31 - 1, -2 ** 31])
        table[rng.random(table.shape) < 0.1] = rng.choice([-1, pool.k.shape[1], 2 ** 31 - 1])
    pool.len.copy_(torch.from_numpy(lens))
    for x in (pool.k, pool.v):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)).to(dt))
    k, v = pool.k.cpu(), pool.v.cpu()
    refs = rng.integers(0, 50, pool.k.shape[1]).astype(np.int32)
    d, drefs = torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda()
    t2, l2 = plain_reorder(table, lens, parents, group, page, pool.k.shape[1], k, v, refs)
    dt2, dl2, dp = torch.full_like(d, 99), torch.full_like(pool.len, 99), torch.from_numpy(parents).cuda()
    for passes in range(2):                                     # a second call finds parents as they were
        assert cuda.ncmb_paged_reorder(pool.handle(d), group, dp.data_ptr(), layers, pool.k.stride(0), dt2.data_ptr(), dl2.data_ptr(), drefs.data_ptr() if passes == 0 else None) == 0
        torch.cuda.synchronize()
        assert np.array_equal(dt2.cpu().numpy(), t2) and np.array_equal(dl2.cpu().numpy(), l2)
        assert np.array_equal(drefs.cpu().numpy(), refs)
        assert torch.equal(pool.k.cpu(), k) and torch.equal(pool.v.cpu(), v)
        assert np.array_equal(d.cpu().numpy(), table)
        if kind == "bad":
            break                                               # rows of other lengths may begin on one another's pages


# ------------------------------------------------------------------------------------------- attention of many query rows

@pytest.fixture(params=[1, 2])
def variant(request, cuda):
    """Tiles of 16 rows, and of 128 where they take the shape."""
    cuda.ncmb_set_cache_variant(request.param)
    yield request.param
    cuda.ncmb_set_cache_variant(0)
    assert cuda.ncmb_gemm_tc_check() == 0


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("H,nkv,hd,T,tree", [(8, 2, 64, 9, True), (8, 1, 64, 5, False), (4, 2, 128, 20, True), (6, 2, 72, 40, False)])
def test_many_query_rows(cuda, variant, kt, qt, page, H, nkv, hd, T, tree):
    run_attention(cuda, page + T, [0, 1, 127 - T, 128, 129, 700], T, H, nkv, hd, kt, qt, ["token", "head", "gap"][(page + T) % 3], page, tree)


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("page", [8, 32, 256])
def test_many_query_rows_without_pages(cuda, variant, kt, qt, page):
    """Entries that are no page in whole tiles, in the last one and at the new tokens; rows of no sequence."""
    run_attention(cuda, 3, [600, -1, 513, 0, 128, -2 ** 31], 18, 4, 2, 64, kt, qt, "token", page, tree=True,
                  holes=[(0, 1, -1), (0, 600 // page, 2 ** 31 - 1), (2, 0, 10 ** 6), (2, 300 // page, -3), (3, 0, -5), (4, 0, -1)])
    run_attention(cuda, 4, [300, 40], 30, 2, 1, 64, kt, qt, "head", page, holes=[(1, 0, -1), (1, 40 // page, -2), (0, 0, -1)])


@pytest.mark.parametrize("kt,qt", TYPES)
@pytest.mark.parametrize("B,n,T,H,nkv,hd,page", [(1, 9000, 16, 32, 8, 64, 16), (7, 2500, 64, 8, 2, 128, 64), (40, 300, 7, 14, 2, 64, 8), (2, 1500, 256, 4, 2, 64, 32)])
def test_many_query_rows_of_long_rows(cuda, variant, kt, qt, B, n, T, H, nkv, hd, page):
    """Units cut over CTAs, query rows in several tiles."""
    run_attention(cuda, B + T, [n] + [(b * 7919) % n for b in range(1, B)], T, H, nkv, hd, kt, qt, "head" if T % 3 else "token", page)


def test_a_call_that_finds_the_error_word_set(cuda):
    """As for contiguous caches: the call ends, the word is reported, results are not written, the next call is right."""
    cuda.ncmb_set_cache_variant(2)
    try:
        rng = np.random.default_rng(6)
        pool = Pool(rng, 2, 60, 64, 2, 64, BF16, "token")
        pool.put(rng, [3040, 57])
        pool.len.copy_(torch.tensor([3000, 17]))
        q = torch.randn(2, 40, 14, 64, device="cuda")
        out = torch.full_like(q, 5.0)
        assert cuda.ncmb_gemm_tc_check() == 0
        cuda.ncmb_gemm_tc_raise(47)
        assert cuda.ncmb_paged_attention(pool.handle(), q.data_ptr(), 14 * 64, out.data_ptr(), 14 * 64, capi.F32, 14, 40, None, 0.0, 0) == 0
        torch.cuda.synchronize()
        assert (out == 5.0).all() and cuda.ncmb_gemm_tc_check() == 47
        run_attention(cuda, 3, [3000, 17], 40, 14, 2, 64, BF16, F32, "token", 64, True)
        assert cuda.ncmb_gemm_tc_check() == 0
    finally:
        cuda.ncmb_set_cache_variant(0)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_prompt_in_pieces(cuda, dt):
    """Appended and attended to in pieces of any sizes, a prompt gives what it gives at once (bf16 products' order aside)."""
    H, nkv, hd, page, n = 8, 2, 64, 16, 700
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(2, n, H + 2 * nkv, hd, device="cuda", generator=g)
    r = make_plan(cuda, hd, 0)
    got = []
    for pieces in ([256, 256, 188], [1, 7, 100, 255, 16, 16, 200, 105]):
        pool = Pool(np.random.default_rng(0), 2, n // page + 2, page, nkv, hd, dt, "token")
        outs, at = [], 0
        for T in pieces:
            x = qkv[:, at:at + T].contiguous()
            ld, w, p = (H + 2 * nkv) * hd, H * hd, x.data_ptr()
            pool.len.fill_(at)
            out = torch.empty(2, T, H, hd, device="cuda")
            assert cuda.ncmb_paged_append(pool.handle(), r, p, ld, p, ld, H, p + w * 4, ld, p + (w + nkv * hd) * 4, ld, capi.F32, 2 * T, None, None) == 0
            assert cuda.ncmb_paged_attention(pool.handle(), p, ld, out.data_ptr(), w, capi.F32, H, T, None, 0.0, 0) == 0
            outs.append(out)
            at += T
        got.append(torch.cat(outs, 1))
        k, v = zip(*(pool.row(b, n) for b in range(2)))
    torch.cuda.synchronize()
    rot = turned(qkv[:, :, :H].double().cpu().numpy(), np.broadcast_to(np.arange(n), (2, n)), r)[0]
    ok = np.tril(np.ones((n, n), bool))
    for b in range(2):
        for h in range(nkv):
            want, _, rel = contiguous.attend64(torch.from_numpy(rot[b, :, 4 * h:4 * h + 4]), k[b][:, h], v[b][:, h], ok, hd ** -0.5)
            for o in got:                                       # queries come rotated in fp32: 2^-21 of a score more
                contiguous.check(o[b, :, 4 * h:4 * h + 4], want, (rel[..., None] * 1.5 + 2.0 ** -18) * v[b][:, h].abs().max().item(), F32)
