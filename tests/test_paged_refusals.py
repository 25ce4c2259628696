"""Arguments that the rotation, paged-cache and beam calls refuse: -1 and nothing queued, before a device is touched."""
import ctypes as C
import math

import pytest

import helpers

capi = helpers.capi
P = 1 << 20                             # an address that is only looked at


@pytest.fixture(scope="module")
def lib():
    return capi.NcmLib(helpers.CUDA_LIB)


def plan(lib, **kw):
    a = dict(dims=64, layout=capi.ROPE_HALVES, theta=10000.0, scaling=capi.ROPE_PLAIN, factor=1.0, trained=0.0, low=0.0, high=0.0, magnitude=1.0)
    a.update(kw)
    r = capi.Rope()
    return lib.ncmb_rope_plan(r, *a.values()), r


@pytest.mark.parametrize("bad", [dict(dims=0), dict(dims=63), dict(dims=258), dict(dims=-2), dict(layout=2), dict(theta=0.0), dict(theta=math.nan), dict(theta=math.inf),
                                 dict(scaling=4), dict(scaling=-1), dict(factor=0.0), dict(factor=math.nan), dict(magnitude=math.inf), dict(scaling=3, trained=0.0, low=1.0, high=4.0),
                                 dict(scaling=3, trained=100.0, low=4.0, high=4.0), dict(scaling=3, trained=100.0, low=math.nan, high=4.0)])
def test_plans(lib, bad):
    assert plan(lib)[0] == 0
    assert plan(lib, **bad)[0] == -1
    assert lib.ncmb_rope_plan(None, 64, 0, 1e4, 0, 1.0, 0.0, 0.0, 0.0, 1.0) == -1


def test_plan_formulas(lib):
    n, theta = 64, 10000.0
    base = [theta ** (-2 * i / n) / (2 * math.pi) for i in range(n // 2)]
    close = lambda r, want: all(abs(x - y) <= 1e-14 * y for x, y in zip(list(r.turns)[:len(want)], want)) and not any(list(r.turns)[len(want):])
    assert close(plan(lib)[1], base)
    assert close(plan(lib, scaling=capi.ROPE_LINEAR, factor=4.0)[1], [f / 4 for f in base])
    r = plan(lib, scaling=capi.ROPE_BASE, factor=4.0)[1]
    assert abs(r.turns[0] - base[0]) <= 1e-15 and abs(r.turns[31] - base[31] / 4) <= 1e-14 * base[31]
    r = plan(lib, scaling=capi.ROPE_PARTS, factor=4.0, trained=8192.0, low=1.0, high=4.0, magnitude=1.25)[1]
    assert r.magnitude == 1.25
    for i, f in enumerate(base):
        g = min(1.0, max(0.0, (8192 * f - 1) / 3))
        assert abs(r.turns[i] - f * (g + (1 - g) / 4)) <= 1e-14 * f
    assert plan(lib, dims=2, scaling=capi.ROPE_BASE, factor=4.0)[1].turns[0] == 1 / (2 * math.pi)


def rope(lib, **kw):
    a = dict(r=plan(lib)[1], x=P, xs=(C.c_int64 * 3)(6400, 640, 64), y=2 * P, ys=(C.c_int64 * 3)(6400, 640, 64), type=capi.F32, rows=2, T=10, n_head=10, hd=64, pos=None, inverse=0)
    a.update(kw)
    return lib.ncmb_rope(*a.values())


@pytest.mark.parametrize("bad", [dict(r=None), dict(xs=None), dict(ys=None), dict(x=None), dict(y=None), dict(x=P + 4), dict(y=P + 8), dict(pos=P + 2), dict(type=2), dict(rows=-1), dict(T=-1),
                                 dict(n_head=0), dict(hd=60), dict(hd=56), dict(hd=264), dict(xs=(C.c_int64 * 3)(6400, 642, 64)), dict(ys=(C.c_int64 * 3)(6400, 640, 63)),
                                 dict(ys=(C.c_int64 * 3)(6400, 640, 60)), dict(xs=(C.c_int64 * 3)(-6400, 640, 64)), dict(y=P, ys=(C.c_int64 * 3)(6400, 1280, 64)),
                                 dict(rows=1 << 16, T=1 << 16), dict(n_head=1 << 20)])
def test_rope(lib, bad):
    assert rope(lib, **bad) == -1


def test_nothing_to_do(lib):
    assert rope(lib, rows=0) == 0 and rope(lib, T=0, x=None) == 0
    assert append(lib, n_tokens=0) == 0 and append(lib, cache=cache(rows=0), n_tokens=0) == 0
    assert attend(lib, cache=cache(rows=0)) == 0
    assert select(lib, groups=0) == 0
    assert reorder(lib, cache=cache(rows=0), group=1) == 0


def cache(**kw):
    a = dict(k=P, v=2 * P, type=capi.F32, rows=4, n_kv=2, hd=64, page=16, n_pages=100, page_stride=2048, head_stride=1024, token_stride=64, table=3 * P, table_stride=8,
             max_pages=8, len=4 * P)
    a.update(kw)
    return capi.PagedCache(*a.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(k=P + 8), dict(table=P + 2), dict(len=P + 1), dict(type=2), dict(rows=-1), dict(rows=65536), dict(n_kv=0),
              dict(hd=4), dict(hd=60), dict(hd=136), dict(page=4), dict(page=24), dict(page=2048), dict(n_pages=0), dict(max_pages=0), dict(max_pages=1 << 28, table_stride=1 << 28),
              dict(table_stride=7), dict(table_stride=-8), dict(page_stride=2050), dict(head_stride=1022), dict(token_stride=62), dict(token_stride=56), dict(head_stride=8),
              dict(page_stride=-2048), dict(token_stride=0)]


def append(lib, **kw):
    a = dict(cache=cache(), r=plan(lib)[1], q=P, ldq=512, q_out=2 * P, ldqo=512, n_head=4, k=3 * P, ldk=128, v=4 * P, ldv=128, act=capi.F32, n_tokens=4, start=None, pos=None)
    a.update(kw)
    return lib.ncmb_paged_append(*a.values())


@pytest.mark.parametrize("bad", [dict(cache=None), dict(r=capi.Rope()), dict(k=None), dict(v=None), dict(k=P + 4), dict(ldk=120), dict(ldv=130), dict(ldk=126),
                                 dict(q_out=None), dict(q=P + 8), dict(ldq=248), dict(ldqo=258), dict(n_head=0), dict(q_out=P, ldqo=1024), dict(act=2), dict(act=capi.BF16), dict(n_tokens=-1),
                                 dict(n_tokens=5), dict(start=P + 2), dict(pos=P + 1)])
def test_append(lib, bad):
    assert append(lib, **bad) == -1


def test_plan_wider_than_a_head(lib):
    assert append(lib, r=plan(lib, dims=66)[1]) == -1
    assert rope(lib, r=plan(lib, dims=66)[1]) == -1


def attend(lib, **kw):
    a = dict(cache=cache(), q=P, ldq=512, out=2 * P, ldo=512, act=capi.F32, n_head=4, T=1, parents=None, scale=0.0, max_len=0)
    a.update(kw)
    return lib.ncmb_paged_attention(*a.values())


@pytest.mark.parametrize("bad", [dict(cache=None), dict(q=None), dict(out=None), dict(q=P + 4), dict(out=P + 8), dict(ldq=248), dict(ldo=250), dict(act=2), dict(act=capi.BF16), dict(n_head=0),
                                 dict(n_head=3), dict(T=0), dict(T=257), dict(T=129), dict(parents=P + 2), dict(scale=math.nan), dict(scale=math.inf)])
def test_attention(lib, bad):
    assert attend(lib, **bad) == -1


def reorder(lib, **kw):
    a = dict(cache=cache(), group=2, parents=P, n_layer=3, layer_stride=1 << 20, table_dst=5 * P, len_dst=6 * P, refs=None)
    a.update(kw)
    return lib.ncmb_paged_reorder(*a.values())


@pytest.mark.parametrize("bad", [dict(cache=None), dict(group=0), dict(group=3), dict(group=257), dict(parents=None), dict(parents=P + 2), dict(n_layer=0), dict(n_layer=65536),
                                 dict(layer_stride=-4), dict(layer_stride=8), dict(layer_stride=(1 << 20) + 2), dict(table_dst=None), dict(len_dst=None), dict(table_dst=3 * P),
                                 dict(table_dst=3 * P + 124), dict(table_dst=3 * P - 124), dict(len_dst=4 * P + 12), dict(len_dst=4 * P - 12), dict(refs=P + 1)])
def test_reorder(lib, bad):
    assert reorder(lib, **bad) == -1


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches(lib, bad):
    c = cache(**bad)
    assert append(lib, cache=c) == -1 and attend(lib, cache=c) == -1 and reorder(lib, cache=c) == -1


def select(lib, **kw):
    a = dict(logits=P, ldl=1000, type=capi.F32, groups=2, beams=4, V=1000, scores=2 * P, done=None, eos=-1, n_out=8, scores_out=3 * P, parents=4 * P, tokens=5 * P, done_out=None)
    a.update(kw)
    return lib.ncmb_beam_select(*a.values())


@pytest.mark.parametrize("bad", [dict(logits=None), dict(logits=P + 2), dict(type=2), dict(groups=-1), dict(beams=0), dict(beams=129), dict(V=0), dict(V=(1 << 24) + 1, ldl=1 << 25),
                                 dict(ldl=999), dict(scores=None), dict(scores=P + 1), dict(eos=1000), dict(done=P, eos=-1), dict(done=P, eos=1000), dict(done=P + 2, eos=5), dict(n_out=0),
                                 dict(n_out=129), dict(V=1, ldl=4, n_out=5), dict(scores_out=None), dict(parents=None), dict(tokens=None), dict(tokens=P + 2), dict(done_out=P + 3),
                                 dict(groups=1 << 23)])
def test_select(lib, bad):
    assert select(lib, **bad) == -1


def test_binding():
    import torch
    k = torch.zeros(5, 2, 16, 64)
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    c = capi.PagedCache.of(k, k, t, n)
    assert (c.rows, c.n_kv, c.hd, c.page, c.n_pages, c.max_pages, c.table_stride, c.page_stride, c.head_stride, c.token_stride) == (3, 2, 64, 16, 5, 4, 4, 2048, 1024, 64)
    wide = torch.zeros(3, 9, dtype=torch.int32)[:, :4]
    assert capi.PagedCache.of(k, k, wide, n).table_stride == 9
    for bad in [(k[0], k[0], t, n), (k, k[:, :1], t, n), (k.half(), k.half(), t, n), (k, k.bfloat16(), t, n), (k.transpose(2, 3), k.transpose(2, 3), t, n), (k, k, t.long(), n), (k, k, t, n.long()),
                (k, k, t.t(), torch.zeros(4, dtype=torch.int32)), (k, k, t[0], n), (k, k, t, n[:2]), (k, k, t, torch.zeros(6, dtype=torch.int32)[::2]), (k.to("meta"), k, t, n)]:
        with pytest.raises(ValueError):
            capi.PagedCache.of(*bad)
    with pytest.raises(ValueError):
        capi.strides(k.transpose(2, 3), 3)
    assert list(capi.strides(k, 3)) == [2048, 1024, 64]
