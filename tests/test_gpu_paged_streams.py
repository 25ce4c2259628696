"""The paged-cache and beam calls on two streams in turn, and a whole search step captured and replayed: the bits of single eager calls."""
import importlib.util
import os

import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    return capi.NcmLib(helpers.CUDA_LIB)


@pytest.fixture(autouse=True)
def default_stream(cuda):
    """A test leaves the library on the stream that torch's calls are on by default."""
    yield
    torch.cuda.synchronize()
    cuda.ncmb_set_stream(None)


class Work:
    """A decode step of 12 groups of 4 beams on tensors of its own."""

    def __init__(self, lib, seed, n, page, H, nkv, hd, V, dt):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.lib, self.H, self.nkv, self.hd, self.V, self.B, self.K = lib, H, nkv, hd, V, 12, 4
        rows, width = 48, n // page + 2
        self.pool0 = r(2, 2, rows * width, nkv, page, hd).to(dt)
        self.pool = self.pool0.clone()
        self.table = torch.randperm(rows * width, device="cuda", generator=g).int().view(rows, width)
        self.len = torch.tensor([max(0, n - 41 * (b // 4)) for b in range(rows)], dtype=torch.int32, device="cuda")
        self.c = capi.PagedCache.of(self.pool[0, 0], self.pool[1, 0], self.table, self.len)
        self.qkv = r(rows, H + 2 * nkv, hd)
        self.q, self.out = torch.zeros(rows, H, hd, device="cuda"), torch.zeros(rows, H, hd, device="cuda")
        self.logits, self.scores = 2 * r(rows, V), -r(12, 4).abs()
        self.so = torch.zeros(12, 4, device="cuda")
        self.po, self.to, self.do = (torch.zeros(12, 4, dtype=torch.int32, device="cuda") for _ in range(3))
        self.t2, self.l2 = torch.zeros_like(self.table), torch.zeros_like(self.len)
        # the last new tokens of every row once more, 24 at a time: tiles of many query rows
        self.q2 = r(rows, 24, H, hd)
        self.out2 = torch.zeros_like(self.q2)
        self.len2 = (self.len - 23).clamp(min=0)
        self.c2 = capi.PagedCache.of(self.pool[0, 0], self.pool[1, 0], self.table, self.len2)
        self.plan = capi.Rope()
        assert lib.ncmb_rope_plan(self.plan, hd, 1, 10000.0, 0, 1.0, 0.0, 0.0, 0.0, 1.0) == 0
        torch.cuda.synchronize()

    def run(self):
        self.pool.copy_(self.pool0)                               # or a second step finds what the first has copied to rows that nobody continues
        lib, p, ld, w = self.lib, self.qkv.data_ptr(), (self.H + 2 * self.nkv) * self.hd, self.H * self.hd
        rc = lib.ncmb_paged_append(self.c, self.plan, p, ld, self.q.data_ptr(), w, self.H, p + w * 4, ld, p + (w + self.nkv * self.hd) * 4, ld, capi.F32, 48, None, None)
        rc |= lib.ncmb_paged_attention(self.c, self.q.data_ptr(), w, self.out.data_ptr(), w, capi.F32, self.H, 1, None, 0.0, 0)
        rc |= lib.ncmb_paged_attention(self.c2, self.q2.data_ptr(), w, self.out2.data_ptr(), w, capi.F32, self.H, 24, None, 0.0, 0)
        rc |= lib.ncmb_beam_select(self.logits.data_ptr(), self.V, capi.F32, 12, 4, self.V, self.scores.data_ptr(), None, 5, 4, self.so.data_ptr(), self.po.data_ptr(), self.to.data_ptr(),
                                   self.do.data_ptr())
        return rc | lib.ncmb_paged_reorder(self.c, 4, self.po.data_ptr(), 2, self.pool.stride(1), self.t2.data_ptr(), self.l2.data_ptr(), None)

    def results(self):
        return [x.clone() for x in (self.pool, self.q, self.out, self.out2, self.so, self.po, self.to, self.do, self.t2, self.l2)]

    def clear(self):
        self.pool.copy_(self.pool0)
        for x in (self.q, self.out, self.out2, self.so, self.po, self.to, self.do, self.t2, self.l2):
            x.zero_()
        torch.cuda.synchronize()


SHAPES = [(700, 16, 14, 2, 64, 5003, BF16), (3000, 64, 8, 4, 128, 50257, BF16), (500, 8, 12, 12, 64, 777, F32)]


def on(lib, stream):
    lib.ncmb_set_stream(stream.cuda_stream)
    return torch.cuda.stream(stream)


@pytest.mark.parametrize("shape", SHAPES)
def test_two_streams_in_turn(cuda, shape):
    a, b = Work(cuda, 1, *shape), Work(cuda, 2, *shape)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    want = []
    for x in (a, b):
        with on(cuda, s):
            assert x.run() == 0
        torch.cuda.synchronize()
        want.append(x.results())
        x.clear()
    for _ in range(15):
        for x, stream in ((a, s), (b, t)):
            with on(cuda, stream):
                assert x.run() == 0
    torch.cuda.synchronize()
    for x, w in zip((a, b), want):
        assert all(torch.equal(one, two) for one, two in zip(x.results(), w))


@pytest.mark.parametrize("shape", SHAPES)
def test_captured(cuda, shape):
    """Two graphs of one stream, and eager calls of another size between their replays."""
    a, b, c = Work(cuda, 3, *shape), Work(cuda, 4, *shape), Work(cuda, 5, 2000, 16, 14, 2, 64, 30011, BF16)
    s = torch.cuda.Stream()
    want, graphs = [], []
    with on(cuda, s):
        assert c.run() == 0
        for x in (a, b):
            assert x.run() == 0
            s.synchronize()
            want.append(x.results())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                assert x.run() == 0
            graphs.append(g)
            x.clear()
        for _ in range(5):
            for g in graphs:
                g.replay()
            assert c.run() == 0
    torch.cuda.synchronize()
    for x, w in zip((a, b), want):
        assert all(torch.equal(one, two) for one, two in zip(x.results(), w))


def test_capture_without_scratch(cuda):
    """On a stream that has made no scratch memory, calls that need some are refused and the capture goes on; those that need none are captured."""
    x = Work(cuda, 6, *SHAPES[1])
    s = torch.cuda.Stream(priority=-1)
    y = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with on(cuda, s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y += 1
            before = cuda.ncmb_launch_count()
            assert cuda.ncmb_beam_select(x.logits.data_ptr(), x.V, capi.F32, 12, 4, x.V, x.scores.data_ptr(), None, 5, 4, x.so.data_ptr(), x.po.data_ptr(), x.to.data_ptr(), None) in (0, -1)
            refused = cuda.ncmb_launch_count() == before
            p, w = x.qkv.data_ptr(), x.H * x.hd
            assert cuda.ncmb_paged_append(x.c, x.plan, p, w + 2 * x.nkv * x.hd, x.q.data_ptr(), w, x.H, p + w * 4, w + 2 * x.nkv * x.hd, p + (w + x.nkv * x.hd) * 4, w + 2 * x.nkv * x.hd,
                                          capi.F32, 48, None, None) == 0
        g.replay()
    torch.cuda.synchronize()
    assert (y == 1).all() and (x.q != 0).any() and (not refused or (x.to == 0).all())


def test_a_search_replayed():
    """A search whose steps are two graphs, replayed in turn, gives what eager steps give."""
    spec = importlib.util.spec_from_file_location("beam_search", os.path.join(helpers.ROOT, "examples", "beam_search.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    G, K, n, new = 2, 5, 61, 21
    w = ex.Weights(7)
    prompts = torch.randint(0, ex.VOCAB, (G, n), generator=torch.Generator().manual_seed(4))
    text, scores, _ = ex.search(w, prompts.tolist(), K, new, BF16)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        with on(ex.lib, stream):
            m = ex.Decoder(w, G, K, n, new, BF16)
            logits = m.forward(prompts.cuda().reshape(-1), m.firsts, G).view(G, -1, ex.VOCAB)[:, -1].contiguous()
            m.len[::K] = n
            state = m.select(logits, 1, torch.zeros(G, 1, device="cuda"), None)
            m.reorder(state[1])
            scores2, parents, tokens, done = (t.clone() for t in state)
            text2 = torch.zeros(G, K, new, dtype=torch.int32, device="cuda")
            text2[:, :, 0] = tokens
            at = torch.ones(1, dtype=torch.int64, device="cuda")

            def step():
                got = m.select(m.forward(tokens.view(-1).long(), m.caches[m.at], m.rows), K, scores2, done)
                (m.len2 if m.at else m.len).add_(1)
                m.reorder(got[1])
                for x, y in zip((scores2, parents, tokens, done), got):
                    x.copy_(y)
                text2.copy_(text2.gather(1, parents.long()[:, :, None].expand_as(text2)))
                text2.index_copy_(2, at, tokens[:, :, None])
                at.add_(1)

            keep = [t.clone() for t in (m.pool, m.table, m.table2, m.len, m.len2, scores2, parents, tokens, done, text2, at)]
            step(); step()                                        # makes the scratch memory; then all as it was
            stream.synchronize()
            for x, y in zip((m.pool, m.table, m.table2, m.len, m.len2, scores2, parents, tokens, done, text2, at), keep):
                x.copy_(y)
            stream.synchronize()
            graphs = []
            for _ in range(2):
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1], stream=stream):
                    step()
            for i in range(new - 1):
                graphs[i % 2].replay()
            stream.synchronize()
    finally:
        ex.lib.ncmb_set_stream(None)
    assert torch.equal(text2, text) and torch.equal(scores2, scores)
