"""The cache operators on several streams and in stream captures: scratch memory belongs to a stream, and a graph keeps what it uses."""
import numpy as np
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    lib = capi.NcmLib(helpers.CUDA_LIB)
    yield lib
    torch.cuda.synchronize()
    lib.ncmb_set_stream(None)
    lib.ncmb_set_cache_variant(0)
    assert lib.ncmb_gemm_tc_check() == 0


class Work:
    """One call of each kind on tensors of its own. `run` queues them, `results` are what they wrote."""

    def __init__(self, lib, seed, B, n, T, H, nkv, hd, weights):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.lib, self.T, self.H, self.hd, self.cap, self.max_len = lib, T, H, hd, n + T, n
        self.k, self.v = r(B, nkv, n + T, hd).to(BF16), r(B, nkv, n + T, hd).to(BF16)
        self.len = torch.tensor([max(0, n - 300 * b) for b in range(B)], dtype=torch.int32, device="cuda")
        self.c = capi.KVCache.of(self.k, self.v, self.len)
        self.q = r(B, T, H, hd)
        self.w0 = torch.rand(B, nkv, n + T, device="cuda", generator=g) if weights else None
        self.w = torch.zeros_like(self.w0) if weights else None
        self.codes = torch.randint(-127, 128, (B, nkv, -(-(n + T) // 32), hd), dtype=torch.int8, device="cuda", generator=g)
        self.scales = torch.rand(self.codes.shape[:3], device="cuda", generator=g)
        self.out, self.out2 = torch.zeros_like(self.q), torch.zeros_like(self.q)
        room = n // 3
        self.k2, self.v2 = (torch.zeros(B, nkv, room, hd, dtype=BF16, device="cuda") for _ in range(2))
        self.w2, self.pos, self.pos2 = torch.zeros(B, nkv, room, device="cuda"), torch.zeros(B, nkv, n + T, dtype=torch.int32, device="cuda"), torch.zeros(B, nkv, room, dtype=torch.int32, device="cuda")
        self.ew, self.room = torch.rand(B, nkv, n + T, device="cuda", generator=g), room
        self.left = torch.zeros_like(self.len)
        self.c2 = capi.KVCache.of(self.k2, self.v2, self.left)
        torch.cuda.synchronize()

    def run(self):
        lib, ld = self.lib, self.H * self.hd
        if self.w is not None:
            self.w.copy_(self.w0)
        rc = lib.ncmb_cache_attention(self.c, self.q.data_ptr(), ld, self.out.data_ptr(), ld, capi.F32, self.H, self.T, None, 0.0, self.max_len,
                                      self.w.data_ptr() if self.w is not None else None)
        rc |= lib.ncmb_block_attention(self.c, self.q.data_ptr(), ld, self.out2.data_ptr(), ld, capi.F32, self.H, self.T, 32, self.codes.data_ptr(), self.scales.data_ptr(),
                                       20, 1, 2, 0.0, self.max_len, None)
        self.left.copy_(self.len)                       # tokens seen, then the new lengths
        rc |= lib.ncmb_cache_evict(self.c, self.c2, self.ew.data_ptr(), self.w2.data_ptr(), self.pos.data_ptr(), self.pos2.data_ptr(), None, self.left.data_ptr(), self.room, 64,
                                   self.max_len, self.left.data_ptr())
        return rc

    def results(self):
        return [x.clone() for x in (self.out, self.out2, self.k2, self.v2, self.w2, self.pos2, self.left) + ((self.w,) if self.w is not None else ())]

    def clear(self):
        for x in (self.out, self.out2, self.k2, self.v2, self.w2, self.pos2, self.left):
            x.zero_()
        torch.cuda.synchronize()


SHAPES = [(4, 6000, 1, 14, 2, 64, False), (4, 6000, 5, 14, 2, 64, True), (3, 5000, 24, 14, 2, 64, True), (2, 4000, 40, 8, 2, 128, False)]


def on(lib, stream):
    lib.ncmb_set_stream(stream.cuda_stream)
    return torch.cuda.stream(stream)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_two_streams_in_turn(cuda, variant, shape):
    cuda.ncmb_set_cache_variant(variant)
    a, b = Work(cuda, 1, *shape), Work(cuda, 2, *shape)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    want = []
    for x in (a, b):
        with on(cuda, s):
            assert x.run() == 0
        torch.cuda.synchronize()
        want.append(x.results())
        x.clear()
    for i in range(20):
        for x, stream in ((a, s), (b, t)):
            with on(cuda, stream):
                assert x.run() == 0
    torch.cuda.synchronize()
    for x, w in zip((a, b), want):
        for one, two in zip(x.results(), w):
            assert torch.equal(one, two)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_graph_outlives_larger_calls(cuda, variant, shape):
    """Captured, then a call on the same stream that needs more scratch, then replayed."""
    cuda.ncmb_set_cache_variant(variant)
    s = torch.cuda.Stream()
    x = Work(cuda, 3, *shape)
    with on(cuda, s):
        assert x.run() == 0
    torch.cuda.synchronize()
    want = x.results()
    graph = torch.cuda.CUDAGraph()
    with on(cuda, s):
        with torch.cuda.graph(graph, stream=s):
            assert x.run() == 0
    B, n, *rest = shape
    big = Work(cuda, 4, 3 * B, n, *rest)
    with on(cuda, s):
        assert big.run() == 0
    torch.cuda.synchronize()
    first = big.results()
    held = [torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]      # what was free is somebody else's now
    for _ in range(3):
        x.clear()
        with on(cuda, s):
            graph.replay()
            assert big.run() == 0
        torch.cuda.synchronize()
        for one, two in zip(x.results() + big.results(), want + first):
            assert torch.equal(one, two)
    assert all(bool((h == 7).all()) for h in held)


@pytest.mark.parametrize("variant", [1, 2])
def test_growth_in_a_capture_is_refused_and_the_capture_goes_on(cuda, variant, capfd):
    cuda.ncmb_set_cache_variant(variant)
    s = torch.cuda.Stream()
    with on(cuda, s):                                   # a stream id of its own: torch hands out streams from a pool
        x, big = Work(cuda, 5, 2, 3000, 24, 14, 2, 64, True), Work(cuda, 6, 40, 3000, 64, 14, 2, 64, True)
        assert x.run() == 0
        torch.cuda.synchronize()
        want = x.results()
        y = torch.zeros(8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert x.run() == 0
            launches = cuda.ncmb_launch_count()
            assert cuda.ncmb_cache_attention(big.c, big.q.data_ptr(), big.H * big.hd, big.out.data_ptr(), big.H * big.hd, capi.F32, big.H, big.T, None, 0.0, 0, big.w.data_ptr()) == -1
            assert cuda.ncmb_launch_count() == launches
            y += 1
        x.clear()
        graph.replay()
        torch.cuda.synchronize()
    assert "while the stream is captured" in capfd.readouterr().err
    assert (y == 1).all()
    for one, two in zip(x.results(), want):
        assert torch.equal(one, two)
