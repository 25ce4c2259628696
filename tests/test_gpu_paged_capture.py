"""Captures of beam and paged-cache calls on a stream whose scratch memory is too small: refused with nothing queued, taken after one call without a capture."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
capi = helpers.capi


def test_a_capture_that_needs_more_scratch():
    cuda = capi.NcmLib(helpers.CUDA_LIB)
    G, K, V, n = 512, 128, 300, 128                             # 65536 rows with 128 keys each: 67 MB, more than any other call of the tests leaves
    x = torch.randn(G * K, V, device="cuda")
    scores = -torch.rand(G, K, device="cuda")
    out = [torch.zeros(G, n, device="cuda")] + [torch.zeros(G, n, dtype=torch.int32, device="cuda") for _ in range(2)]
    call = lambda: cuda.ncmb_beam_select(x.data_ptr(), V, capi.F32, G, K, V, scores.data_ptr(), None, -1, n, *(o.data_ptr() for o in out), None)
    y = torch.zeros(8, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        cuda.ncmb_set_stream(s.cuda_stream)
        with torch.cuda.stream(s):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                y += 1
                before = cuda.ncmb_launch_count()
                assert call() == -1 and cuda.ncmb_launch_count() == before
            graph.replay()
            s.synchronize()
            assert (y == 1).all() and not out[0].any()
            assert call() == 0
            s.synchronize()
            want = [o.clone() for o in out]
            for o in out:
                o.zero_()
            again = torch.cuda.CUDAGraph()
            with torch.cuda.graph(again, stream=s):
                assert call() == 0
            again.replay()
            s.synchronize()
    finally:
        cuda.ncmb_set_stream(None)
    assert want[0].any() and all(torch.equal(a, b) for a, b in zip(want, out))
