"""A call of the cache operators that is refused late -- for want of scratch memory -- has queued nothing."""
import pytest
import torch

import helpers
import test_gpu_cache_streams as streams

pytestmark = pytest.mark.gpu
capi = helpers.capi


@pytest.fixture(scope="module")
def cuda():
    lib = capi.NcmLib(helpers.CUDA_LIB)
    yield lib
    torch.cuda.synchronize()
    lib.ncmb_set_stream(None)


def test_block_attention_without_scratch_for_its_results(cuda):
    """In a capture on a stream that has made no scratch: the picks have room of the caller's, the results of many rows have none."""
    s = torch.cuda.Stream(priority=-1)                  # from a pool that no other test takes streams from
    with streams.on(cuda, s):
        x = streams.Work(cuda, 5, 40, 3000, 24, 14, 2, 64, False)
        picks = torch.full((40, 24, 2, 20), -9, dtype=torch.int32, device="cuda")
        y = torch.zeros(8, device="cuda")
        args = (x.c, x.q.data_ptr(), x.H * x.hd, x.out.data_ptr(), x.H * x.hd, capi.F32, x.H, x.T, 32, x.codes.data_ptr(), x.scales.data_ptr(), 20, 1, 2, 0.0, 0, picks.data_ptr())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y += 1
            before = cuda.ncmb_launch_count()
            assert cuda.ncmb_block_attention(*args) == -1
            assert cuda.ncmb_launch_count() == before
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 1).all() and (picks == -9).all() and (x.out == 0).all()
        assert cuda.ncmb_block_attention(*args) == 0
        torch.cuda.synchronize()
        assert (picks >= -1).all() and (x.out != 0).any()
