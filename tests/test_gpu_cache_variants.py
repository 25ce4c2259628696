"""ncmb_cache_attention with either kind of tiles (16 query rows on mma.sync, 128 on tcgen05) at sizes where the rule would take
only one of them. Bounds and inputs are test_gpu_cache_operators.py's and test_gpu_cache_nonfinite.py's."""
import pytest

import helpers
import test_gpu_cache_nonfinite as nonfinite
import test_gpu_cache_operators as ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[1, 2])
def cuda(request):
    lib = helpers.capi.NcmLib(helpers.CUDA_LIB)
    lib.ncmb_set_cache_variant(request.param)
    yield lib
    lib.ncmb_set_cache_variant(0)
    assert lib.ncmb_gemm_tc_check() == 0                # no wait ran out


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("hd,H,nkv", [(64, 14, 2), (128, 8, 2), (64, 3, 3), (40, 10, 2), (72, 5, 1), (128, 48, 3), (96, 1, 1)])
@pytest.mark.parametrize("T,tree", [(19, True), (33, False), (64, True)])
def test_shapes(cuda, kt, qt, hd, H, nkv, T, tree):
    ops.run_attention(cuda, 3 * hd + T, [0, 1, 40, 333], T, H, nkv, hd, kt, qt, ["token", "head", "gap"][(hd + T) % 3], tree, T % 2 == 1)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("n", [0, 1, 63, 64, 95, 96, 97, 127, 128, 129, 223, 224, 225, 256, 385])
def test_tile_ends(cuda, kt, qt, n):
    ops.run_attention(cuda, n, [n, max(0, n - 1)], 32, 4, 2, 64, kt, qt, "token", True, True, cap=n + 32)
    ops.run_attention(cuda, n, [n], 31, 4, 2, 128, kt, qt, "head", False, True, cap=n + 31)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", [(24, 14, 2, 64), (16, 32, 8, 128), (100, 14, 2, 64), (256, 4, 1, 64)])
def test_long_rows(cuda, kt, qt, T, H, nkv, hd):
    ops.run_attention(cuda, T, [9001], T, H, nkv, hd, kt, qt, "token", True, True)
    ops.run_attention(cuda, T, [5000, 3, 12000], T, H, nkv, hd, kt, qt, "head", True, False, max_len=700)
    ops.run_attention(cuda, T, [300, 70], T, H, nkv, hd, kt, qt, "token", False, False, scale=-0.25)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
@pytest.mark.parametrize("T,H,nkv,hd", [(12, 14, 2, 64), (40, 14, 2, 64), (33, 8, 2, 128), (30, 5, 1, 40)])
@pytest.mark.parametrize("n", [0, 61, 700])
def test_unseen_tokens(cuda, kt, qt, T, H, nkv, hd, n):
    nonfinite.test_unseen_tokens(cuda, kt, qt, T, H, nkv, hd, n)


@pytest.mark.parametrize("kt,qt", ops.TYPES)
def test_tokens_to_come_and_weights(cuda, kt, qt):
    nonfinite.test_tokens_to_come(cuda, kt, qt, 20, 14, 2, 64)
    nonfinite.test_tokens_to_come(cuda, kt, qt, 33, 8, 2, 128)
    nonfinite.test_weights_of_unseen_tokens(cuda, kt, qt)
