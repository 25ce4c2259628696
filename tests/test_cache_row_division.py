"""The wide tiles of ncmb_cache_attention find the token of a query row by an fp32 product instead of a division; here the same arithmetic, on the CPU,
over the range of rows that they take. And the range of rows that the call takes at all."""
import os
import re

import numpy as np

import helpers
import test_gpu_cache_operators as ops


def test_the_product_is_the_division_over_the_range():
    src = open(os.path.join(helpers.ROOT, "saphira-cncm_b200", "csrc", "cache_tc.cuh")).read()
    assert "t = (int)(((float)mm + 0.5f) * per_g)" in src and "per_g = 1.0f / (float)G" in src
    most = 1 << int(re.search(r"CT_MOST_ROWS = 1 << (\d+);", src).group(1))
    for G in list(range(1, 130)) + [255, 1000, 1023, 3001, 4095, 4096]:
        rows = np.arange(0, min(256 * G, most) + 128)
        t = ((rows.astype(np.float32) + np.float32(0.5)) * (np.float32(1) / np.float32(G))).astype(np.int64)
        assert (t == rows // G).all(), G
    # and at the ends of every token's rows where groups are larger
    for G in range(4097, most, 997):
        ends = np.arange(0, most + 128, G)
        rows = np.unique(np.concatenate([ends, ends + 1, ends[1:] - 1, [most + 127]]))
        t = ((rows.astype(np.float32) + np.float32(0.5)) * (np.float32(1) / np.float32(G))).astype(np.int64)
        assert (t == rows // G).all(), G


def test_more_rows_than_can_be_counted_are_refused():
    lib, p, H = helpers.capi.NcmLib(helpers.CUDA_LIB), 1 << 22, 1 << 24
    c = ops.fake_cache(n_kv=1, hd=8, capacity=300, token_stride=8, row_stride=4800)
    assert lib.ncmb_cache_attention(c, p, 8 * H, p, 8 * H, helpers.capi.F32, H, 256, None, 0.0, 0, None) == -1
