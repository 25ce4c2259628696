"""capi.KVCache.of takes what the library can read and nothing else (CPU tensors: nothing is launched)."""
import pytest
import torch

import helpers

KVCache, F32, BF16 = helpers.capi.KVCache, helpers.capi.F32, helpers.capi.BF16


def views(dtype, rows=3):
    buf = torch.zeros(rows, 20, 2, 4, 16).to(dtype)
    return tuple(buf[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))


@pytest.mark.parametrize("dtype,kind", [(torch.float32, F32), (torch.bfloat16, BF16)])
def test_types_it_takes(dtype, kind):
    k, v = views(dtype)
    assert KVCache.of(k, v, torch.zeros(3, dtype=torch.int32)).type == kind


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32, torch.uint32, torch.int16, torch.int8, torch.complex32, torch.float8_e4m3fn])
def test_types_it_cannot_mean(dtype):
    k, v = views(dtype)
    with pytest.raises(ValueError):
        KVCache.of(k, v, torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("length", [torch.zeros(3, dtype=torch.int64), torch.zeros(3), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                                    torch.zeros(3, 1, dtype=torch.int32), torch.zeros((), dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2],
                                    torch.zeros(1, dtype=torch.int32).expand(3)])
def test_lengths_it_cannot_read(length):
    with pytest.raises(ValueError):
        KVCache.of(*views(torch.float32), length)


def test_lengths_of_one_row_and_of_none():
    for rows in (0, 1):
        k, v = views(torch.bfloat16, rows)
        assert KVCache.of(k, v, torch.zeros(2, dtype=torch.int32)[::2][:rows]).rows == rows


def test_shapes_and_places_it_cannot_mean():
    k, v = views(torch.float32)
    n = torch.zeros(3, dtype=torch.int32)
    for bad in ((k[0], v[0], n), (k, v.to("meta"), n), (k, v, n.to("meta"))):
        with pytest.raises(ValueError):
            KVCache.of(*bad)
