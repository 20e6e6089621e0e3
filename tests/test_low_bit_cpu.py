"""Refusals and host-side logic of the low-bit operators (no GPU)."""
import pytest
import torch

import tensorcache_b200 as tc
from tests import low_bit_plain as plain


def test_library_refuses_bad_arguments_before_any_device_work(built_lib):
    from tensorcache_b200 import _lib

    L = built_lib
    p = 1 << 20   # a 16-byte aligned address that is never dereferenced: every call below is refused first
    assert L.tcb_quantize_mxfp4(None, 0, 0, 64, None, None, None) == _lib.TCB_OK
    assert L.tcb_quantize_mxfp4(p, 3, 4, 64, p, p, None) == _lib.ERR_BAD_ARG          # dtype
    assert L.tcb_quantize_mxfp4(p, 0, 4, 48, p, p, None) == _lib.ERR_BAD_ARG          # not a multiple of 32
    assert L.tcb_quantize_mxfp4(p, 0, -1, 64, p, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_quantize_mxfp4(None, 0, 4, 64, p, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_quantize_mxfp4(p + 2, 0, 4, 64, p, p, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_quantize_mxfp4(p, 0, 1 << 40, 1 << 10, p, p, None) == _lib.ERR_TOO_LARGE
    assert L.tcb_dequantize_mxfp4(None, None, 0, 64, None, None) == _lib.TCB_OK
    assert L.tcb_dequantize_mxfp4(p, p, 4, 33, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_dequantize_mxfp4(p, p, 4, 64, p + 8, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_cache_write(p, 0, p, 0, p, p, 10, 64, 32, p, None) == _lib.TCB_OK
    assert L.tcb_cache_write(p, 5, p, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_write(p, 0, p, 4, p, p, 10, 64, 20, p, None) == _lib.ERR_GROUP_SIZE
    assert L.tcb_cache_write(p, 0, p, 4, p, p, 10, 72, 32, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_write(p, 0, p, 4, p, p, 10, 64, 32, None, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_write(p, 0, None, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_write(p + 4, 0, p, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_cache_write(p, 0, p + 4, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_cache_write(p, 0, p, 1 << 31, p, p, 10, 64, 32, p, None) == _lib.ERR_TOO_LARGE
    assert L.tcb_cache_read(p, p, 10, 64, 32, p, -1, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_read(None, p, 10, 64, 32, p, 4, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_read(p, p, 10, 64, 7, p, 4, p, None) == _lib.ERR_GROUP_SIZE
    assert L.tcb_cache_read(p, p, 10, 64, 32, p, 0, p, None) == _lib.TCB_OK


def test_mxfp4_refusals():
    with pytest.raises(ValueError, match="multiple of 32"):
        tc.quantize_mxfp4(torch.zeros(4, 33))
    with pytest.raises(ValueError, match="0-dimensional"):
        tc.quantize_mxfp4(torch.zeros(()))
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(ValueError, match="bytes of codes"):
        tc.dequantize_mxfp4(codes, scales, (4, 64))
    with pytest.raises(ValueError, match="scales"):
        tc.dequantize_mxfp4(codes, scales[:-1], (4, 32))
    with pytest.raises(ValueError, match="uint8"):
        tc.dequantize_mxfp4(codes.to(torch.int8), scales, (4, 32))
    with pytest.raises(ValueError, match="scales"):
        tc.mxfp4_scales_to_rows(scales, 129, 32)
    with pytest.raises(ValueError, match="uint8"):
        tc.mxfp4_scales_from_rows(torch.zeros(4, 2))


@pytest.mark.parametrize("rows,cols", [(1, 32), (128, 128), (129, 160), (300, 992)])
def test_scale_tiles_follow_the_documented_order(rows, cols):
    per_row = torch.randint(0, 256, (rows, cols // 32), dtype=torch.uint8, generator=torch.Generator().manual_seed(rows))
    tiles = tc.mxfp4_scales_from_rows(per_row)
    assert tiles.numel() == -(-rows // 128) * -(-cols // 128) * 512
    used = torch.zeros(tiles.numel(), dtype=torch.bool)
    for r in range(rows):
        for b in range(cols // 32):
            at = plain.mx_scale_offset(r, b, cols)
            assert int(tiles[at]) == int(per_row[r, b])
            used[at] = True
    assert not bool(tiles[~used].any())
    assert torch.equal(tc.mxfp4_scales_to_rows(tiles, rows, cols), per_row)


def test_device_cache_refusals():
    with pytest.raises(ValueError, match="group_size"):
        tc.DeviceFeatureCache(4, 64, group_size=20)
    with pytest.raises(ValueError, match="multiple of the group size"):
        tc.DeviceFeatureCache(4, 72, group_size=32)
    with pytest.raises(ValueError, match="negative"):
        tc.DeviceFeatureCache(-1, 64)
    if torch.cuda.is_available():
        with pytest.raises(ValueError, match="CUDA device"):
            tc.DeviceFeatureCache(4, 64, device="cpu")
        cache = tc.DeviceFeatureCache(4, (2, 32))
        with pytest.raises(IndexError):
            cache.write([4], torch.zeros(1, 2, 32))
        with pytest.raises(IndexError):
            cache.read([0, 4])
        with pytest.raises(ValueError, match="rows"):
            cache.write([0], torch.zeros(2, 64))
        with pytest.raises(ValueError, match="int64"):
            cache.read(torch.zeros(2))
        with pytest.raises(ValueError, match="one-dimensional"):
            cache.read(torch.zeros(1, 2, dtype=torch.int64))
        with pytest.raises(ValueError, match="out_buffer"):
            cache.read([0], out_buffer=torch.zeros(64))
    else:
        with pytest.raises(RuntimeError, match="CUDA device"):
            tc.DeviceFeatureCache(4, 64)
