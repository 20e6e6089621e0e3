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
    assert L.tcb_cache_write(p + 16, 0, p, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_cache_write(p, 0, p + 4, 4, p, p, 10, 64, 32, p, None) == _lib.ERR_ALIGNMENT
    assert L.tcb_cache_write(p, 0, p, 1 << 31, p, p, 10, 64, 32, p, None) == _lib.ERR_TOO_LARGE
    assert L.tcb_cache_read(p, p, 10, 64, 32, p, -1, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_read(None, p, 10, 64, 32, p, 4, p, None) == _lib.ERR_BAD_ARG
    assert L.tcb_cache_read(p, p, 10, 64, 7, p, 4, p, None) == _lib.ERR_GROUP_SIZE
    assert L.tcb_cache_read(p, p, 10, 64, 32, p, 0, p, None) == _lib.TCB_OK


def test_mxfp4_product_refusals(built_lib):
    from tensorcache_b200 import _lib

    L, p = built_lib, 1 << 20
    need = L.tcb_mxfp4_linear_workspace(40, 8, 64)
    assert need == 40 * 32 + 256 + 512 and L.tcb_mxfp4_linear_workspace(0, 8, 64) == 0 and L.tcb_mxfp4_linear_workspace(4, 8, 64) == 0
    f = lambda *a: L.tcb_mxfp4_linear(*a, None)  # noqa: E731
    assert f(None, 0, None, None, None, None, 0, 8, 64, None, 0) == _lib.TCB_OK
    assert f(p, 3, p, p, None, p, 4, 8, 64, p, need) == _lib.ERR_BAD_ARG            # dtype
    assert f(p, 0, p, p, None, p, 4, 8, 48, p, need) == _lib.ERR_BAD_ARG            # K % 32
    assert f(p, 0, p, p, None, p, 4, -8, 64, p, need) == _lib.ERR_BAD_ARG
    assert f(p, 0, None, p, None, p, 4, 8, 64, p, need) == _lib.ERR_BAD_ARG
    assert f(p + 8, 0, p, p, None, p, 4, 8, 64, p, need) == _lib.ERR_ALIGNMENT
    assert f(p, 0, p, p, None, p + 1, 4, 8, 64, p, need) == _lib.ERR_ALIGNMENT
    assert f(p, 0, p, p, None, p, 40, 8, 64, p, need - 1) == _lib.ERR_BAD_ARG       # workspace
    assert f(p, 0, p, p, None, p, 1 << 31, 8, 64, p, need) == _lib.ERR_TOO_LARGE
    x, wq, ws = torch.zeros(4, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    for bad, match in (((x[:, :32], wq, ws), "inner dimensions"), ((x, wq.view(-1), ws), "wq"), ((x, wq, ws[:-1]), "scales"),
                       ((x, wq.to(torch.int8), ws), "uint8"), ((x.double(), wq, ws), "fp32"), ((x, wq, ws, torch.zeros(8)), "bias"),
                       ((x.clone().requires_grad_(True), wq, ws), "no gradient")):
        with pytest.raises(ValueError, match=match):
            tc.mxfp4_matmul(*bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        tc.mxfp4_matmul(x, wq, ws)


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


def test_linear_entry_points_refuse_bad_arguments(built_lib):
    from tensorcache_b200 import _lib

    L, p = built_lib, 1 << 20
    fwd = lambda *a: L.tcb_linear_forward(*a, None)  # noqa: E731
    assert fwd(None, None, None, None, None, None, 0, 8, 32, 32, None, 0) == _lib.TCB_OK
    assert fwd(p, p, None, p, None, None, 4, 8, 12, 32, p, 0) == _lib.ERR_BAD_ARG            # K % 8
    assert fwd(p, p, None, p, None, None, 4, -8, 16, 32, p, 0) == _lib.ERR_BAD_ARG
    assert fwd(None, p, None, p, None, None, 4, 8, 16, 32, p, 0) == _lib.ERR_BAD_ARG
    assert fwd(p + 2, p, None, p, None, None, 4, 8, 16, 32, p, 0) == _lib.ERR_ALIGNMENT
    assert fwd(p, p, p + 1, p, None, None, 4, 8, 16, 32, p, 0) == _lib.ERR_ALIGNMENT
    assert fwd(p, p, None, p, None, None, 1 << 31, 8, 16, 32, p, 0) == _lib.ERR_TOO_LARGE
    assert fwd(p, p, None, p, p, p, 4, 8, 48, 24, p, 0) == _lib.ERR_GROUP_SIZE
    assert fwd(p, p, None, p, p, p, 4, 8, 48, 32, p, 0) == _lib.ERR_BAD_ARG                  # K % G
    assert fwd(p, p, None, p, p, None, 4, 8, 64, 32, p, 0) == _lib.ERR_BAD_ARG               # codes without scales
    bwd = lambda *a: L.tcb_linear_backward(*a, None)  # noqa: E731
    assert bwd(p, 8, p, p, p, None, p, p, p, 4, 16, 32, 32, p, 0) == _lib.ERR_BAD_ARG        # ld < N
    assert bwd(p, 20, p, p, p, None, p, p, p, 4, 16, 32, 32, p, 0) == _lib.ERR_BAD_ARG       # ld % 8
    assert bwd(p, 8, p, p, p, None, None, p, None, 4, 8, 32, 24, p, 0) == _lib.ERR_GROUP_SIZE
    assert bwd(p, 8, p, p, p, None, None, p, None, 4, 8, 48, 32, p, 0) == _lib.ERR_BAD_ARG
    assert bwd(p, 8, p, p, None, None, None, p, None, 4, 8, 32, 32, p, 0) == _lib.ERR_BAD_ARG    # scales missing
    assert bwd(p, 8, p, p, p, None, None, p + 2, None, 4, 8, 32, 32, p, 0) == _lib.ERR_ALIGNMENT  # dw
    assert bwd(p, 8, None, p, p, None, p, None, None, 4, 8, 32, 32, p, 0) == _lib.ERR_BAD_ARG    # weight missing
    assert bwd(p, 8, None, None, None, None, None, None, p, 4, 8, 32, 32, p, 4) == _lib.ERR_BAD_ARG  # workspace too small
    assert L.tcb_linear_workspace(0, 8, 32, 7) == 0 and L.tcb_linear_workspace(4, 8, 32, 0) == 0 and L.tcb_linear_workspace(4, 8, 32, 3) == 0
    assert L.tcb_linear_workspace(4, 8, 32, 4) > 0 and L.tcb_linear_workspace(100000, 8, 32, 2) > 0 and L.tcb_linear_workspace(4, 8, 4096, 0) > 0


def test_linear_layer_refusals():
    bf = torch.bfloat16
    x, w, b = torch.zeros(4, 64, dtype=bf), torch.zeros(8, 64, dtype=bf), torch.zeros(8, dtype=bf)
    for bad, match in (((x.float(), w, b), "bf16"), ((x, w.float(), b), "bf16"), ((x, w, b.float()), "bf16"), ((x, w[:, :32], b), "weight"),
                       ((x, w, b[:4]), "bias"), ((x, w[0], b), "weight"), ((x[:, :24], w[:, :24], b), "multiple")):
        with pytest.raises(ValueError, match=match):
            tc.int8_checkpoint_linear(*bad)
    with pytest.raises(ValueError, match="group_size"):
        tc.int8_checkpoint_linear(x, w, b, group_size=24)
    with pytest.raises(RuntimeError, match="CUDA"):
        tc.int8_checkpoint_linear(x, w, b)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(8, dtype=bf)
    with pytest.raises(RuntimeError, match="CUDA"):
        tc.fused_dequant_linear(q, s, w, b)
    with pytest.raises(ValueError, match="scales"):
        tc.fused_dequant_linear(q, s[:-1], w, b)
    with pytest.raises(ValueError, match="int8"):
        tc.fused_dequant_linear(q.to(torch.uint8), s, w, b)


def test_operands_whose_gradient_would_be_dropped_are_refused():
    from torch.autograd import forward_ad

    bf = torch.bfloat16
    x, wq, ws = torch.zeros(4, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    b = torch.zeros(8, dtype=bf)
    q, s, w = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(8, dtype=bf), torch.zeros(8, 64, dtype=bf)
    calls = {"x": (lambda t: tc.mxfp4_matmul(t, wq, ws, b), x), "bias": (lambda t: tc.mxfp4_matmul(x, wq, ws, bias=t), b),
             "scales": (lambda t: tc.fused_dequant_linear(q, t, w, b), s)}
    for name, (call, t) in calls.items():
        wants = t.clone().requires_grad_(True)
        with pytest.raises(ValueError, match=f"{name} has no gradient"):
            call(wants)
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match=f"{name} has no gradient.* tangent"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(RuntimeError, match="CUDA"):      # nothing to refuse but the device
                call(t)
        for allowed in (wants.detach(), wants):
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
                call(allowed)
