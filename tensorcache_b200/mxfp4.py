"""Microscaled 4-bit floating point (MXFP4): codec and matrix product.

Blocks of 32 values along the last dimension, E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) and one power-of-two scale byte per block: 4.25 bits a value, a quarter of bf16.  The 8-bit
codecs next door (``compress`` / ``decompress``) have no 4-bit counterpart in the reference that keeps its
scales as powers of two, so there is nothing to mirror here; argument checks, staging of CPU tensors and
errors follow ``codec.py``.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .codec import _DTYPES, _compute_device
from .fused_linear import _operand_on, _refuse_gradient

BLOCK = 32          # values that share a scale
_TILE_ROWS = 128    # a scale tile covers 128 rows x 4 blocks
_TILE_BLOCKS = 4


def _rows_cols(shape) -> Tuple[int, int]:
    if len(shape) == 0:
        raise ValueError("MXFP4 blocks run along the last dimension: a 0-dimensional tensor has none")
    cols = int(shape[-1])
    if cols % BLOCK != 0:
        raise ValueError(f"the last dimension ({cols}) must be a multiple of {BLOCK}")
    return int(shape[0]) if len(shape) == 2 else math.prod(shape[:-1]), cols


def mxfp4_scale_bytes(rows: int, cols: int) -> int:
    """Number of scale bytes of a ``[rows, cols]`` tensor: whole tiles of 128 rows x 128 values."""
    return -(-rows // _TILE_ROWS) * -(-cols // (BLOCK * _TILE_BLOCKS)) * 512


def mxfp4_scales_to_rows(scales: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """Scale bytes in tile order -> uint8 ``[rows, cols / 32]`` (one row of scales per row of codes)."""
    _rows_cols((rows, cols))
    if scales.dtype != torch.uint8 or scales.numel() != mxfp4_scale_bytes(rows, cols):
        raise ValueError(f"expected {mxfp4_scale_bytes(rows, cols)} uint8 scales, got {scales.numel()} of {scales.dtype}")
    tr, tk = -(-rows // _TILE_ROWS), -(-cols // (BLOCK * _TILE_BLOCKS))
    t = scales.reshape(tr, tk, 32, 4, _TILE_BLOCKS).permute(0, 3, 2, 1, 4)
    return t.reshape(tr * _TILE_ROWS, tk * _TILE_BLOCKS)[:rows, :cols // BLOCK].contiguous()


def mxfp4_scales_from_rows(row_scales: torch.Tensor) -> torch.Tensor:
    """uint8 ``[rows, cols / 32]`` -> scale bytes in the tile order the kernels read (padding 0)."""
    if row_scales.dim() != 2 or row_scales.dtype != torch.uint8:
        raise ValueError("row scales are a uint8 tensor [rows, cols / 32]")
    rows, blocks = row_scales.shape
    tr, tk = -(-rows // _TILE_ROWS), -(-blocks // _TILE_BLOCKS)
    t = torch.zeros((tr * _TILE_ROWS, tk * _TILE_BLOCKS), dtype=torch.uint8, device=row_scales.device)
    t[:rows, :blocks] = row_scales
    return t.view(tr, 4, 32, tk, _TILE_BLOCKS).permute(0, 3, 2, 1, 4).reshape(-1)


def quantize_mxfp4(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, Tuple[int, ...]]:
    """Encode -> ``(codes uint8 [..., K / 2], scales uint8 [...], orig_shape)`` on ``x.device``.

    The last dimension K is a multiple of 32.  Element 2i of a row is the low half of byte i; the scales
    are in tile order (``mxfp4_scales_to_rows`` gives them per row).  A block's scale is
    ``2^(floor(log2 max|x|) - 2)``, codes round to nearest even and saturate at 6, values that are not
    finite become 0.  Inputs other than bf16, fp16 and fp32 are converted to fp32.  For CUDA inputs nothing
    synchronises with the host, so the call can be captured in a CUDA graph.
    """
    rows, cols = _rows_cols(x.shape)
    if x.dtype not in _DTYPES:
        x = x.float()
    dev = _compute_device(x)
    with _lib.on_device(dev):
        codes = torch.empty((rows, cols // 2) if x.dim() == 2 else (*x.shape[:-1], cols // 2), dtype=torch.uint8, device=dev)
        scales = codes.new_empty(mxfp4_scale_bytes(rows, cols))
        if rows and cols:
            xd = _operand_on(x, dev, 32)
            _lib.check(_lib.lib().tcb_quantize_mxfp4(xd.data_ptr(), _DTYPES[x.dtype], rows, cols, codes.data_ptr(), scales.data_ptr(),
                                                     _lib.stream_of(dev)))
    if not x.is_cuda:
        codes, scales = codes.cpu(), scales.cpu()
    return codes, scales, x.shape


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int) -> None:
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("MXFP4 operands are uint8 codes with uint8 scales")
    if codes.numel() * 2 != rows * cols:
        raise ValueError(f"expected {rows * cols // 2} bytes of codes for [{rows}, {cols}], got {codes.numel()}")
    if scales.numel() != mxfp4_scale_bytes(rows, cols):
        raise ValueError(f"expected {mxfp4_scale_bytes(rows, cols)} scales in tile order for [{rows}, {cols}], got {scales.numel()}")
    if codes.device != scales.device:
        raise ValueError(f"codes and scales are on different devices ({codes.device}, {scales.device})")


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, orig_shape: Tuple[int, ...],
                     out_buffer: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode to bf16 of ``orig_shape`` (exact: a code has two significant bits).  If ``out_buffer`` is given
    it is written in place and returned.  A scale byte of 255 decodes to NaN."""
    rows, cols = _rows_cols(orig_shape)
    _check_codes(codes, scales, rows, cols)
    dev = _compute_device(codes)
    if out_buffer is None:
        out_buffer = torch.empty(tuple(orig_shape), dtype=torch.bfloat16, device=codes.device)
    elif out_buffer.numel() != rows * cols or out_buffer.dtype != torch.bfloat16:
        raise ValueError("out_buffer must be a bf16 tensor of the decoded size")
    else:
        increment_version(out_buffer)   # the kernel writes through its address
    if rows == 0 or cols == 0:
        return out_buffer
    with _lib.on_device(dev):
        cd, sd = _operand_on(codes, dev, 16), _operand_on(scales, dev, 16)
        direct = out_buffer.device == dev and out_buffer.is_contiguous() and out_buffer.data_ptr() % 32 == 0
        od = out_buffer if direct else torch.empty(rows * cols, dtype=torch.bfloat16, device=dev)
        _lib.check(_lib.lib().tcb_dequantize_mxfp4(cd.data_ptr(), sd.data_ptr(), rows, cols, od.data_ptr(), _lib.stream_of(dev)))
        if not direct:
            out_buffer.copy_(od.view(out_buffer.shape))
    return out_buffer


@lru_cache(maxsize=1024)
def _workspace_bytes(M: int, N: int, K: int, device_index: int) -> int:
    """Scratch bytes of a product of these sizes (which kernel runs depends on the device's number of SMs)."""
    return _lib.lib().tcb_mxfp4_linear_workspace(M, N, K)


def mxfp4_matmul(x: torch.Tensor, wq: torch.Tensor, w_scales: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mxfp4(x) @ dequant(W).T (+ bias)`` on the 4-bit tensor cores, with W stored as MXFP4 (``wq`` uint8 ``[N, K / 2]``,
    ``w_scales`` in tile order, both as ``quantize_mxfp4`` returns them for ``[N, K]``).

    ``x`` is bf16, fp16 or fp32 ``[..., K]`` and is quantised by the call, each row in blocks of 32 as ``quantize_mxfp4`` does it:
    infinities and NaN count as 0 and do NOT show in the result (test ``x.isfinite()`` where that matters).  The result is bf16
    ``[..., N]``, summed in fp32 and rounded once.  The counterpart of ``fused_dequant_matmul`` for 4-bit weights, and
    like it without a gradient: an ``x`` or ``bias`` that requires one (or carries a forward-mode tangent) is refused.  CUDA tensors only.
    """
    if wq.dim() != 2 or x.dim() == 0:
        raise ValueError(f"x must be [..., K] and wq [N, K / 2], got {tuple(x.shape)} and {tuple(wq.shape)}")
    N, K = wq.shape[0], wq.shape[1] * 2
    if K <= 0 or K % BLOCK != 0 or x.shape[-1] != K:
        raise ValueError(f"the inner dimensions must agree and be a positive multiple of {BLOCK}, got {x.shape[-1]} and {K}")
    _check_codes(wq, w_scales, N, K)
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != N or bias.dtype != torch.bfloat16 or bias.device != x.device):
        raise ValueError(f"bias must be bf16 [{N}] on {x.device}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    if wq.device != x.device:
        raise ValueError(f"x is on {x.device}, the weight on {wq.device}")
    _refuse_gradient("mxfp4_matmul: x", x)
    if bias is not None:
        _refuse_gradient("mxfp4_matmul: bias", bias)
    if not x.is_cuda:
        raise RuntimeError("mxfp4_matmul runs on CUDA tensors only (no CPU fallback)")
    dev = x.device
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    out = torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    if M and N:
        with _lib.on_device(dev):
            x2, cd, sd = _operand_on(x2, dev, 32), _operand_on(wq, dev, 16), _operand_on(w_scales, dev, 16)
            b = None if bias is None else bias.contiguous()
            nbytes = _workspace_bytes(M, N, K, dev.index)     # x in MXFP4; 0 for few rows
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            _lib.check(_lib.lib().tcb_mxfp4_linear(x2.data_ptr(), _DTYPES[x2.dtype], cd.data_ptr(), sd.data_ptr(), _lib.address(b), out.data_ptr(),
                                                   M, N, K, _lib.address(ws), nbytes, _lib.stream_of(dev)))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], N)
