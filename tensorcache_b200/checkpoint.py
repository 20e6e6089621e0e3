"""Linear layers that train with their input kept in 8 bits.

* ``int8_checkpoint_linear(x, weight, bias)`` / ``Int8CheckpointLinear``: ``x @ weight.T + bias`` whose graph
  keeps ``quantize_int8_g32(x)`` instead of ``x`` (``1 + 2 / group_size`` bytes a value instead of 2).
* ``fused_dequant_linear(q, scales, weight, bias, zero_points)``: the product of ``FusedDequantLinear`` on codes
  that come out of a feature cache, differentiable in ``weight`` and ``bias``.

The weight gradient is computed from the codes: the kernel decodes them in shared memory, so the bf16 input never
exists again.  Products run on the tensor cores with fp32 sums and one rounding to bf16; a long sum over few output
tiles is split over the GPU and added in a fixed order, so results do not change from run to run.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .fused_linear import SUPPORTED_GROUP_SIZES, _check_common, _launch, _operand_on, _refuse_gradient


def _check_dense(name: str, t: torch.Tensor, device: torch.device) -> None:
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bf16, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the input is on {device}")


def _check_layer(weight: torch.Tensor, bias: Optional[torch.Tensor], K: int, device: torch.device) -> None:
    if weight.dim() != 2 or weight.shape[1] != K:
        raise ValueError(f"weight must be [out_features, {K}], got {tuple(weight.shape)}")
    _check_dense("weight", weight, device)
    if bias is not None:
        if tuple(bias.shape) != (weight.shape[0],):
            raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
        _check_dense("bias", bias, device)


def _operand(t: torch.Tensor) -> torch.Tensor:
    return _operand_on(t, t.device, 16)


@lru_cache(maxsize=1024)
def _workspace_bytes(M: int, N: int, K: int, gradients: int, device_index: int) -> int:
    """Scratch bytes of a pass of these sizes (they depend on the device's number of SMs)."""
    return _lib.lib().tcb_linear_workspace(M, N, K, gradients)


def _workspace(M: int, N: int, K: int, gradients: int, device: torch.device):
    """(buffer or None, bytes): the split sums of one call, from the caching allocator of the current stream."""
    nbytes = _workspace_bytes(M, N, K, gradients, device.index)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


def _backward(dy: torch.Tensor, sizes, weight, q, scales, zp, group_size: int, need_dx: bool, need_dw: bool, need_db: bool):
    """``(dx, dw, db)`` of a layer, None where not needed; ``dx`` is ``[M, K]``.  ``scales`` None: they follow the codes
    in ``q``, which is one buffer then."""
    M, N, K = sizes
    dev = dy.device
    with _lib.on_device(dev):
        if dy.dim() != 2:
            dy = dy.reshape(M, N)
        if N % 8 == 0:
            dy, ld = _operand(dy), N
        else:       # rows of dy must start on 16-byte boundaries; what lies between them is never used
            ld = -(-N // 8) * 8
            padded = dy.new_empty((M, ld))
            padded.narrow(1, 0, N).copy_(dy)
            dy = padded
        make = dy.new_empty if M and N else dy.new_zeros
        dx = make((M, K)) if need_dx else None
        dw = make((N, K)) if need_dw else None
        db = make(N) if need_db else None
        if M and N and (need_dx or need_dw or need_db):
            ws, nbytes = _workspace(M, N, K, need_dx + 2 * need_dw + 4 * need_db, dev)
            w = _operand(weight) if need_dx else None
            adr = _lib.address
            codes = sc = None
            if need_dw:
                q = _operand(q)
                codes = q.data_ptr()
                sc = codes + M * K if scales is None else scales.data_ptr()
            _lib.check(_lib.lib().tcb_linear_backward(dy.data_ptr(), ld, adr(w), codes, sc, adr(zp), adr(dx), adr(dw), adr(db),
                                                      M, N, K, group_size, adr(ws), nbytes, _lib.stream_of(dev)))
    return dx, dw, db


class _CheckpointLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, group_size, grad_mode):
        N, K = weight.shape
        dev = x.device
        x2 = _operand(x if x.dim() == 2 else x.reshape(-1, K))
        M = x2.shape[0]
        y = x2.new_empty((M, N))
        # needs_input_grad tells what requires a gradient even where no graph is recorded, and in here grad mode is always off
        need_dx, need_dw = (grad_mode and need for need in ctx.needs_input_grad[:2])
        # codes [M, K], then scales [M, K / G]: one buffer (M K is a multiple of 16, so the scales are aligned)
        kept = torch.empty(M * K + 2 * (M * K // group_size), dtype=torch.uint8, device=dev) if need_dw else None
        if M and N:
            with _lib.on_device(dev):
                w, b = _operand(weight), None if bias is None else bias.contiguous()
                ws, nbytes = _workspace(M, N, K, 0, dev)
                adr = _lib.address
                q = adr(kept)
                _lib.check(_lib.lib().tcb_linear_forward(x2.data_ptr(), w.data_ptr(), adr(b), y.data_ptr(), q, q + M * K if need_dw else None,
                                                         M, N, K, group_size, adr(ws), nbytes, _lib.stream_of(dev)))
        ctx.save_for_backward(kept, weight if need_dx else None)
        ctx.x_shape, ctx.sizes, ctx.group_size = x.shape, (M, N, K), group_size
        return y if x.dim() == 2 else y.view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        return _checkpoint_backward_once(ctx, dy) if torch.is_grad_enabled() else _checkpoint_backward(ctx, dy)


def _checkpoint_backward(ctx, dy):
    kept, weight = ctx.saved_tensors
    need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
    dx, dw, db = _backward(dy, ctx.sizes, weight, kept, None, None, ctx.group_size, need_dx, need_dw, need_db)
    return dx.view(ctx.x_shape) if need_dx and len(ctx.x_shape) != 2 else dx, dw, db, None, None


# with create_graph the results refuse to be differentiated; the wrapper is left out where nobody could
_checkpoint_backward_once = once_differentiable(_checkpoint_backward)


class _FusedDequantLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, bias, q, scales, zp, group_size):
        N, K = weight.shape
        M = q.shape[0]
        y = torch.empty((M, N), dtype=torch.bfloat16, device=q.device)
        if M and N:
            _launch(weight.contiguous(), q, scales, zp, None if bias is None else bias.contiguous(), y, N, M, K, group_size, False)
        ctx.save_for_backward(q, scales, zp)
        ctx.sizes, ctx.group_size = (M, N, K), group_size
        return y

    @staticmethod
    def backward(ctx, dy):
        return _fused_backward_once(ctx, dy) if torch.is_grad_enabled() else _fused_backward(ctx, dy)


def _fused_backward(ctx, dy):
    q, scales, zp = ctx.saved_tensors
    need_dw, need_db = ctx.needs_input_grad[:2]
    _, dw, db = _backward(dy, ctx.sizes, None, q, scales, zp, ctx.group_size, False, need_dw, need_db)
    return dw, db, None, None, None, None


_fused_backward_once = once_differentiable(_fused_backward)


def int8_checkpoint_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, group_size: int = 32) -> torch.Tensor:
    """``x @ weight.T + bias`` (bf16 ``[..., K]`` -> ``[..., N]``) that keeps ``x`` in 8 bits for the backward pass.

    Without a graph (``torch.no_grad()``, nothing that requires a gradient) no codes are made.
    The forward product and the gradients of ``x`` and ``bias`` use the bf16 values; the gradient of ``weight`` is
    ``dy.T @ dequantize_int8_g32(quantize_int8_g32(x))``.  K is a multiple of ``group_size`` (16, 32, 64 or 128).
    Values of ``x`` that are not finite enter the weight gradient as 0, as the codec stores them; decoded values past the largest bf16
    number stay at it, so that a row of the lowest number adds nothing where its ``dy`` is 0.  CUDA tensors
    only; gradients of gradients are not available.  A training step can be captured in a CUDA graph under torch's own
    condition: no eager graph of the same leaves is alive during the capture (``del`` the outputs of warm-up steps).
    """
    if x.dim() == 0 or weight.dim() != 2:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    K = x.shape[-1]
    if group_size not in SUPPORTED_GROUP_SIZES:
        raise ValueError(f"group_size {group_size} is not supported, choose from {SUPPORTED_GROUP_SIZES}")
    if K <= 0 or K % group_size != 0:
        raise ValueError(f"the inner dimension ({K}) must be a positive multiple of the group size {group_size}")
    _check_dense("x", x, x.device)
    _check_layer(weight, bias, K, x.device)
    if not x.is_cuda:
        raise RuntimeError("int8_checkpoint_linear runs on CUDA tensors only (no CPU fallback)")
    return _CheckpointLinear.apply(x, weight, bias, group_size, torch.is_grad_enabled())


def fused_dequant_linear(q: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         zero_points: Optional[torch.Tensor] = None, group_size: int = 32) -> torch.Tensor:
    """``dequant(q) @ weight.T + bias`` for codes ``[..., K]`` (int8, or uint8 with zero points), differentiable in
    ``weight`` and ``bias``: ``dweight = dy.T @ dequant(q)``, straight from the codes.  ``dequant`` rounds to bf16, as the decoding
    functions do; the values are those of ``FusedDequantLinear``, which has no gradient.  K is a multiple of ``group_size`` (16, 32, 64 or 128).
    ``scales`` that require a gradient are refused."""
    if q.dim() == 0:
        raise ValueError("q must be [..., K]")
    _refuse_gradient("fused_dequant_linear: scales", scales)
    K = q.shape[-1]
    flat = q.dim() == 2      # a view of the result would be one more node of the graph
    q2 = (q if flat else q.reshape(-1, K) if K else q.reshape(0, 0)).contiguous()
    _check_common(q2, scales, zero_points, K, q2.shape[0], group_size)
    _check_layer(weight, bias, K, q.device)
    for name, t in (("scales", scales), ("zero_points", zero_points)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q is on {q.device}")
    y = _FusedDequantLinear.apply(weight, bias, q2, scales.contiguous(), None if zero_points is None else zero_points.contiguous(), group_size)
    return y if flat else y.view(*q.shape[:-1], weight.shape[0])


class Int8CheckpointLinear(nn.Module):
    """``nn.Linear`` in bf16 whose input is kept in 8 bits between the forward and the backward pass."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_size: int = 32):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = group_size
        self.weight = nn.Parameter(torch.empty((out_features, in_features), dtype=torch.bfloat16))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_features, dtype=torch.bfloat16))
        else:
            self.register_parameter("bias", None)
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            nn.init.zeros_(self.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int8_checkpoint_linear(x, self.weight, self.bias, self.group_size)
