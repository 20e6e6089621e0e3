"""``DeviceFeatureCache``: feature rows kept in GPU memory as symmetric int8 codes.

The device-resident counterpart of ``FeatureCacheWriter`` / ``FeatureCacheDataset``: rows are quantised as
they are written and decoded as they are read, at any row index, with the codec of ``quantize_int8_g32``
(codes, bf16 scales and decoded values have its bits).  A row takes ``1 + 2 / group_size`` bytes a value, so a
180 GB GPU holds about twice the rows that bf16 would.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .codec import _DTYPES, _check_group_size
from .fused_linear import _operand_on

Indices = Union[torch.Tensor, Sequence[int]]


class DeviceFeatureCache:
    """``num_rows`` rows of ``row_shape`` values (an int, or a tuple such as ``(seq_len, dim)``) on one GPU.

    ``codes`` (int8 ``[num_rows, width]``) and ``scales`` (bf16 ``[num_rows, width / group_size]``) are plain
    tensors that start as zeros; rows that were never written read as zeros.  The number of values of a row must be
    a multiple of ``group_size``.

    To autograd a ``write`` is an in-place change of both tensors: a graph that keeps one of them (``fused_dequant_linear`` on the cache's own
    codes) and is differentiated after the next write raises torch's error.

    Calls only enqueue work on the current stream of the cache's device (index tensors on the GPU are not looked
    at by the host), so they can be captured in a CUDA graph.  As with any tensor, calls on different streams need
    an order from the caller.
    """

    def __init__(self, num_rows: int, row_shape: Union[int, Tuple[int, ...]], group_size: int = 32,
                 device: Optional[Union[str, torch.device]] = None):
        _check_group_size(group_size)
        self.row_shape = (int(row_shape),) if isinstance(row_shape, int) else tuple(int(v) for v in row_shape)
        if num_rows < 0 or any(v < 0 for v in self.row_shape):
            raise ValueError(f"negative size: {num_rows} rows of {self.row_shape}")
        self.num_rows, self.group_size = int(num_rows), group_size
        self.width = math.prod(self.row_shape)
        if self.width % group_size != 0:
            raise ValueError(f"{self.width} values a row is not a multiple of the group size {group_size}")
        if not torch.cuda.is_available():
            raise RuntimeError("DeviceFeatureCache keeps its rows on a CUDA device (no CPU fallback) and none is available")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"DeviceFeatureCache keeps its rows on a CUDA device, got {dev}")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self.codes = torch.zeros((self.num_rows, self.width), dtype=torch.int8, device=self.device)
        self.scales = torch.zeros((self.num_rows, self.width // group_size), dtype=torch.bfloat16, device=self.device)
        # per row: which call wrote it last and from where in the call's list (settles an index that occurs twice);
        # the last word counts calls
        self._claims = torch.zeros(self.num_rows + 1, dtype=torch.int64, device=self.device)

    def __len__(self) -> int:
        return self.num_rows

    def __repr__(self):
        return f"DeviceFeatureCache({self.num_rows} x {self.row_shape}, G={self.group_size}, {self.device})"

    def _indices(self, indices: Indices) -> torch.Tensor:
        idx = indices if isinstance(indices, torch.Tensor) else torch.as_tensor(indices)
        if idx.dtype != torch.int64 or idx.dim() != 1:
            if idx.dim() != 1 or idx.dtype != torch.int32 and idx.numel():
                raise ValueError(f"indices must be one-dimensional int64 or int32, got {tuple(idx.shape)} of {idx.dtype}")
            idx = idx.long()
        if not idx.is_cuda:
            if idx.numel() and int(idx.max()) >= self.num_rows:
                raise IndexError(f"row {int(idx.max())} in a cache of {self.num_rows} rows")
        elif idx.device != self.device:
            raise ValueError(f"indices are on {idx.device}, the cache is on {self.device}")
        return _operand_on(idx, self.device, 8)

    def write(self, indices: Indices, x: torch.Tensor) -> None:
        """Quantises row ``t`` of ``x`` (``[n, *row_shape]`` or ``[n, width]``) into row ``indices[t]``.

        A negative index leaves its row out (padding); so does, in an index tensor on the GPU, one past the end --
        given on the host that raises ``IndexError``.  Of an index that occurs more than once the last occurrence stays.  Values that are
        not finite are stored as 0.  bf16, fp16 and fp32 are read as they are, other types are converted to fp32.
        """
        with _lib.on_device(self.device):
            idx = self._indices(indices)
            n = idx.numel()
            if x.shape != (n, self.width) and x.shape != (n, *self.row_shape):
                raise ValueError(f"expected {n} rows of {self.row_shape}, got {tuple(x.shape)}")
            if x.is_cuda and x.device != self.device:
                raise ValueError(f"x is on {x.device}, the cache is on {self.device}")
            if x.dtype not in _DTYPES:
                x = x.float()
            xd = _operand_on(x, self.device, 32)
            _lib.check(_lib.lib().tcb_cache_write(xd.data_ptr(), _DTYPES[xd.dtype], idx.data_ptr(), n, self.codes.data_ptr(),
                                                  self.scales.data_ptr(), self.num_rows, self.width, self.group_size,
                                                  self._claims.data_ptr(), _lib.stream_of(self.device)))
            increment_version((self.codes, self.scales))

    def read(self, indices: Indices, out_buffer: Optional[torch.Tensor] = None) -> torch.Tensor:
        """bf16 ``[n, *row_shape]``: row ``indices[t]`` decoded; a row that ``write`` would leave out is zeros.
        If ``out_buffer`` is given it is written in place and returned."""
        with _lib.on_device(self.device):
            idx = self._indices(indices)
            n = idx.numel()
            if out_buffer is None:
                out_buffer = self.scales.new_empty((n, *self.row_shape))
            elif out_buffer.numel() != n * self.width or out_buffer.dtype != torch.bfloat16:
                raise ValueError(f"out_buffer must be a bf16 tensor of {n} rows of {self.width} values")
            else:
                increment_version(out_buffer)   # the kernel writes through its address
            if n == 0 or self.width == 0:
                return out_buffer
            direct = out_buffer.device == self.device and out_buffer.is_contiguous() and out_buffer.data_ptr() % 32 == 0
            od = out_buffer if direct else self.scales.new_empty(n * self.width)
            _lib.check(_lib.lib().tcb_cache_read(self.codes.data_ptr(), self.scales.data_ptr(), self.num_rows, self.width, self.group_size,
                                                 idx.data_ptr(), n, od.data_ptr(), _lib.stream_of(self.device)))
            if not direct:
                out_buffer.copy_(od.view(out_buffer.shape))
        return out_buffer
