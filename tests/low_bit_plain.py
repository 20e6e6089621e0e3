"""Plain 64-bit restatements of the low-bit operators, for the tests."""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e for whole numbers, exactly (from the bits of a double; a power function may be an ulp off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def mx_encode(x: torch.Tensor):
    """[r, k] -> (code 0..15 as int64 [r, k], scale byte int64 [r, k / 32]); nearest neighbour on the grid, ties to even codes."""
    v = x.double().view(x.shape[0], -1, 32)
    v = torch.where(v.isfinite(), v, torch.zeros_like(v))
    grid = GRID.to(x.device)
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))          # max = m 2^e, m in [0.5, 1)
    byte = torch.where(v.abs().amax(-1, keepdim=True) > 0, (e - 1 - 2 + 127).clamp(min=0), torch.zeros_like(e)).long()
    a = v.abs() * pow2(127 - byte)
    d = (a.unsqueeze(-1) - grid).abs()                           # [..., 8]
    best = d.amin(-1, keepdim=True)
    hit = d == best
    even = torch.arange(8, device=x.device) % 2 == 0
    prefer = torch.where((hit & even).any(-1, keepdim=True), hit & even, hit)
    code = prefer.double().argmax(-1) + 8 * torch.signbit(v).long()
    return code.view(x.shape), byte.squeeze(-1)


def mx_values(code: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """codes [r, k] and scale bytes [r, k / 32] -> fp64 values (255: NaN)."""
    m = GRID.to(code.device)[code % 8] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.where(byte == 255, torch.full_like(byte, float("nan"), dtype=torch.float64), pow2(byte - 127))
    return (m.view(code.shape[0], -1, 32) * s.unsqueeze(-1)).view(code.shape)


def mx_pack(code: torch.Tensor) -> torch.Tensor:
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)


def mx_scale_offset(r: int, b: int, cols: int) -> int:
    """Byte of block b of row r in the tile order."""
    return (r // 128 * -(-cols // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def int8_encode(x: torch.Tensor, group: int):
    """[r, k] -> (codes fp64 [r, k], bf16 scales [r, k / group]); the scale is the bf16 rounding of the fp32 quotient."""
    v = x.double().view(x.shape[0], -1, group)
    v = torch.where(v.isfinite(), v, torch.zeros_like(v))
    floor = float(torch.tensor(1e-8, dtype=torch.float32))
    scale = (v.abs().amax(-1, keepdim=True).clamp(min=floor) / 127).float().to(torch.bfloat16)
    q = torch.round((v / scale.double()).float().double()).clamp(-128, 127)
    return q.view(x.shape), scale.squeeze(-1)


def int8_values(q, scales, group, zp=None) -> torch.Tensor:
    v = q.double().view(q.shape[0], -1, group)
    if zp is not None:
        v = v - zp.double().view(q.shape[0], -1, 1)
    return (v * scales.double().view(q.shape[0], -1, 1)).view(q.shape)
