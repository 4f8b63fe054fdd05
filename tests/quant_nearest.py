"""Whether codes are the nearest ones, element by element."""

from __future__ import annotations

import torch

from tests import quant_util as Q


def spacing(y: torch.Tensor, code_dtype) -> torch.Tensor:
    """Between neighbouring codes at ``y``."""
    if code_dtype == torch.int8:
        return torch.ones_like(y)
    return torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)


def assert_nearest(codes: torch.Tensor, scales: torch.Tensor, x64: torch.Tensor, off: torch.Tensor, code_dtype) -> None:
    """``quant_util.assert_quantises`` with every element held to half the spacing of codes beside ``off``: that of the binade
    that its 32-bit value, up to ``off`` larger, may lie in."""
    Q_ASSERT(codes, scales, x64, off, code_dtype)
    step = torch.pow(2.0, scales.view(torch.uint8).double() - 127)[..., None]
    y, room = x64.clamp(-Q.LIMIT[code_dtype], Q.LIMIT[code_dtype]) / step, off / step
    err = (codes.float().double() - y).abs()
    worst = (err - (spacing(y.abs() + room, code_dtype) / 2 + room) * (1 + 1e-9)).max().item() if err.numel() else 0.0
    assert worst <= 0, f"a code is {worst:.3e} further from its element than the nearest one may be"


Q_ASSERT = Q.assert_quantises  # (tests put the stricter one in its place)
