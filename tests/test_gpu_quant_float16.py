"""Chunks of float16 activations are as exact as their steps of single tokens: operands hold more bits than the result."""

import pytest
import torch

from tests import quant_util as Q


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 4, 256), (32, 8, 64)])
def test_large_chunks_round_once(heads, codes):
    """Work for which bf16 activations are read back: the error against 64 bits is that of rounding the result.

    Beside that rounding (r of the norm of the result, measured on the 64-bit one) the operands' are 2^-17 of a query's and a weight's
    elements, 2^-6 of a float16 rounding's: even where they add up over cancelling values they stay below r / 2, and independent
    errors add in squares."""
    dev = torch.device("cuda")
    new, context = 300, 3700
    op, pool, g = Q.make(dev, heads, 16, 280, torch.float16, codes)
    pages = Q.Pages(280, 16)
    step = Q.prefill_step(op, [([pages.block(dev, context)], pages.block(dev, 0, room=new), new)])
    q = torch.randn(new, heads[0] * heads[2], generator=g).half().to(dev)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    expected = Q.attention64(op, q.cpu().view(new, heads[0], heads[2]), step.segments[0])
    Q.assert_attends(out, lse, expected, torch.float16, context + new)
    want = expected[0]
    rounding = (want.half().double() - want).norm()
    assert (out.cpu().double() - want).norm() <= (1 + 0.5**2) ** 0.5 * rounding
