"""Attention over codes where its kernels' tiles are unusual: scattered pages at every head dim, and scores that rise by less
in a tile than sums are rescaled for."""

import pytest
import torch

from tests import quant_util as Q
from tests.test_gpu_quant_attend import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("page", [1, 2, 8, 24, 48])
@pytest.mark.parametrize("heads", [(16, 4, 256), (8, 8, 256), (32, 2, 128), (8, 4, 64)])
@pytest.mark.parametrize("dtype,codes", [(BF16, E4M3), (F16, INT8)])
def test_scattered_pages(page, heads, dtype, codes):
    """Decodes and a chunk: pages of fewer than sixteen tokens, and of numbers that no power of two is."""
    num_pages = 1600 // page + 40
    op, pool, g = Q.make(DEV, heads, page, num_pages, dtype, codes)
    op._reads_back = lambda pairs, pages: False
    pages = Q.Pages(num_pages, page)
    common = pages.block(DEV, 333)
    views = [[common, pages.block(DEV, n, room=1)] for n in (200, 31, 64, 1)] + [[pages.block(DEV, 130, room=1)]]
    step = Q.decode_step(op, pages, views, [v[-1] for v in views], g)
    q = torch.randn(5, heads[0] * heads[2], generator=g).to(dtype).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check(op, step, q, range(5), [1] * 5, out, lse)
    step = Q.prefill_step(op, [([common], pages.block(DEV, 9, room=41), 41), ([], pages.block(DEV, 0, room=19), 19)])
    q = torch.randn(60, heads[0] * heads[2], generator=g).to(dtype).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check(op, step, q, [0, 41], [41, 19], out, lse)


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("heads,codes", [((4, 1, 64), E4M3), ((4, 1, 128), INT8), ((4, 1, 256), E4M3)])
@pytest.mark.parametrize("rise", ["slow", "fast", "falling", "waves"])
def test_scores_that_rise_slowly(page, heads, codes, rise):
    """A wave's next tile is 128 tokens further: scores rise by 1.4 powers of two in it (slow) or by 11 (fast), fall, or do both."""
    op, pool, g = Q.make(DEV, heads, page, 4200 // page, BF16, codes, rotary=0)
    pages = Q.Pages(4200 // page, page)
    block, own = pages.block(DEV, 4000), pages.block(DEV, 3, room=1)
    t = torch.arange(4000, dtype=torch.float32) / 128
    height = {"slow": t, "fast": 8 * t, "falling": 31 - t, "waves": 6 * torch.sin(t / 2) + t / 2}[rise]
    D = heads[2]
    k = torch.randn(4000, 1, D, generator=g) * 0.25 + (height * D**-0.5)[:, None, None]  # under queries of ones: the height, and noise
    Q.write(pool, 0, 0, Q.slots_of(block), *Q.quantised32(k, codes))
    step = Q.decode_step(op, pages, [[block, own]] * 1, [own], g)
    q = torch.ones(1, 4, D)
    q[0, 1], q[0, 2], q[0, 3] = -1, 0.5, torch.randn(D, generator=g)
    q = q.view(1, 4 * D).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check(op, step, q, [0], [1], out, lse)
