"""Chunks that are read back over the smallest scales: powers of two that undo a scale are no smaller than 32 bits hold."""

import pytest
import torch

from tests import quant_util as Q
from tests.test_gpu_quant_attend import check
from tests.test_gpu_quant_range import BF16, DEV, E4M3, INT8, chunk_step


def fill(op, step, which, codes, size, g):
    for segments in step.segments:
        for slots, _, _ in segments:
            x = torch.randn(len(slots), op.num_kv_heads, op.head_dim, generator=g) * size
            Q.write(op.kv_cache, which, 0, slots, *Q.quantised32(x, codes))


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("size", [2.0**-113, 2.0**-116, 2.0**-118])
def test_the_smallest_values_come_back(codes, size):
    op, pool, g, step, contexts = chunk_step(codes)
    fill(op, step, 1, codes, size, g)
    q = torch.randn(53, 512, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    assert step.meta.launch.readback.scratch[:4].view(torch.int32).item() == 0
    # results are a few 2^-120, far over bf16's smallest normal number: within an eighth of the largest value they are not zero
    check(op, step, q, [0, 33], [33, 20], out, lse)
    assert (out.abs().float().amax(-1) > size / 64).all()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_the_smallest_keys_under_large_queries(codes):
    op, pool, g, step, contexts = chunk_step(codes)
    fill(op, step, 0, codes, 2.0**-121.5, g)
    q = (torch.randn(53, 512, generator=g) * 2.0**121.5).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    assert step.meta.launch.readback.scratch[:4].view(torch.int32).item() == 0
    check(op, step, q, [0, 33], [33, 20], out, lse)
