"""Plans of attention weights and pools of one shape."""

import random

import pytest
import torch

from async_llm_amd import native
from async_llm_amd.shared_cache import CacheEviction
from tests.eviction_util import fill, make_op
from tests.test_gpu_weigh import decode_step, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, codes", [(torch.bfloat16, None), (torch.float32, None), (torch.bfloat16, torch.int8)])
def test_a_plan_serves_pools_of_its_size_only(dtype, codes):
    """Pools of other layers share a step's plan; one with fewer or more pages has other slots."""
    dev, r, gen = torch.device("cuda:0"), random.Random(1), torch.Generator().manual_seed(1)
    op, alike, small, large = (make_op(dev, 8, 2, 64, 16, dtype, pages, codes) for pages in (100, 100, 60, 101))
    fill(op, gen)
    fill(alike, torch.Generator().manual_seed(1))
    meta = decode_step(op, r, 3, [40, 17], shared=90)
    q, lse = inputs(op, meta, gen)
    e = CacheEviction(op)
    plan = e.plan(meta)
    want = e.accumulate(q, lse, 0, plan, e.new_weights())
    other = CacheEviction(alike)
    assert torch.equal(other.accumulate(q, lse, 0, plan, other.new_weights()), want) and bool((want > 0).any())
    for wrong in (small, large):
        f = CacheEviction(wrong)
        weights, out = f.new_weights(), f.new_weights()
        with pytest.raises(native.ViewAttnError, match="another shape or pool"):
            f.accumulate(q, lse, 0, plan, weights)
        with pytest.raises(native.ViewAttnError, match="another shape or pool"):
            f.accumulate(q, lse, 0, plan, weights, out=out)
        assert not bool(weights.any()) and not bool(out.any())
