"""Evictions that fail half-way hand their pages back."""

from types import SimpleNamespace

import pytest
import torch

from async_llm_amd.kvcache import PageAllocator
from async_llm_amd.shared_cache import BlockKVOps, CacheEviction
from tests.eviction_util import fill, make_op

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["clear", "select", "move"])
def test_pages_go_back(where, monkeypatch):
    dev = torch.device("cuda:0")
    op = make_op(dev, 4, 2, 64, 16, torch.bfloat16, 40)
    fill(op, torch.Generator().manual_seed(1))
    allocator = PageAllocator(40, 16, dev)
    ops = BlockKVOps(op.kv_cache, op, allocator)
    weights = CacheEviction(op).new_weights()
    block = ops.create_block()
    block.grow_pages(allocator.alloc_pages(3), 45)
    block.token_ids = list(range(45))
    before, free = op.kv_cache.k_cache(0).clone(), sorted(allocator.free_page_starts.tolist())

    def full(*args, **more):
        raise torch.cuda.OutOfMemoryError("no room")

    with monkeypatch.context() as patch:
        patch.setattr(CacheEviction, where, full)
        with pytest.raises(torch.cuda.OutOfMemoryError, match="no room"):
            ops.evict_tokens(block, weights, 20)
        assert sorted(allocator.free_page_starts.tolist()) == free
        # an allocator that takes nothing back
        ops.page_allocator = SimpleNamespace(alloc_pages=allocator.alloc_pages)
        with pytest.raises(torch.cuda.OutOfMemoryError, match="no room"):
            ops.evict_tokens(block, weights, 20)
        assert allocator.num_free_pages == len(free) - 2
    assert torch.equal(op.kv_cache.k_cache(0), before)
    assert (block.num_tokens, block.num_pages, block.token_ids) == (45, 3, list(range(45)))
    assert ops.evict_tokens(block, weights, 20).num_tokens == 20
