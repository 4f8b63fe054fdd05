"""Blocks of keys turned by a stretched rotation: merged over its unit table, refused over its table with the attention factor."""

import pytest
import torch

from async_llm_amd.kvcache import MHAKVCache, PageAllocator
from async_llm_amd.rotary import RotaryEmbedding
from async_llm_amd.shared_cache import BlockKVOps, SharedCacheAttention
from async_llm_amd.shared_cache.block_ops import token_slots

pytestmark = pytest.mark.gpu
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("append", [False, True])
def test_merged_keys_are_those_of_their_new_positions(append):
    dev, gen = torch.device("cuda:0"), torch.Generator().manual_seed(12)
    r = RotaryEmbedding(64, 32, 1e5, scaling=YARN, device=dev)
    plain = RotaryEmbedding(64, 32, 1e5, scaling=dict(YARN, attention_factor=1.0), device=dev)
    pool = MHAKVCache(2, 2, 64, 40, 8, torch.float32, dev)
    op, scaled = (SharedCacheAttention(pool, r.cos_sin_cache(3000, unit=unit), 4, 2, 64, 8, torch.float32, dev, rotary_dim=32)
                  for unit in (True, False))
    allocator = PageAllocator(40, 8, dev)
    ops, refused = BlockKVOps(pool, op, allocator), BlockKVOps(pool, scaled, allocator)
    left, right = ops.create_block(), ops.create_block()
    for b, n in ((left, 61), (right, 50)):
        b.grow_pages(allocator.alloc_pages(b.pages_needed(n)), n)
    left.mrope_span_override = 2000  # (far enough for every pair to turn)
    k = torch.randn(2, 50, 2, 64, generator=gen)
    at, slots = torch.arange(50, device=dev), torch.from_numpy(token_slots(right)).to(dev)
    for layer in range(2):
        pool.k_cache(layer).view(-1, 2, 64)[slots] = plain(at, k[layer].to(dev))[0]
    before, free = pool.k_cache(0).clone(), allocator.num_free_pages
    for call in (refused.merge_blocks, refused.append_block):
        with pytest.raises(ValueError, match="unit"):
            call(left, right)
    assert allocator.num_free_pages == free and torch.equal(pool.k_cache(0), before) and left.num_tokens == 61
    result = (ops.append_block if append else ops.merge_blocks)(left, right)
    slots = torch.from_numpy(token_slots(result))[61:]
    angle = (2000 + torch.arange(50)).double()[:, None] * r.inv_freq.cpu()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    for layer in range(2):
        x = k[layer].double()
        a, b = x[..., :16], x[..., 16:32]
        want = torch.cat([a * c - b * s, b * c + a * s, x[..., 32:]], dim=-1)
        # a rotation is off by its cosine (four units), two products and a sum, of both elements of a pair; twice
        size = torch.cat([a.abs() + b.abs()] * 2 + [torch.zeros(50, 2, 32)], dim=-1)
        got = pool.k_cache(layer).view(-1, 2, 64).cpu()[slots].double()
        assert bool(((got - want).abs() <= 2 * 7 * 2.0**-24 * size).all())
