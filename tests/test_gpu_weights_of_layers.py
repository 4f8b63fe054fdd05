"""Weights of several layers over one pool: all of them follow their tokens."""

import random

import pytest
import torch

from async_llm_amd.kvcache import PageAllocator
from async_llm_amd.shared_cache import BlockKVOps, CacheEviction
from async_llm_amd.shared_cache.block_ops import token_slots
from tests.eviction_util import fill, make_op
from tests.test_gpu_eviction import chosen

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("codes", [None, E4M3])
@pytest.mark.parametrize("n", [1, 40, 700])
@pytest.mark.parametrize("several", [0, 1, 2, 5])
def test_moves(dev, codes, n, several):
    gen = torch.Generator().manual_seed(n + several)
    op = make_op(dev, 12, 3, 64, 16, BF16, 100, codes, layers=2)
    e = CacheEviction(op)
    order = torch.randperm(e.num_slots, generator=gen)
    source, target = order[:n].clone(), order[n: 2 * n].clone()
    if n > 10:  # slots outside the pool: such tokens are skipped
        source[3], target[5], source[7] = -1, e.num_slots, 1 << 40
    ok = (source >= 0) & (source < e.num_slots) & (target < e.num_slots)
    weights = [torch.rand(3, e.num_slots, generator=gen).to(dev) for _ in range(several)]
    want = [w.cpu() for w in weights]
    for w in want:
        w[:, target[ok]] = w[:, source[ok]]
    e.move(source.to(dev), target.to(dev), weights=weights)
    for w, x in zip(weights, want):
        assert torch.equal(w.cpu(), x)


def test_weights_follow_where_no_layer_does(dev):
    """The entry with no layers, of either kind of pool, moves weights alone."""
    from async_llm_amd import native

    gen = torch.Generator().manual_seed(5)
    for codes in (None, E4M3):
        op = make_op(dev, 4, 2, 64, 16, BF16, 10, codes)
        weights = torch.rand(2, 160, generator=gen).to(dev)
        want = weights.clone()
        source, target = torch.arange(20, 50, device=dev), torch.arange(100, 130, device=dev)
        want[:, target] = want[:, source]
        rest = (source.data_ptr(), target.data_ptr(), None, 30, weights.data_ptr(), op._shape, None, native.current_stream_ptr(dev))
        if codes is None:
            native.call_on(dev, native.lib.va_move_kv, None, None, 0, 0, 0, 160, *rest)
        else:
            native.call_on(dev, native.lib.va_move_kv_q8, op.kv_cache.layer(0), 0, 0, 0, *rest)
        assert torch.equal(weights, want)


@pytest.mark.parametrize("codes", [None, E4M3])
def test_evictions(dev, codes):
    r, gen = random.Random(2), torch.Generator().manual_seed(2)
    op = make_op(dev, 8, 2, 64, 16, BF16, 60, codes, layers=3)
    fill(op, gen)
    allocator = PageAllocator(60, 16, dev)
    ops, e = BlockKVOps(op.kv_cache, op, allocator), CacheEviction(op)
    block = ops.create_block()
    block.grow_pages(allocator.alloc_pages(block.pages_needed(301)), 301)
    block.token_ids = [r.randrange(100) for _ in range(301)]
    layers = [torch.rand(2, e.num_slots, generator=gen).to(dev) for _ in range(3)]  # (new pages were someone else's)
    total = layers[0] + layers[1] + layers[2]
    old = [w.cpu() for w in (total, *layers)]
    slots = torch.from_numpy(token_slots(block))
    want = chosen(old[0], slots, 90, 2, 8)
    small = ops.evict_tokens(block, total, 90, first=2, last=8, close_gaps=True, others=layers)
    assert small.token_ids == [block.token_ids[i] for i in want.tolist()]
    new = torch.from_numpy(token_slots(small))
    tail = torch.arange(small.page_starts[-1] + 90 % 16, small.page_starts[-1] + 16)
    rest = torch.ones(e.num_slots, dtype=torch.bool)
    rest[new] = rest[tail] = False
    for w, x in zip((total, *layers), old):
        assert torch.equal(w.cpu()[:, new], x[:, slots[want]])
        assert bool((w.cpu()[:, tail] == 0).all())
        assert torch.equal(w.cpu()[:, rest], x[:, rest])
    free = allocator.num_free_pages
    for bad in ([layers[0], layers[1][:, :-1]], [layers[0].double()], layers[0]):
        with pytest.raises(ValueError, match="weights"):
            ops.evict_tokens(block, total, 90, others=bad)
        with pytest.raises(ValueError, match="weights"):
            e.move(new.to(dev), slots[:90].to(dev), weights=list(bad))
    assert allocator.num_free_pages == free
