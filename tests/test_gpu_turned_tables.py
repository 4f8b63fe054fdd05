"""Blocks of keys turned by a stretched rotation: merged over its unit table, refused over its table with the attention factor."""

from types import SimpleNamespace

import pytest
import torch

from async_llm_amd.kvcache import MHAKVCache, PageAllocator
from async_llm_amd.rotary import RotaryEmbedding
from async_llm_amd.shared_cache import BlockKVOps, SharedCacheAttention, WorkerGroup
from async_llm_amd.shared_cache.block_ops import token_slots
from tests.eviction_util import fill, make_op

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
    before, free = pool.k_cache(0).view(torch.int32).clone(), allocator.num_free_pages  # (bits: nobody has written the other slots)
    for call in (refused.merge_blocks, refused.append_block):
        with pytest.raises(ValueError, match="unit"):
            call(left, right)
    assert allocator.num_free_pages == free and torch.equal(pool.k_cache(0).view(torch.int32), before) and left.num_tokens == 61
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


def test_attention_over_a_unit_table_is_that_of_the_factor():
    """With the first rotary_dim elements of every query head multiplied by the factor's square, those that pass through as they
    are, a view over the unit table gives what q and k at their absolute positions, both times the factor, give."""
    dev, gen = torch.device("cuda:0"), torch.Generator().manual_seed(13)
    hq, hkv, D, rotary, P, n = 4, 2, 64, 32, 8, 50
    r = RotaryEmbedding(D, rotary, 1e5, scaling=YARN, device=dev)
    assert r.attention_factor > 1.1
    pool = MHAKVCache(hkv, 1, D, 40, P, torch.float32, dev)
    op = SharedCacheAttention(pool, r.cos_sin_cache(500, unit=True), hq, hkv, D, P, torch.float32, dev, rotary_dim=rotary)
    allocator = PageAllocator(40, P, dev)
    ops = BlockKVOps(pool, op, allocator)
    block, own = ops.create_block(), ops.create_block()
    block.grow_pages(allocator.alloc_pages(block.pages_needed(n)), n)
    block.mrope_span_override = 300
    k, v = torch.randn(2, n + 1, hkv, D, generator=gen)
    q = torch.randn(1, hq, D, generator=gen)
    old = SimpleNamespace(positions=torch.arange(n, device=dev), mrope_positions=None, out_loc=torch.from_numpy(token_slots(block)).to(dev))
    op.store_new_kv(k[:n].view(n, -1).to(dev), v[:n].view(n, -1).to(dev), 0, old)
    page = int(allocator.alloc_pages(1))
    slot = torch.tensor([page], dtype=torch.int32, device=dev)
    meta = op.prepare(WorkerGroup(cache_structure=[[block, own]], write_to=[own]), {id(own): page}, slot)
    batch = SimpleNamespace(attn_metadata=meta, positions=torch.zeros(1, dtype=torch.int64, device=dev), mrope_positions=None, out_loc=slot)
    mine = q.clone()
    mine[..., :rotary] *= r.attention_factor ** 2
    got, lse = op.forward_with_lse(mine.view(1, -1).to(dev), k[n:].view(1, -1).to(dev), v[n:].view(1, -1).to(dev), 0, batch)

    def turned(x, at):
        x, h = x.double(), rotary // 2
        unit = torch.polar(torch.full((len(at), h), r.attention_factor, dtype=torch.float64), at.double()[:, None] * r.inv_freq.cpu())[:, None]
        z = torch.complex(x[..., :h].contiguous(), x[..., h: 2 * h].contiguous()) * unit
        return torch.cat([z.real, z.imag, x[..., 2 * h:]], dim=-1)

    at = torch.cat([torch.arange(n), torch.tensor([300])])
    x, y = turned(q, at[n:]).view(hkv, hq // hkv, D), turned(k, at)
    score = torch.einsum("hgd,nhd->hgn", x, y) / D**0.5
    weight = torch.softmax(score, -1)
    want = torch.einsum("hgn,nhd->hgd", weight, v.double())
    # a score: both turns mix two elements and lose eight units each, the query's scaling one, a sum of D products D; a result:
    # twice the worst score's error (numerator and denominator), and a sum of n weights and n products
    mixed = torch.cat([torch.cat([q[..., :16].abs() + q[..., 16:32].abs()] * 2, -1) * r.attention_factor**2, q[..., 32:].abs()], -1).double()
    keys = torch.cat([torch.cat([k[..., :16].abs() + k[..., 16:32].abs()] * 2, -1), k[..., 32:].abs()], -1).double()
    off = (D + 20) * 2.0**-24 * torch.einsum("hgd,nhd->hgn", mixed.view(hkv, -1, D), keys).amax(-1, keepdim=True) / D**0.5
    off = off + 2.0**-24 * score.abs().amax(-1, keepdim=True)
    room = (2 * off + 2 * (n + 1) * 2.0**-24) * torch.einsum("hgn,nhd->hgd", weight, v.double().abs())
    assert bool(((got.cpu().double().view(hkv, -1, D) - want).abs() <= room).all())
    total = torch.logsumexp(score, -1)
    assert bool(((lse.cpu().double().view(hkv, -1) - total).abs() <= off[..., 0] + (n + 1) * 2.0**-24 + 2.0**-23 * total.abs()).all())
    # (what the bound is there to tell apart: the factor on all of a query)
    whole = torch.softmax(torch.einsum("hgd,nhd->hgn", torch.cat([x[..., :32], x[..., 32:] * r.attention_factor**2], -1), y) / D**0.5, -1)
    assert bool(((torch.einsum("hgn,nhd->hgd", whole, v.double()) - want).abs().amax(-1) > 4 * room.amax(-1)).all())


def test_ops_and_turns_while_a_graph_is_recorded():
    """A turn may be recorded first of all; an op that is made while recording looks at its table later."""
    dev, gen = torch.device("cuda:0"), torch.Generator().manual_seed(14)
    r = RotaryEmbedding(64, scaling=YARN, device=dev)
    unit, scaled = r.cos_sin_cache(100, unit=True), r.cos_sin_cache(100)
    op = make_op(dev, 4, 2, 64, 16, torch.bfloat16, 10, torch.int8)
    fill(op, gen)
    source, target = torch.arange(20, 50, device=dev), torch.arange(100, 130, device=dev)
    graph, made, x = torch.cuda.CUDAGraph(), [], torch.zeros(4, device=dev)
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph):
        x += 1
        op.copy_shifted(source, target, 7)
        for table in (unit, scaled):
            made.append(SharedCacheAttention(MHAKVCache(2, 1, 64, 4, 16, torch.bfloat16, dev), table, 4, 2, 64, 16, torch.bfloat16, dev))
    made[0]._check_turns()
    with pytest.raises(ValueError, match="unit"):
        made[1]._check_turns()
    codes = op.kv_cache.k_codes(0).view(torch.uint8)
    for _ in range(3):
        codes[6:].zero_()
        graph.replay()
        torch.cuda.synchronize(dev)
        got = codes.clone()
        codes[6:].zero_()
        op.copy_shifted(source, target, 7)
        assert torch.equal(got, codes) and bool(codes[7].any())
    assert float(x[0]) == 3.0
