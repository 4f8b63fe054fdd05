"""Choosing and moving tokens, and a block that is evicted from and read again."""

import random

import pytest
import torch

from async_llm_amd import native
from async_llm_amd.kvcache import MHAKVCache, PageAllocator
from async_llm_amd.rotary import RotaryEmbedding
from async_llm_amd.shared_cache import BlockKVOps, CacheEviction, SharedCacheAttention, WorkerGroup
from async_llm_amd.shared_cache.block_ops import token_slots
from tests.eviction_util import blocks_of, fill, keys64, make_op, turned64, turned64_abs, weights64
from tests.quant_util import quantised32, rows64, scales_of

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
HALF = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


# ---------------------------------------------------------------------------
# choosing
# ---------------------------------------------------------------------------
def chosen(weights, slots, keep, first, last):
    """Positions that stay of one block, by sorting."""
    n = len(slots)
    inside = (slots >= 0) & (slots < weights.shape[1])
    score = torch.where(inside, weights.double()[:, slots.clamp(0, weights.shape[1] - 1)].sum(0), 0.0).float()
    t = torch.arange(n)
    rank = torch.where(torch.isnan(score), 2, 1)
    rank = torch.where((t < first) | (t >= n - last), 3, rank).tolist()
    score = torch.where(torch.isnan(score), 0.0, score).tolist()
    order = sorted(range(n), key=lambda i: (-rank[i], 0.0 if rank[i] == 3 else -score[i], i))
    return torch.tensor(sorted(order[: min(keep, n)]), dtype=torch.int64)


def check_select(dev, weights, blocks, keep, first, last):
    slots = torch.cat([b for b in blocks]) if blocks else torch.zeros(0, dtype=torch.int64)
    kept = CacheEviction.select(weights.to(dev), slots.to(dev), [len(b) for b in blocks], keep, first, last)
    want = [chosen(weights, b, k, first, last) for b, k in zip(blocks, keep)]
    assert kept.counts == [len(w) for w in want]
    at = 0
    for b, w in zip(blocks, want):
        part = slice(at, at + len(w))
        assert torch.equal(kept.positions[part].cpu(), w)
        assert torch.equal(kept.slots[part].cpu(), b[w])
        assert torch.equal(kept.shifts[part].cpu(), torch.arange(len(w)) - w)
        at += len(w)
    assert kept.positions.numel() == at


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 1000, 1024, 1500, 10239, 10240, 10241, 16384, 20481, 70001, 300001, 600001])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_one_block(dev, count, heads):
    gen = torch.Generator().manual_seed(count + heads)
    slots = torch.randperm(count + 100, generator=gen)[:count]
    w = torch.exp(3 * torch.randn(heads, count + 100, generator=gen)) * (torch.rand(count + 100, generator=gen) > 0.4)
    for keep in {1, count // 3, count // 2, count - 1, count, count + 5}:
        check_select(dev, w, [slots], [max(keep, 0)], 2, count // 20)


@pytest.mark.parametrize("count", [777, 30000])
def test_ties_and_strange_weights(dev, count):
    gen = torch.Generator().manual_seed(2)
    slots = torch.arange(count).flip(0)
    for w in (torch.zeros(2, count), torch.full((2, count), 0.25), torch.randint(0, 3, (2, count), generator=gen).float(),
              torch.randint(-2, 2, (1, count), generator=gen).float() * 0.0, torch.randn(2, count, generator=gen),
              torch.tensor([1.0, float("inf"), float("nan"), -float("nan"), -float("inf"), 0.0, -0.0])[torch.randint(0, 7, (1, count), generator=gen)]):
        check_select(dev, w, [slots], [count // 2], 0, 0)
        check_select(dev, w, [slots], [count // 3], 3, 5)


def test_many_blocks_long_and_short(dev):
    r, gen = random.Random(3), torch.Generator().manual_seed(3)
    counts = [r.choice([0, 1, 5, 100, 3000]) for _ in range(150)] + [17000, 16384, 0, 40000] + [2000] * 70 + [20000] * 3
    r.shuffle(counts)
    order = torch.randperm(sum(counts), generator=gen)
    blocks = list(order.split(counts))
    w = torch.randint(0, 50, (4, len(order)), generator=gen).float()
    check_select(dev, w, blocks, [r.choice([0, 1, n // 2, n, n + 3]) for n in counts], 1, 2)


def test_protected_ends_that_are_more_than_stays_and_slots_outside(dev):
    gen = torch.Generator().manual_seed(4)
    w = torch.rand(2, 500, generator=gen) - 0.2
    slots = torch.randint(-300, 800, (400,), generator=gen)
    for keep, first, last in ((10, 20, 20), (30, 20, 20), (400, 0, 1000), (5, 1000, 0), (100, 0, 0)):
        check_select(dev, w, [slots], [keep], first, last)


def test_selection_recorded_and_on_another_stream(dev):
    gen = torch.Generator().manual_seed(5)
    for count in (900, 40000):
        w = torch.rand(2, count, generator=gen).to(dev)
        slots = torch.randperm(count, generator=gen).to(dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            other = CacheEviction.select(w, slots, [count], count // 2)
        torch.cuda.current_stream(dev).wait_stream(side)
        want = CacheEviction.select(w, slots, [count], count // 2)
        assert torch.equal(other.positions, want.positions)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph):
            kept = CacheEviction.select(w, slots, [count], count // 2)
        for _ in range(3):
            w.copy_(torch.rand(2, count, generator=gen))
            graph.replay()
            torch.cuda.synchronize(dev)
            assert torch.equal(kept.slots, CacheEviction.select(w, slots, [count], count // 2).slots)


def test_select_refuses(dev):
    w, slots = torch.zeros(2, 10, device=dev), torch.arange(10, device=dev)
    for args in ((w, slots, [9], 3), (w, slots, [10], -1), (w, slots, [11, -1], 3), (w.double(), slots, [10], 3), (w[0], slots, [10], 3),
                 (w, slots.int(), [10], 3), (w.t().contiguous().t(), slots, [10], 3)):
        with pytest.raises(ValueError):
            CacheEviction.select(*args)
    for more in (dict(first=-1), dict(last=-1)):
        with pytest.raises(ValueError):
            CacheEviction.select(w, slots, [10], 3, **more)
    assert CacheEviction.select(w, slots[:0], [], 3).counts == []
    assert CacheEviction.select(w, slots[:0], [0, 0], 3).positions.numel() == 0


# ---------------------------------------------------------------------------
# moving
# ---------------------------------------------------------------------------
def pool_values(op, layer, slots):
    pool = op.kv_cache
    if hasattr(pool, "k_codes"):
        return rows64(pool, 0, layer, slots), rows64(pool, 1, layer, slots)
    return keys64(op, layer, slots), pool.v_cache(layer).cpu().double().reshape(-1, op.num_kv_heads, op.head_dim)[slots]


def raw(op):
    pool = op.kv_cache
    if hasattr(pool, "k_codes"):
        return [t.view(torch.uint8).clone() for i in range(pool.num_layers)
                for t in (pool.k_codes(i), pool.v_codes(i), pool.k_scales(i), pool.v_scales(i))]
    return [t.clone().view(torch.uint8) for i in range(pool.num_layers) for t in (pool.k_cache(i), pool.v_cache(i))]


@pytest.mark.parametrize("dtype, codes", [(BF16, None), (F16, None), (F32, None), (BF16, E4M3), (F16, INT8)])
@pytest.mark.parametrize("heads, rotary, mrope", [((4, 2, 128), 128, None), ((16, 16, 64), 32, None), ((4, 1, 256), 128, (24, 20, 20)),
                                                  ((2, 1, 16), 6, None), ((3, 3, 64), 0, None)])
@pytest.mark.parametrize("n", [1, 15, 200])
def test_moves(dev, dtype, codes, heads, rotary, mrope, n):
    gen = torch.Generator().manual_seed(n)
    op = make_op(dev, *heads, 8, dtype, 70, codes, rotary=rotary, mrope=mrope, layers=3)
    for layer in range(3):
        fill(op, gen, layer)
    e = CacheEviction(op)
    order = torch.randperm(e.num_slots, generator=gen)
    source, target = order[:n].clone(), order[n: 2 * n].clone()
    shifts = torch.randint(-500, 500, (n,), generator=gen)
    shifts[::4] = 0
    if n > 10:  # slots outside the pool: such tokens are skipped
        source[3], target[5], source[7] = -1, e.num_slots, 1 << 40
    ok = (source >= 0) & (source < e.num_slots) & (target < e.num_slots)
    weights = torch.rand(op.num_kv_heads, e.num_slots, generator=gen).to(dev)
    old_weights, old, old_raw = weights.cpu(), [pool_values(op, i, source[ok]) for i in range(3)], raw(op)
    e.move(source.to(dev), target.to(dev), shifts.to(dev), weights)
    want = old_weights.clone()
    want[:, target[ok]] = old_weights[:, source[ok]]
    assert torch.equal(weights.cpu(), want)
    still = shifts[ok] == 0
    for layer in range(3):
        (k, v), (k0, v0) = pool_values(op, layer, target[ok]), old[layer]
        assert torch.equal(v, v0)
        assert torch.equal(k[still], k0[still])
        exact, size = turned64(op, k0, shifts[ok]), turned64_abs(op, k0)
        # products and sum (three units of their sizes) and the cosine (two more under mRoPE), then the one rounding to the type
        slack = 6 * 2.0**-24 * size
        if codes is None:
            assert bool(((k - exact).abs() <= slack + HALF[dtype] * (exact.abs() + slack)).all())
        else:
            # half a step of the row's scale, which may come out one power off where the maximum lies on an edge: e4m3 steps
            # are 2^-3 of an element (2^-9 of the largest for the smallest elements), int8 ones 1/64 of the largest
            top = exact.abs().amax(-1, keepdim=True)
            step = torch.maximum(exact.abs() / 16, top * 2.0**-16) if codes == E4M3 else top / 126
            assert bool(((k - exact).abs() <= step * (1 + 2.0**-10) + 2 * slack).all())
    # everything else is as it was
    touched = torch.zeros(e.num_slots, dtype=torch.bool)
    touched[target[ok]] = True
    for a, b in zip(raw(op), old_raw):
        if codes is not None:
            a, b = (t.view(t.shape[0], t.shape[1], t.shape[2], -1).transpose(1, 2) for t in (a, b))
        a, b = (t.reshape(e.num_slots, -1).cpu() for t in (a, b))
        assert torch.equal(a[~touched], b[~touched])
    # again without shifts: bit for bit
    e.move(target.to(dev), torch.where(ok, source, -1).to(dev))
    for layer in range(3):
        k, v = pool_values(op, layer, source[ok])
        k2, v2 = pool_values(op, layer, target[ok])
        assert torch.equal(k, k2) and torch.equal(v, v2)


def test_moves_between_layers_that_are_tensors_of_their_own(dev):
    from types import SimpleNamespace

    gen = torch.Generator().manual_seed(1)
    op = make_op(dev, 4, 2, 64, 8, BF16, 30)
    layers = [[torch.randn(30, 8, 2, 64, generator=gen).to(dev, BF16) for _ in range(2)] for _ in range(3)]
    op.kv_cache = SimpleNamespace(num_layers=3, k_cache=lambda i: layers[i][0], v_cache=lambda i: layers[i][1])
    e = CacheEviction(op)
    before = [[t.clone() for t in pair] for pair in layers]
    weights = torch.rand(2, 240, generator=gen).to(dev)
    w0 = weights.clone()
    source, target = torch.arange(10, 20, device=dev), torch.arange(100, 110, device=dev)
    e.move(source, target, weights=weights)
    for pair, old in zip(layers, before):
        for t, o in zip(pair, old):
            assert torch.equal(t.view(240, -1)[target], o.view(240, -1)[source])
    assert torch.equal(weights[:, target], w0[:, source])


def test_move_refuses(dev):
    op = make_op(dev, 4, 2, 64, 8, BF16, 30)
    e = CacheEviction(op)
    a, b = torch.arange(4, device=dev), torch.arange(10, 14, device=dev)
    for args in ((a, b[:3]), (a.int(), b), (a, b, b[:2]), (a, b.cpu()), (a, b, b.int())):
        with pytest.raises((ValueError, native.ViewAttnError)):
            e.move(*args)
    with pytest.raises(ValueError, match="weights"):
        e.move(a, b, weights=torch.zeros(2, 3, device=dev))
    e.move(a[:0], b[:0], a[:0])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, codes", [(BF16, None), (F32, None), (BF16, E4M3)])
@pytest.mark.parametrize("close_gaps", [False, True])
def test_a_block_is_read_evicted_from_and_read_again(dev, dtype, codes, close_gaps):
    r, gen = random.Random(1), torch.Generator().manual_seed(1)
    P, D, hq, hkv, layers = 16, 128, 8, 2, 2
    op = make_op(dev, hq, hkv, D, P, dtype, 100, codes, layers=layers)
    for layer in range(layers):
        fill(op, gen, layer)
    allocator = PageAllocator(100, P, dev)
    ops, e = BlockKVOps(op.kv_cache, op, allocator), CacheEviction(op)
    block, own = (ops.create_block() for _ in range(2))
    for b, n in ((block, 333), (own, 21)):
        b.page_starts = allocator.alloc_pages(-(-n // P)).tolist()
        b.num_tokens, b.token_ids = n, [r.randrange(1000) for _ in range(n)]
    weights = e.new_weights()
    weights.fill_(7.0)  # pages were someone else's: what is handed out anew starts from nothing
    for b in (block, own):
        e.clear(weights, torch.from_numpy(token_slots(b)))

    def step(view, seed):
        g = torch.Generator().manual_seed(seed)
        group = WorkerGroup(cache_structure=[view])
        slot = own.page_starts[own.num_tokens // P] + own.num_tokens % P
        meta = op.prepare(group, {id(own): None}, torch.tensor([slot], dtype=torch.int32, device=dev))
        q = torch.randn(1, hq * D, generator=g).to(dev, dtype)
        return meta, q

    sums = torch.zeros(hkv, e.num_slots, dtype=torch.float64)
    sums += weights.cpu().double()
    slack = torch.zeros_like(sums)
    for seed in range(3):
        meta, q = step([block, own], seed)
        plan = e.plan(meta)
        for layer in range(layers):
            _, lse = op.attend(q, layer, meta, return_lse=True)
            sums, s = weights64(op, q, lse, meta, sums, layer)
            slack += s
            e.accumulate(q, lse, layer, plan, weights)
    assert bool(((weights.cpu().double() - sums).abs() <= slack).all())

    slots = torch.from_numpy(token_slots(block))
    want = chosen(weights.cpu(), slots, 100, 4, 16)
    old = [pool_values(op, layer, slots) for layer in range(layers)]
    old_sums, ids, pages = weights.cpu(), list(block.token_ids), list(block.page_starts)
    small = ops.evict_tokens(block, weights, 100, first=4, last=16, close_gaps=close_gaps)
    assert (small.num_tokens, small.num_pages, small.mrope_span) == (100, 7, 100 if close_gaps else 333)
    assert small.token_ids == [ids[i] for i in want.tolist()]
    assert (block.num_tokens, block.page_starts, block.token_ids) == (333, pages, ids)
    new = torch.from_numpy(token_slots(small))
    assert torch.equal(weights.cpu()[:, new], old_sums[:, slots[want]])
    tail = torch.arange(small.page_starts[-1] + 4, small.page_starts[-1] + P)
    assert bool((weights.cpu()[:, tail] == 0).all())
    for layer in range(layers):
        k, v = pool_values(op, layer, new)
        assert torch.equal(v, old[layer][1][want])
        if not close_gaps:
            assert torch.equal(k, old[layer][0][want])

    # attention over what is left: the old view with everything else masked
    meta, q = step([small, own], 9)
    out, lse = op.attend(q, 0, meta, return_lse=True)
    order = torch.cat([new, torch.from_numpy(token_slots(own)), torch.tensor([own.page_starts[1] + 5])])
    k, v = pool_values(op, 0, order)
    loc = meta.sub_loc.cpu()
    x = q.cpu().double().view(1, hq, D)
    parts = [turned64(op, x, loc[i: i + 1])[0].view(hkv, hq // hkv, D) for i in range(2)]
    score = torch.cat([torch.einsum("hgd,nhd->hgn", p, kk) for p, kk in zip(parts, (k[:100], k[100:]))], dim=-1) / D**0.5
    exact = torch.einsum("hgn,nhd->hgd", torch.softmax(score, -1), v).reshape(1, -1)
    bound = 2e-2 + 1e-2 * exact.abs() if dtype == BF16 else 1e-5 + 1e-5 * exact.abs()  # the attention's own
    assert bool(((out.cpu().double() - exact).abs() <= bound).all())
    assert bool(((lse.cpu().double() - torch.logsumexp(score, -1).reshape(1, -1)).abs() <= (2e-2 if dtype == BF16 else 1e-5)).all())
    # the block grows on from its span
    before = small.mrope_span
    small.append_token(None)
    assert small.mrope_span == before + 1


def test_evictions_that_leave_all_or_nothing(dev):
    op = make_op(dev, 4, 2, 64, 16, BF16, 40)
    fill(op, torch.Generator().manual_seed(2))
    allocator = PageAllocator(40, 16, dev)
    ops = BlockKVOps(op.kv_cache, op, allocator)
    weights = CacheEviction(op).new_weights()
    block = ops.create_block()
    block.page_starts, block.num_tokens = allocator.alloc_pages(2).tolist(), 20
    same = ops.evict_tokens(block, weights, 50)
    assert same.num_tokens == 20 and same.mrope_span_override is None and same.page_starts != block.page_starts
    none = ops.evict_tokens(block, weights, 0)
    assert (none.num_tokens, none.num_pages, none.mrope_span) == (0, 0, 20)
    image = ops.create_block()
    image.page_starts, image.num_tokens, image.mrope_span_override = block.page_starts, 20, 9
    with pytest.raises(ValueError, match="close_gaps"):
        ops.evict_tokens(image, weights, 5, close_gaps=True)
    assert ops.evict_tokens(image, weights, 5).mrope_span == 9
    for bad in (dict(keep=-1), dict(keep=3, first=-1), dict(keep=3, last=-2)):
        with pytest.raises(ValueError, match="negative"):
            ops.evict_tokens(block, weights, **bad)
    with pytest.raises(ValueError, match="weights"):
        ops.evict_tokens(block, weights[:, :-1], 5)


def test_weights_are_forgotten(dev):
    """Of the slots that are in the pool; a slot may be named twice, and in any whole type."""
    e = CacheEviction(make_op(dev, 8, 4, 64, 16, torch.float16, 8))
    for slots in ([], [5], [-1, 3, 127, 128, 3, 2**40], [0, 64]):
        weights = torch.rand(4, 128, device=dev)
        want = weights.clone()
        for s in slots:
            if 0 <= s < 128:
                want[:, s] = 0.0
        e.clear(weights, torch.tensor(slots, dtype=torch.int64, device=dev))
        assert torch.equal(weights, want)
    weights = torch.rand(4, 128, device=dev)
    want = weights.clone()
    want[:, 1:9:2] = 0.0
    e.clear(weights, torch.arange(10, dtype=torch.int32)[1:9:2])
    assert torch.equal(weights, want)


def test_rotated_keys_move_to_where_they_would_have_been_rotated(dev):
    """Keys turned by a stretched rotation and moved with its unit table: those of the new positions. Over its table with the
    attention factor, by which they would grow, a turn is refused before anything is taken; a plain move is not."""
    gen = torch.Generator().manual_seed(11)
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    r = RotaryEmbedding(64, 32, 1e5, scaling=yarn, device=dev)
    pool = MHAKVCache(2, 1, 64, 40, 8, F32, dev)
    op, scaled = (SharedCacheAttention(pool, r.cos_sin_cache(5000, unit=unit), 4, 2, 64, 8, F32, dev, rotary_dim=32) for unit in (True, False))
    k = torch.randn(100, 2, 64, generator=gen)
    positions, shifts = torch.randint(2000, 4000, (100,), generator=gen), torch.randint(-2000, 1000, (100,), generator=gen)
    plain = RotaryEmbedding(64, 32, 1e5, scaling=dict(yarn, attention_factor=1.0), device=dev)
    pool.k_cache(0).view(-1, 2, 64)[:100] = plain(positions.to(dev), k.to(dev))[0]
    pool.v_cache(0).zero_()
    source, target = torch.arange(100, device=dev), torch.arange(150, 250, device=dev)
    CacheEviction(op).move(source, target, shifts.to(dev))
    got = pool.k_cache(0).view(-1, 2, 64)[150:250].cpu().double()
    angle = (positions + shifts).double()[:, None] * r.inv_freq.cpu()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = k.double()[..., :16], k.double()[..., 16:32]
    want = torch.cat([a * c - b * s, b * c + a * s, k.double()[..., 32:]], dim=-1)
    # a rotation is off by its cosine (four units), two products and a sum, of both elements of a pair; twice
    size = torch.cat([a.abs() + b.abs()] * 2 + [torch.zeros(100, 2, 32)], dim=-1)
    assert bool(((got - want).abs() <= 2 * 7 * 2.0**-24 * size).all())
    e, allocator = CacheEviction(scaled), PageAllocator(40, 8, dev)
    with pytest.raises(ValueError, match="unit"):
        e.move(source, target, shifts.to(dev))
    e.move(source, target)
    ops = BlockKVOps(pool, scaled, allocator)
    block = ops.create_block()
    block.page_starts, block.num_tokens = allocator.alloc_pages(3).tolist(), 20
    free = allocator.free_page_starts.numel()
    with pytest.raises(ValueError, match="unit"):
        ops.evict_tokens(block, e.new_weights(), 10, close_gaps=True)
    assert allocator.free_page_starts.numel() == free
    assert ops.evict_tokens(block, e.new_weights(), 10).num_tokens == 10
