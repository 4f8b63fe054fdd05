"""Attention weights by cached token against their definition in 64 bits."""

import random

import pytest
import torch

from async_llm_amd import native
from async_llm_amd.kvcache.mha_pool import MHAKVCache
from async_llm_amd.shared_cache import CacheEviction, PrefillSpec, SharedCacheAttention, WorkerGroup
from tests.eviction_util import blocks_of, fill, make_op, weights64
from tests.quant_util import quantised32, write

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def decode_step(op, r, workers, lengths, shared=None, aside=False):
    """A decode plan: every worker reads the shared block and one or two of its own and writes the last (``aside``: a block outside
    its view)."""
    P = op.page_size
    pages = list(range(op.kv_cache.num_pages if hasattr(op.kv_cache, "num_pages") else op.kv_cache.k_cache(0).shape[0]))
    r.shuffle(pages)
    common = blocks_of(op, r, [shared], pages) if shared else []
    views, targets, pending, slots = [], [], {}, []
    for w in range(workers):
        mine = blocks_of(op, r, [r.choice(lengths) for _ in range(r.randint(1, 2))], pages)
        target = blocks_of(op, r, [r.choice(lengths)], pages)[0] if aside and w % 2 else mine[-1]
        views.append(common + mine)
        targets.append(target)
        opened = None if target.has_capacity else pages.pop() * P
        pending[id(target)] = opened
        starts = target.page_starts + ([] if opened is None else [opened])
        slots.append(starts[target.num_tokens // P] + target.num_tokens % P)
    group = WorkerGroup(cache_structure=views, write_to=targets)
    return op.prepare(group, pending, torch.tensor(slots, dtype=torch.int32, device=op.device))


def chunk_specs(op, r, news, prefix, context, pages, three=False):
    P, specs = op.page_size, []
    shared = blocks_of(op, r, [context], pages) if context else []
    for n in news:
        held = r.randint(0, prefix)
        own = blocks_of(op, r, [held + n], pages)[0]
        rel = torch.stack([torch.arange(n), torch.arange(n) // 2, torch.arange(n) % 5]) if three else None
        specs.append(PrefillSpec(shared + blocks_of(op, r, [r.randint(1, 40)], pages), torch.tensor(own.page_starts), n, held, mrope_rel=rel))
    return specs


def inputs(op, meta, gen):
    """Queries, and the log-sums that the op's own attention gives (the definition takes any)."""
    q = torch.randn(meta.num_workers, op.num_qo_heads * op.head_dim, generator=gen).to(op.device, op.dtype)
    _, lse = op.attend(q, 0, meta, return_lse=True)
    return q, lse


def check(op, meta, gen, window=0, q=None, lse=None):
    if q is None:
        q, lse = inputs(op, meta, gen)
    e = CacheEviction(op)
    weights = (torch.rand(op.num_kv_heads, e.num_slots, generator=gen) * 0.1).to(op.device)
    want, slack = weights64(op, q, lse, meta, weights, window=window)
    before = weights.clone()
    got = e.accumulate(q, lse, 0, e.plan(meta, window), weights, out=before.clone())
    assert torch.equal(weights, before)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= slack).all()), f"off by {float((off / slack).max())} times what rounding allows"
    # in place: the same bits
    assert e.accumulate(q, lse, 0, e.plan(meta, window), weights) is weights and torch.equal(weights, got)
    return got


@pytest.mark.parametrize("dtype, codes", [(BF16, None), (F16, None), (F32, None), (BF16, E4M3), (F16, INT8), (F32, E4M3)])
@pytest.mark.parametrize("heads", [(4, 1, 128), (4, 4, 64), (32, 2, 64), (6, 2, 256), (5, 1, 32), (6, 3, 128), (12, 12, 64)])
def test_decode_steps(dev, dtype, codes, heads):
    r, gen = random.Random(1), torch.Generator().manual_seed(1)
    op = make_op(dev, *heads, 16, dtype, 200, codes)
    fill(op, gen)
    check(op, decode_step(op, r, 5, [1, 15, 16, 17, 130], shared=300), gen)


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("codes", [None, E4M3])
def test_pages_and_writers_outside_their_views(dev, page, codes):
    r, gen = random.Random(page), torch.Generator().manual_seed(page)
    op = make_op(dev, 8, 2, 64, page, BF16, 2400 // page + 60, codes)
    fill(op, gen)
    check(op, decode_step(op, r, 6, [1, 3, 64, 129], shared=200, aside=True), gen)


@pytest.mark.parametrize("dtype, codes", [(BF16, None), (F16, None), (F32, None), (BF16, INT8), (F32, E4M3)])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (6, 2, 256), (3, 1, 16)])
@pytest.mark.parametrize("window", [0, 7])
def test_chunks(dev, dtype, codes, heads, window):
    r, gen = random.Random(3), torch.Generator().manual_seed(3)
    op = make_op(dev, *heads, 16, dtype, 120, codes)
    fill(op, gen)
    specs = chunk_specs(op, r, [1, 33, 150], 20, 300, list(range(120)))
    check(op, op.prepare_prefill_batch(specs), gen, window)


@pytest.mark.parametrize("codes", [None, E4M3])
@pytest.mark.parametrize("rotary", [32, 20, 0])
def test_parts_of_a_head_and_three_axes(dev, codes, rotary):
    r, gen = random.Random(4), torch.Generator().manual_seed(4)
    op = make_op(dev, 8, 2, 64, 16, BF16, 120, codes, rotary=rotary)
    fill(op, gen)
    check(op, op.prepare_prefill_batch(chunk_specs(op, r, [40, 5], 20, 100, list(range(120)))), gen)
    if rotary == 32:
        op = make_op(dev, 8, 2, 64, 16, BF16, 120, codes, rotary=32, mrope=(6, 5, 5))
        fill(op, gen)
        check(op, op.prepare_prefill_batch(chunk_specs(op, r, [40, 5], 20, 100, list(range(120)), three=True)), gen)


def test_mixed_steps(dev):
    r, gen = random.Random(5), torch.Generator().manual_seed(5)
    op = make_op(dev, 8, 2, 128, 16, BF16, 200)
    fill(op, gen)
    pages = list(range(200))
    shared = blocks_of(op, r, [100], pages)[0]
    own, aside = blocks_of(op, r, [33, 20], pages)
    group = WorkerGroup(cache_structure=[[shared, own], [shared]], write_to=[own, aside])
    slots = torch.tensor([own.page_starts[2] + 1, aside.page_starts[1] + 4], dtype=torch.int32, device=dev)
    specs = chunk_specs(op, r, [50], 10, 200, pages)
    meta = op.prepare_mixed(group, {id(own): None, id(aside): None}, slots, specs)
    check(op, meta, gen)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_pools_off_16_byte_boundaries(dev, dtype):
    """Pools that the matrix cores do not read from, under plans with items of all kinds."""
    class Apart(MHAKVCache):
        def __init__(self, pages):
            self._num_layers, self._device = 1, dev
            self._arrays = [torch.zeros(pages * 16 * 2 * 64 + 1, dtype=dtype, device=dev)[1:].view(pages, 16, 2, 64) for _ in "kv"]
            self._kv_buffer = self._arrays[0]

        def k_cache(self, layer):
            return self._arrays[0]

        def v_cache(self, layer):
            return self._arrays[1]

    r, gen = random.Random(6), torch.Generator().manual_seed(6)
    like = make_op(dev, 8, 2, 64, 16, dtype, 4)
    op = SharedCacheAttention(Apart(120), like.cos_sin_cache, 8, 2, 64, 16, dtype, dev)
    fill(op, gen)
    assert op.kv_cache.k_cache(0).data_ptr() % 16
    pages = list(range(120))
    for meta in (op.prepare_prefill_batch(chunk_specs(op, r, [70, 3], 20, 300, pages)), decode_step(op, r, 6, [1, 17, 130], shared=200)):
        q = torch.randn(meta.num_workers, 512, generator=gen).to(dev, dtype)
        check(op, meta, gen, q=q, lse=5.0 + torch.rand(meta.num_workers, 8, generator=gen).to(dev))  # (attention takes no such pool)


def test_a_view_that_lists_a_block_twice(dev):
    r, gen = random.Random(6), torch.Generator().manual_seed(6)
    op = make_op(dev, 4, 2, 64, 16, BF16, 40)
    fill(op, gen)
    pages = list(range(40))
    a, b = blocks_of(op, r, [70, 20], pages)
    group = WorkerGroup(cache_structure=[[a, a, b]], write_to=[b])
    slot = b.page_starts[1] + 4
    check(op, op.prepare(group, {id(b): None}, torch.tensor([slot], dtype=torch.int32, device=dev)), gen)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_nobody_sees_does_not_matter(dev, dtype):
    """NaN and infinities in slots behind the last token and in later tokens of a chunk reach no other sum; rows whose log-sum
    is -inf count nothing."""
    r, gen = random.Random(7), torch.Generator().manual_seed(7)
    op = make_op(dev, 8, 2, 128, 16, dtype, 60)
    fill(op, gen)
    pages = list(range(60))
    specs = chunk_specs(op, r, [37], 0, 50, pages)
    meta = op.prepare_prefill_batch(specs)
    q, lse = inputs(op, meta, gen)
    starts = specs[0].self_page_starts.tolist()
    k = op.kv_cache.k_cache(0)
    k[starts[-1] // 16, 5:] = float("nan")  # behind the 37 tokens
    k[starts[1] // 16, 3] = float("inf")  # token 19: rows before it do not see it
    k[pages[0]] = float("nan")
    lse[3] = -float("inf")
    e = CacheEviction(op)
    got = e.accumulate(q, lse, 0, e.plan(meta), e.new_weights()).cpu().double()
    bad = starts[1] + 3
    k[starts[1] // 16, 3] = 0.0  # (the definition of the others does not look at it)
    k.nan_to_num_()
    want, slack = weights64(op, q, lse, meta, torch.zeros(2, e.num_slots))
    keep = torch.arange(e.num_slots) != bad
    assert bool(((got - want).abs() <= slack)[:, keep].all())
    unseen = want == 0
    assert bool((got[unseen] == 0).all())


def test_large_and_small_queries_and_keys(dev):
    """Scores as sums of large and small products in float16, whose queries are brought into range row by row."""
    r, gen = random.Random(8), torch.Generator().manual_seed(8)
    op = make_op(dev, 4, 2, 64, 16, F16, 40)
    fill(op, gen)
    op.kv_cache.k_cache(0).mul_(1000.0)
    meta = decode_step(op, r, 3, [50, 90], shared=100)
    size = torch.tensor([1e-6, 1e-3, 1e-2])[:, None]
    q = (torch.randn(3, 256, generator=gen) * size).to(dev, F16)
    _, lse = op.attend(q, 0, meta, return_lse=True)
    check(op, meta, gen, q=q, lse=lse)


@pytest.mark.parametrize("dtype, codes", [(BF16, None), (BF16, E4M3), (F16, INT8)])
@pytest.mark.parametrize("least", [-5, -7, -60])
def test_keys_of_very_different_sizes_under_many_rows(dev, dtype, codes, least):
    """Tiles of many rows scale the keys of a token, or of 32 tokens, by a power of two: rows of zeros and tiny rows beside others."""
    r, gen = random.Random(least), torch.Generator().manual_seed(-least)
    op = make_op(dev, 8, 2, 64, 16, dtype, 80, codes)
    size = 2.0 ** torch.randint(least, 2, (80, 16, 2, 1), generator=gen)
    size[torch.rand(80, 16, 2, 1, generator=gen) < 0.1] = 0.0
    x = torch.randn(80, 16, 2, 64, generator=gen) * size
    if codes is None:
        op.kv_cache.k_cache(0).copy_(x)
        op.kv_cache.v_cache(0).zero_()
    else:
        for which in (0, 1):
            write(op.kv_cache, which, 0, torch.arange(1280), *quantised32(x.view(1280, 2, 64), op.kv_cache.code_dtype))
    check(op, op.prepare_prefill_batch(chunk_specs(op, r, [90, 35], 20, 300, list(range(80)))), gen)


def test_sums_are_one_for_each_row(dev):
    """The weights that a row gives away add up to 1 within its log-sum's and the attention's own rounding of the query."""
    r, gen = random.Random(9), torch.Generator().manual_seed(9)
    op = make_op(dev, 8, 2, 128, 16, F32, 100)
    fill(op, gen)
    meta = decode_step(op, r, 4, [100, 200], shared=300)
    q, lse = inputs(op, meta, gen)
    e = CacheEviction(op)
    got = e.accumulate(q, lse, 0, e.plan(meta), e.new_weights())
    assert abs(float(got.double().sum()) - 4 * 8) < 1e-3
    base2 = e.accumulate(q, lse / 0.6931471805599453, 0, e.plan(meta), e.new_weights(), lse_base2=True)
    assert torch.allclose(got, base2, rtol=1e-4, atol=1e-9)


def test_recorded_streams_and_strided_queries(dev):
    r, gen = random.Random(10), torch.Generator().manual_seed(10)
    op = make_op(dev, 8, 2, 128, 16, BF16, 100)
    fill(op, gen)
    meta = op.prepare_prefill_batch(chunk_specs(op, r, [60], 10, 200, list(range(100))))
    q, lse = inputs(op, meta, gen)
    e = CacheEviction(op)
    plan = e.plan(meta)
    want = e.accumulate(q, lse, 0, plan, e.new_weights())
    wide = torch.randn(60, 8 * 128 + 24, generator=gen).to(dev, BF16)  # rows at odd places
    wide[:, 3: 3 + 1024] = q
    assert torch.equal(e.accumulate(wide[:, 3: 1027], lse, 0, plan, e.new_weights()), want)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = e.accumulate(q, lse, 0, plan, e.new_weights())
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(other, want)
    weights, sums = e.new_weights(), e.new_weights()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph):
        e.accumulate(q, lse, 0, plan, weights, out=sums)
    for _ in range(3):
        sums.zero_()
        weights.copy_(torch.rand(weights.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(sums, e.accumulate(q, lse, 0, plan, weights, out=e.new_weights()))


def test_refusals(dev):
    r, gen = random.Random(11), torch.Generator().manual_seed(11)
    op = make_op(dev, 8, 2, 128, 16, BF16, 100)
    fill(op, gen)
    meta = decode_step(op, r, 3, [40])
    q, lse = inputs(op, meta, gen)
    e = CacheEviction(op)
    plan, weights = e.plan(meta), e.new_weights()
    with pytest.raises(ValueError, match="window"):
        e.plan(meta, -1)
    with pytest.raises(ValueError, match="this op planned"):
        CacheEviction(make_op(dev, 8, 2, 128, 16, BF16, 100)).plan(meta)
    for bad in (q[:2], q.float(), q.cpu()):
        with pytest.raises((ValueError, native.ViewAttnError)):
            e.accumulate(bad, lse, 0, plan, weights)
    for bad in (lse[:2], lse.double(), lse[:, :4]):
        with pytest.raises(ValueError, match="lse"):
            e.accumulate(q, bad, 0, plan, weights)
    for bad in (weights[:1], weights.double(), weights[:, :-1]):
        with pytest.raises(ValueError, match="weights"):
            e.accumulate(q, lse, 0, plan, bad)
        with pytest.raises(ValueError, match="out"):
            e.accumulate(q, lse, 0, plan, weights, out=bad)
    coded = CacheEviction(make_op(dev, 8, 2, 128, 16, BF16, 100, E4M3))
    with pytest.raises(native.ViewAttnError, match="another shape"):
        coded.accumulate(q, lse, 0, plan, coded.new_weights())
    other = make_op(dev, 8, 4, 128, 16, BF16, 100)
    f = CacheEviction(other)
    with pytest.raises(native.ViewAttnError, match="another shape"):
        f.accumulate(q, lse, 0, plan, f.new_weights())
