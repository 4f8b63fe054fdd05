"""The 8-bit cache as it is used: steps that store and attend, recorded and replayed, on other streams, over pools whose
offsets pass 32 bits, with blocks merged in between."""

from types import SimpleNamespace

import pytest
import torch

from async_llm_amd import native
from async_llm_amd.kvcache import QuantizedKVCache
from async_llm_amd.shared_cache import BlockKVOps, PrefillSpec, QuantizedCacheAttention
from async_llm_amd.shared_cache.attention_graph import SharedDecodeAttentionBuffers, SharedPrefillAttentionBuffers
from tests import quant_util as Q
from tests.test_gpu_quant_attend import check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(g, n, width, dtype):
    return torch.randn(n, width, generator=g).to(dtype).to(DEV)


def stored(op, step, k, v, layer=0):
    """The pool holds the codes of ``k`` (rotated in 32 bits) and ``v`` at the step's slots."""
    pool, s = op.kv_cache, step.slots.cpu().long()
    heads, D = pool.num_kv_heads, pool.head_dim
    k64 = Q.rotated(op, k.cpu().view(-1, heads, D), step.positions.cpu())
    off = Q.turn_error(k.cpu().view(-1, heads, D))
    for which, (x, room) in enumerate(((k64, off), (v.cpu().double().view(-1, heads, D), torch.zeros_like(off)))):
        codes = (pool.k_codes, pool.v_codes)[which](layer).cpu()[s // op.page_size, :, s % op.page_size]
        Q.assert_quantises(codes, Q.scales_of(pool, which, layer, s), x, room, pool.code_dtype)


@pytest.mark.parametrize("heads,page,dtype,codes", [((8, 2, 64), 16, BF16, E4M3), ((8, 2, 128), 4, F16, INT8), ((4, 2, 256), 16, F32, E4M3)])
def test_recorded_decode_steps(heads, page, dtype, codes):
    """A graph over fixed buffers follows every new plan; eager steps of the same op run between its replays."""
    W, depth, n_pages = 4, 3, 1024
    Hq, Hkv, D = heads
    op, pool, g = Q.make(DEV, heads, page, n_pages, dtype, codes)
    buffers = SharedDecodeAttentionBuffers(op, W, depth, max_pages=700, dummy_slots=torch.zeros(W, dtype=torch.int64))
    op.prepare_workspace([buffers])
    q, k, v = (torch.zeros(W, n * D, dtype=dtype, device=DEV) for n in (Hq, Hkv, Hkv))
    where, loc = torch.zeros(W, dtype=torch.int64, device=DEV), torch.full((W,), -1, dtype=torch.int32, device=DEV)
    batch = SimpleNamespace(attn_metadata=buffers.meta, positions=where, out_loc=loc, mrope_positions=None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        op.forward_with_lse(q, k, v, 0, batch)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = op.forward_with_lse(q, k, v, 0, batch)
    pages = Q.Pages(n_pages, page)
    common = pages.block(DEV, 70)
    for n, lengths in ((2, (900, 33)), (4, (5, 64, 300, 17)), (1, (40,)), (3, (16, 15, 1))):
        own = [pages.block(DEV, length, room=1) for length in lengths]
        step = Q.decode_step(op, pages, [[common, b] for b in own], own, g, buffers)
        loc.fill_(-1), where.zero_(), q.zero_()
        q[:n], k[:n], v[:n] = rows(g, n, Hq * D, dtype), rows(g, n, Hkv * D, dtype), rows(g, n, Hkv * D, dtype)
        loc[:n], where[:n] = step.slots, step.positions
        graph.replay()
        torch.cuda.synchronize()
        first, sums = out.clone(), lse.clone()
        stored(op, step, k[:n], v[:n])
        check(op, step, q[:n], range(n), [1] * n, first[:n], sums[:n])
        assert not first[n:].any() and torch.isinf(sums[n:]).all()
        eager = Q.decode_step(op, pages, [[common, b] for b in own], own, g)
        other = rows(g, n, Hq * D, dtype)
        got, got_lse = op.attend(other, 0, eager.meta, return_lse=True)
        check(op, eager, other, range(n), [1] * n, got, got_lse)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, first) and torch.equal(lse, sums)


@pytest.mark.parametrize("dtype,codes", [(BF16, E4M3), (F16, INT8)])
def test_recorded_chunks_over_fixed_buffers(dtype, codes):
    heads, page, workers, depth, most = (4, 2, 64), 16, 3, 2, 200
    op, pool, g = Q.make(DEV, heads, page, 300, dtype, codes)
    buffers = SharedPrefillAttentionBuffers(op, workers, depth, most, max_pages=200)
    op.prepare_workspace([buffers])
    q = torch.zeros(most, 4 * 64, dtype=dtype, device=DEV)
    op.attend(q, 0, buffers.meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = op.attend(q, 0, buffers.meta, return_lse=True)
    pages = Q.Pages(300, page)
    common = [pages.block(DEV, 90), pages.block(DEV, 16)]
    for new in ([1], [63, 65, 3], [130, 70], [16, 16, 16]):
        step = Q.prefill_step(op, [(common, pages.block(DEV, 7 * i, room=n), n) for i, n in enumerate(new)], buffers=buffers)
        assert step.meta.launch.readback is None
        n = sum(new)
        q.zero_()
        q[:n] = rows(g, n, 4 * 64, dtype)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            check(op, step, q, [sum(new[:r]) for r in range(len(new))], new, out[:n], lse[:n])
            assert not out[n:].any()
            op.attend(torch.randn_like(q), 0, buffers.meta)  # (the same workspace)


def test_recorded_chunks_that_are_read_back():
    """Two graphs of two plans share the op's scratch; replays follow the queries and the pool of their time."""
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 400, BF16, E4M3)
    op._reads_back = lambda pairs, pages: True
    pages = Q.Pages(400, 16)
    context = [pages.block(DEV, 700), pages.block(DEV, 30)]
    steps = [Q.prefill_step(op, [(context, pages.block(DEV, 9, room=n), n), (context[1:], pages.block(DEV, 0, room=40), 40)]) for n in (150, 260)]
    graphs = []
    for step in steps:
        n = sum(step.new)
        q = rows(g, n, 8 * 128, BF16)
        op.attend(q, 0, step.meta)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = op.attend(q, 0, step.meta, return_lse=True)
        graphs.append((graph, q, out, lse))
    slots = torch.cat([Q.slots_of(b) for b in context])
    for turn in range(3):
        for step, (graph, q, out, lse) in zip(steps, graphs):
            x = torch.randn(2, len(slots), 2, 128, generator=g) * 2.0 ** (4 * turn)  # (another largest scale as well)
            for which in range(2):
                Q.write(pool, which, 0, slots, *Q.quantised32(x[which] if which else x[which] * 2.0 ** (-3 * turn), E4M3))
            q.copy_(torch.randn(q.shape, generator=g).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            check(op, step, q, [0, step.new[0]], step.new, out, lse)
            eager, eager_lse = op.attend(q, 0, step.meta, return_lse=True)
            assert torch.equal(eager, out) and torch.equal(eager_lse, lse)


@pytest.mark.parametrize("back", [False, True])
def test_decodes_and_chunks_in_one_step(back):
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 400, BF16, INT8)
    op._reads_back = lambda pairs, pages: back
    pages = Q.Pages(400, 16)
    prompt = pages.block(DEV, 500)
    own = [pages.block(DEV, n, room=1) for n in (40, 16, 3)]
    alone = pages.block(DEV, 31, room=1)  # written from outside its writer's view
    chunk_context, chunks = [prompt, pages.block(DEV, 20)], [(pages.block(DEV, 5, room=70), 70), (pages.block(DEV, 0, room=9), 9)]
    views = [[prompt, own[0]], [own[1], own[2]], [own[1], own[2]], [prompt]]
    writers = [own[0], own[1], own[2], alone]
    decode = Q.decode_step(op, pages, views, writers, g)
    prefill = Q.prefill_step(op, [(chunk_context, b, n) for b, n in chunks])
    meta = op.prepare_mixed(decode.group, decode.pending, decode.slots, prefill.specs)
    assert (meta.launch.readback is not None) == back
    n = 4 + 79
    q, k, v = (rows(g, n, heads * 128, BF16) for heads in (8, 2, 2))
    step = SimpleNamespace(meta=meta, segments=decode.segments + prefill.segments, slots=torch.cat([decode.slots.long(), prefill.slots]),
                           positions=torch.cat([decode.positions, prefill.positions]))
    batch = SimpleNamespace(attn_metadata=meta, positions=step.positions, out_loc=step.slots, mrope_positions=None)
    out, lse = op.forward_with_lse(q, k, v, 0, batch)
    stored(op, step, k, v)
    check(op, step, q, [0, 1, 2, 3, 4, 74], [1, 1, 1, 1, 70, 9], out, lse)
    again, _ = op.attend(q, 0, meta, return_lse=True)
    assert torch.equal(again, out)


def test_tensors_of_another_stream():
    """Every entry point runs on the caller's current stream, behind what produced its tensors there."""
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 600, BF16, E4M3)
    pages = Q.Pages(600, 16)
    view = [[pages.block(DEV, 3000, room=1)]]
    a, b = torch.randn(4096, 4096, device=DEV), None
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            b = a @ a  # the stream is busy when the calls below are queued
        step = Q.decode_step(op, pages, view, [view[0][0]], g)
        q, k, v = (torch.randn(1, n * 128, generator=g).to(BF16).to(DEV, non_blocking=True) for n in (8, 2, 2))
        batch = SimpleNamespace(attn_metadata=step.meta, positions=step.positions, out_loc=step.slots, mrope_positions=None)
        out, lse = op.forward_with_lse(q, k, v, 0, batch)
        k_row, v_row = pool.load_kv(step.slots.long(), 0)
        target = torch.tensor([Q.slots_of(pages.block(DEV, 16))[3].item()], device=DEV)
        op.copy_shifted(step.slots.long(), target, 5)
    side.synchronize()
    stored(op, step, k, v)
    check(op, step, q, [0], [1], out, lse)
    for which, row in enumerate((k_row, v_row)):
        assert torch.equal(row.cpu(), Q.rows64(pool, which, 0, step.slots.cpu()).to(BF16))
    assert torch.equal(Q.rows64(pool, 1, 0, target.cpu()), Q.rows64(pool, 1, 0, step.slots.cpu()))


def test_offsets_past_32_bits():
    """Pages at both ends of a layer of more than 2^32 bytes of codes."""
    heads, page = (4, 4, 256), 16
    n_pages = (2**32 + 2**24) // (page * 4 * 256)
    codes = torch.zeros(2, 1, n_pages, 4, page, 256, dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.full((2, 1, n_pages, 4, page), 127, dtype=torch.uint8, device=DEV)
    pool = QuantizedKVCache.from_buffers(codes, scales, BF16)
    angle = torch.arange(4096, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, 256, 2, dtype=torch.float64) / 256)
    table = torch.cat([angle.cos(), angle.sin()], dim=1).float().to(DEV)
    op = QuantizedCacheAttention(pool, table, 4, 4, 256, page, BF16, DEV)
    g = torch.Generator().manual_seed(5)
    order = [n_pages - 1, 0, n_pages - 2, 5, n_pages - 30, 2**32 // (page * 1024), 77, n_pages - 9]
    slots = (torch.tensor(order)[:, None] * page + torch.arange(page)).reshape(-1)
    k, v = (rows(g, len(slots), 1024, BF16) for _ in range(2))
    pool.store_kv(k, v, slots.to(DEV), 0)
    back_k, back_v = pool.load_kv(slots.to(DEV), 0)

    def held(which, at):  # (a layer is too large to be brought to the host whole)
        at = torch.as_tensor(at, dtype=torch.int64).to(DEV)
        return Q.values64(codes.view(torch.uint8)[which, 0, at // page, :, at % page].cpu().view(E4M3), scales[which, 0, at // page, :, at % page].cpu())

    for which, (x, back) in enumerate(((k, back_k), (v, back_v))):
        c, s = Q.quantised32(x.cpu().float().view(-1, 4, 256), E4M3)
        assert torch.equal(held(which, slots), Q.values64(c, s))
        assert torch.equal(back.cpu(), held(which, slots).to(BF16))
    moved = (torch.tensor([n_pages - 3, 9])[:, None] * page + torch.arange(page)).reshape(-1)
    op.copy_shifted(slots[:32].to(DEV), moved.to(DEV), 0)
    assert all(torch.equal(held(w, moved), held(w, slots[:32])) for w in range(2))
    blocks = []
    for part in (order[:5], order[5:]):
        b = Q.Pages(1, page).block(DEV, 0)
        b.page_starts, b.spare, b.num_tokens = [p * page for p in part], [], len(part) * page - 1
        blocks.append(b)
    original = Q.rows64
    Q.rows64 = lambda pool_, which, layer, at: held(which, at)
    try:
        step = Q.decode_step(op, None, [blocks], [blocks[1]], g)
        q = rows(g, 1, 1024, BF16)
        out, lse = op.attend(q, 0, step.meta, return_lse=True)
        check(op, step, q, [0], [1], out, lse)
    finally:
        Q.rows64 = original


@pytest.mark.parametrize("heads,rotary,codes,dtype", [((8, 2, 128), None, E4M3, BF16), ((4, 4, 64), 32, INT8, F16), ((2, 1, 32), 18, E4M3, F32)])
def test_blocks_are_merged_and_read(heads, rotary, codes, dtype):
    """Two blocks are written, merged and appended to, then attended to and read back."""
    Hq, Hkv, D = heads
    op, pool, g = Q.make(DEV, heads, 16, 60, dtype, codes, rotary, layers=2)
    pages = Q.Pages(60, 16)
    allocator = SimpleNamespace(alloc_pages=lambda n: torch.tensor([pages.order.pop() * 16 for _ in range(n)], dtype=torch.int32))
    ops = BlockKVOps(pool, op, allocator)
    left, right = pages.block(op.device, 21), pages.block(op.device, 35)
    for block in (left, right):
        at = Q.slots_of(block)
        for layer in range(2):
            k, v = (rows(g, len(at), Hkv * D, dtype) for _ in range(2))
            batch = SimpleNamespace(positions=torch.arange(len(at), device=DEV), mrope_positions=None, out_loc=at.to(DEV))
            op.store_new_kv(k, v, layer, batch)
    merged = ops.merge_blocks(left, right)
    assert merged.num_tokens == 56
    for layer in range(2):
        for which in range(2):
            new, old = (Q.rows64(pool, which, layer, s) for s in (Q.slots_of(merged), torch.cat([Q.slots_of(left), Q.slots_of(right)])))
            assert torch.equal(new[:21], old[:21])
            if which:
                assert torch.equal(new[21:], old[21:])
            else:
                x = Q.rotated(op, old[21:].float(), torch.tensor([21]))
                s = Q.slots_of(merged)[21:]
                Q.assert_quantises(pool.k_codes(layer).cpu()[s // 16, :, s % 16], Q.scales_of(pool, 0, layer, s), x, Q.turn_error(old[21:]), codes)
    tail = pages.block(op.device, 5, room=1)
    step = Q.decode_step(op, pages, [[merged, tail]], [tail], g)
    q = rows(g, 1, Hq * D, dtype)
    for layer in range(2):
        out, lse = op.attend(q, layer, step.meta, return_lse=True)
        check(op, step, q, [0], [1], out, lse, layer)


def test_work_of_no_rows_and_slots_twice():
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 20, BF16, E4M3)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    before = pool.k_codes(0).view(torch.uint8).clone()
    pool.store_kv(torch.empty(0, 256, dtype=BF16, device=DEV), torch.empty(0, 256, dtype=BF16, device=DEV), none, 0)
    k, v = pool.load_kv(none, 0)
    assert k.shape == v.shape == (0, 2, 128)
    op.copy_shifted(none, none, 7)
    assert torch.equal(pool.k_codes(0).view(torch.uint8), before)
    twice = torch.tensor([40, 40, 3, 40, -1], device=DEV)
    k, v = pool.load_kv(twice, 0)
    assert torch.equal(k.cpu()[:4], Q.rows64(pool, 0, 0, [40, 40, 3, 40]).to(BF16)) and not k[4].any()
    # one source for several targets
    op.copy_shifted(torch.tensor([40, 40], device=DEV), torch.tensor([200, 201], device=DEV), 0)
    assert torch.equal(Q.rows64(pool, 0, 0, [200, 201]), Q.rows64(pool, 0, 0, [40, 40]))
