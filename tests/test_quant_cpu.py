"""The 8-bit cache without a GPU: what it refuses, what its plans hold, and its number format against a second reading of
its definition."""

import math
import random
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from async_llm_amd import native
from async_llm_amd.attention_backend import ViewAttnBackend
from async_llm_amd.kvcache import MHAKVCache, QuantizedKVCache
from async_llm_amd.shared_cache import BlockKVOps, CacheBlock, PrefillSpec, QuantizedCacheAttention, SharedCacheAttention, WorkerGroup
from async_llm_amd.shared_cache.attention_graph import SharedDecodeAttentionBuffers, SharedPrefillAttentionBuffers
from tests import quant_util as Q
from tests.test_native_abi_cpu import decode_plan

CPU = torch.device("cpu")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROPE = native.VaRope(native.VA_ROPE_TABLE, 0, None, 0, 0, 0, None)
FAKE = 1 << 20  # an address that nothing reads: every call below is refused on the host


def make(heads=(8, 2, 64), page=16, pages=40, dtype=BF16, codes=E4M3, **more):
    pool = QuantizedKVCache(heads[1], 2, heads[2], pages, page, dtype, CPU, codes)
    return QuantizedCacheAttention(pool, torch.zeros(64, heads[2]), *heads, page, dtype, CPU, **more), pool


def block(starts, tokens, page=16):
    b = CacheBlock(CPU, page)
    b.page_starts, b.num_tokens = [s * page for s in starts], tokens
    return b


# ---------------------------------------------------------------------------
# the format
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_scales_hold_their_rows(codes):
    """The smallest power of two under which a row's largest element is no larger than the largest code."""
    largest = 448.0 if codes == E4M3 else 127.0
    r = random.Random(3)
    for top in [0.0, 1e-45, 2.0**-149, 1.0, largest, math.nextafter(largest, 1e9), 2.0 * largest] + [r.uniform(0.5, 1) * 2.0 ** r.randint(-126, 100) for _ in range(50)]:
        x = torch.tensor([[top, -top / 3, 0.0]], dtype=torch.float64).float().double()
        b = int(Q.scale_bytes(x, codes))
        held = float(x.max())
        assert 1 <= b <= 254 and held <= largest * 2.0 ** (b - 127)
        assert b == 1 or held > largest * 2.0 ** (b - 128)


def test_pools_start_empty_and_take_existing_arrays():
    pool = QuantizedKVCache(2, 3, 64, 5, 16, BF16, CPU)
    assert pool.k_codes(0).dtype == E4M3 and pool.k_codes(0).shape == (5, 2, 16, 64)
    assert pool.v_scales(2).dtype == torch.float8_e8m0fnu and pool.v_scales(2).shape == (5, 2, 16)
    assert (pool.v_scales(2).view(torch.uint8) == 127).all() and not pool.k_codes(1).view(torch.uint8).any()
    codes, scales = torch.zeros(2, 1, 4, 2, 8, 32, dtype=INT8), torch.full((2, 1, 4, 2, 8), 120, dtype=torch.uint8)
    other = QuantizedKVCache.from_buffers(codes, scales.view(torch.float8_e8m0fnu), F16)
    codes[1, 0, 3, 1, 7, 31] = 5
    assert other.v_codes(0)[3, 1, 7, 31] == 5 and other.code_dtype == INT8 and other.dtype == F16
    assert (other.num_layers, other.num_pages, other.page_size, other.num_kv_heads, other.head_dim) == (1, 4, 8, 2, 32)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("codes,scales,error", [
    (torch.zeros(2, 1, 4, 2, 8, 32, dtype=torch.uint8), torch.zeros(2, 1, 4, 2, 8, dtype=torch.uint8), native.ViewAttnError),
    (torch.zeros(1, 1, 4, 2, 8, 32, dtype=INT8), torch.zeros(1, 1, 4, 2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(2, 4, 2, 8, 32, dtype=INT8), torch.zeros(2, 4, 2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(2, 1, 4, 2, 8, 32, dtype=INT8), torch.zeros(2, 1, 4, 2, 4, dtype=torch.uint8), ValueError),
    (torch.zeros(2, 1, 4, 2, 8, 32, dtype=INT8), torch.zeros(2, 1, 4, 2, 8), ValueError),
    (torch.zeros(2, 1, 4, 2, 8, 48, dtype=INT8), torch.zeros(2, 1, 4, 2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(2, 1, 4, 2, 8, 64, dtype=INT8)[..., ::2], torch.zeros(2, 1, 4, 2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(2 * 4 * 2 * 8 * 32 + 1, dtype=INT8)[1:].view(2, 1, 4, 2, 8, 32), torch.zeros(2, 1, 4, 2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(1, dtype=INT8).expand(2, 1, 1 << 28, 1, 16, 16), torch.zeros(1, dtype=torch.uint8).expand(2, 1, 1 << 28, 1, 16), ValueError),
])
def test_arrays_that_are_no_pool(codes, scales, error):
    with pytest.raises(error):
        QuantizedKVCache.from_buffers(codes, scales, BF16)


def test_ops_that_do_not_fit_their_pool():
    op, pool = make()
    table = torch.zeros(64, 64)
    with pytest.raises(TypeError):
        SharedCacheAttention(pool, table, 8, 2, 64, 16, BF16, CPU)
    with pytest.raises(TypeError):
        QuantizedCacheAttention(MHAKVCache(2, 1, 64, 4, 16, BF16, CPU), table, 8, 2, 64, 16, BF16, CPU)
    for heads, page, dtype in (((8, 4, 64), 16, BF16), ((8, 2, 128), 16, BF16), ((8, 2, 64), 8, BF16), ((8, 2, 64), 16, F16), ((7, 2, 64), 16, BF16)):
        with pytest.raises(ValueError):
            QuantizedCacheAttention(pool, table, *heads, page, dtype, CPU)
    with pytest.raises(ValueError):
        QuantizedCacheAttention(pool, table, 8, 2, 64, 16, BF16, torch.device("meta"))
    with pytest.raises(ValueError):
        BlockKVOps(pool, make()[0], None)
    with pytest.raises(TypeError):
        ViewAttnBackend(SimpleNamespace(num_qo_heads=8, num_kv_heads=2, head_dim=64), pool, torch.zeros(1, 8, dtype=torch.int32))
    with pytest.raises(IndexError):
        pool.layer(2)
    with pytest.raises(IndexError):
        pool.layer(-1)


def test_tensors_that_no_gpu_holds():
    op, pool = make()
    batch = SimpleNamespace(positions=torch.zeros(1, dtype=torch.int64), mrope_positions=None, out_loc=torch.zeros(1, dtype=torch.int64))
    x = torch.zeros(1, 128, dtype=BF16)
    with pytest.raises(native.ViewAttnError):
        op.store_new_kv(x, x, 0, batch)
    with pytest.raises(native.ViewAttnError):
        pool.load_kv(torch.zeros(1, dtype=torch.int64), 0)
    with pytest.raises(native.ViewAttnError):
        op.copy_shifted(torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    step = op.prepare_prefill_batch([PrefillSpec([], torch.tensor([0], dtype=torch.int32), 3, 0)])
    with pytest.raises(native.ViewAttnError):
        op.attend(torch.zeros(3, 512, dtype=BF16), 0, step)
    with pytest.raises(ValueError):
        op.attend(torch.zeros(3, 512, dtype=BF16), 0, step, static_scratch=True)


@pytest.mark.parametrize("k,v,loc,where", [
    (torch.zeros(2, 128, dtype=F16), torch.zeros(2, 128, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)),
    (torch.zeros(2, 128, dtype=BF16), torch.zeros(3, 128, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)),
    (torch.zeros(2, 64, dtype=BF16), torch.zeros(2, 64, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)),
    (torch.zeros(2, 128, dtype=BF16), torch.zeros(2, 128, dtype=BF16), torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)),
    (torch.zeros(2, 128, dtype=BF16), torch.zeros(2, 128, dtype=BF16), torch.zeros(2), torch.zeros(2, dtype=torch.int64)),
    (torch.zeros(2, 128, dtype=BF16), torch.zeros(2, 128, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)),
    (torch.zeros(2, 128, dtype=BF16), torch.zeros(2, 128, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.zeros(2, 2, dtype=torch.int64)),
])
def test_rows_that_do_not_fit(k, v, loc, where, monkeypatch):
    op, pool = make()
    monkeypatch.setattr(native, "require_device", lambda t, name: None)
    monkeypatch.setattr(native, "call_on", lambda *a: pytest.fail("called"))
    with pytest.raises(ValueError):
        op.store_new_kv(k, v, 0, SimpleNamespace(positions=where, mrope_positions=None, out_loc=loc))


def test_outputs_and_queries_that_do_not_fit(monkeypatch):
    op, pool = make()
    monkeypatch.setattr(native, "require_device", lambda t, name: None)
    monkeypatch.setattr(native, "current_stream_ptr", lambda device: 0)
    monkeypatch.setattr(native, "call_on", lambda *a: pytest.fail("called"))
    step = op.prepare_prefill_batch([PrefillSpec([], torch.tensor([0], dtype=torch.int32), 3, 0)])
    q = torch.zeros(3, 512, dtype=BF16)
    for bad in (dict(q=q[:2]), dict(q=q.half()), dict(q=q, out=torch.zeros(3, 512)), dict(q=q, out=torch.zeros(3, 1024, dtype=BF16)[:, ::2]),
                dict(q=q, out=torch.zeros(2, 512, dtype=BF16)), dict(q=q, return_lse=True, lse=torch.zeros(3, 8, dtype=F16)),
                dict(q=q, return_lse=True, lse=torch.zeros(3, 4))):
        with pytest.raises(ValueError):
            op.attend(bad.pop("q"), 0, step, **bad)
    with pytest.raises(IndexError):
        op.attend(q, 2, step)
    slots = torch.zeros(4, dtype=torch.int64)
    ok = torch.zeros(4, 2, 64, dtype=BF16)
    for bad_slots, out in ((slots.int(), None), (slots.view(2, 2), None), (slots, (ok[:3], ok[:3])), (slots, (ok, ok.half())),
                           (slots, (ok, torch.zeros(4, 4, 64, dtype=BF16)[:, ::2])), (slots, (ok[:1].expand(4, 2, 64),) * 2)):
        with pytest.raises(ValueError):
            pool.load_kv(bad_slots, 0, out)
    for source, target in ((slots, slots[:3]), (slots.int(), slots.int()), (slots.view(2, 2), slots.view(2, 2))):
        with pytest.raises(ValueError):
            op.copy_shifted(source, target)


def test_pages_outside_the_pool():
    op, pool = make(pages=10)
    inside = block([9], 16)
    for bad in (block([10], 3), block([2, 1 << 20], 20), block([-1], 1)):
        with pytest.raises(ValueError, match="outside the pool"):
            op.prepare(WorkerGroup(cache_structure=[[inside, bad]], write_to=[bad]), {id(bad): None}, torch.tensor([3], dtype=torch.int32))
        with pytest.raises(ValueError, match="outside the pool"):
            op.prepare_prefill_batch([PrefillSpec([inside, bad], torch.tensor([32], dtype=torch.int32), 3, 0)])
    with pytest.raises(ValueError, match="outside the pool"):
        op.prepare_prefill_batch([PrefillSpec([inside], torch.tensor([160], dtype=torch.int32), 3, 0)])
    other = block([3], 2)
    for slot, fits in ((159, True), (160, False), (-1, False)):
        group = WorkerGroup(cache_structure=[[inside]], write_to=[other])
        args = group, {id(other): None}, torch.tensor([slot], dtype=torch.int32)
        if fits:
            op.prepare(*args)
        else:
            with pytest.raises(ValueError, match="outside the pool"):
                op.prepare(*args)
    decode = SharedDecodeAttentionBuffers(op, 2, 2, max_pages=8)
    with pytest.raises(ValueError, match="outside the pool"):
        decode.plan([0], [0], [0], [[10]], [1], [3], [3], [], [], [])
    chunks = SharedPrefillAttentionBuffers(op, 2, 2, 16, max_pages=8)
    with pytest.raises(ValueError, match="outside the pool"):
        chunks.plan([PrefillSpec([block([11], 4)], torch.tensor([0], dtype=torch.int32), 3, 0)])


def pool_struct(**more):
    fields = dict(k_codes_dev=FAKE, v_codes_dev=FAKE, k_scales_dev=FAKE, v_scales_dev=FAKE, code_type=0, num_pages=8)
    return native.VaQuantPool(**{**fields, **more})


@pytest.mark.parametrize("pool,shape", [
    (pool_struct(code_type=7), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(k_codes_dev=None), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(v_scales_dev=None), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(v_codes_dev=FAKE + 8), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(num_pages=-1), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(num_pages=1 << 28), native.make_shape(4, 2, 64, 16, BF16)),
    (pool_struct(), native.make_shape(4, 0, 64, 16, BF16)),
    (pool_struct(), native.make_shape(4, 2, 48, 16, BF16)),
    (pool_struct(), native.make_shape(4, 2, 64, 0, BF16)),
])
def test_entries_refuse_what_is_no_pool(pool, shape):
    lib = native.lib
    blob = np.zeros(64, dtype=np.int32)
    blob[0] = 0x56415031
    blob[9] = 1  # a row
    for rc in (lib.va_store_kv_rope_q8(FAKE, FAKE, 128, 128, pool, FAKE, 1, None, 0, 1, shape, ROPE, None),
               lib.va_load_kv_q8(pool, FAKE, 1, FAKE, FAKE, 128, shape, None),
               lib.va_copy_shift_kv_q8(pool, 0, 0, 1, FAKE, FAKE, 1, 0, shape, None, None),
               lib.va_attention_q8(FAKE, 256, pool, FAKE, blob.ctypes.data, FAKE, FAKE, FAKE, 0, FAKE, None, 0, None, 0, shape, ROPE, None),
               lib.va_attention_read_back_q8(FAKE, 256, pool, FAKE, 16, FAKE, blob.ctypes.data, FAKE, FAKE, FAKE, 0, FAKE, None, 0, None, 0,
                                             FAKE, 1 << 30, shape, ROPE, None)):
        assert rc < 0, native.lib.va_last_error()


def test_entries_refuse_what_does_not_fit_a_plan():
    op, pool = make()
    op._reads_back = lambda pairs, pages: True
    step = op.prepare_prefill_batch([PrefillSpec([block([1, 2], 20)], torch.tensor([48], dtype=torch.int32), 9, 0)])
    back = step.launch.readback
    struct, shape = pool_struct(num_pages=40), op._shape

    def call(plan=back.launch.header, n_slots=16, scratch=FAKE, nbytes=1 << 30, shape=shape, q=FAKE, slots=FAKE):
        return native.lib.va_attention_read_back_q8(q, 512, struct, slots, n_slots, FAKE, plan.ctypes.data, FAKE, FAKE, FAKE, 0, FAKE, None, 0,
                                                    None, 0, scratch, nbytes, shape, ROPE, None)

    need = native.lib.va_read_back_bytes(16, 9, shape)
    wrong = back.launch.header.copy()
    wrong[0] = 0
    assert call(plan=wrong) < 0 and call(n_slots=-1) < 0 and call(q=None) < 0 and call(slots=None) < 0
    assert call(nbytes=need - 1) == native.VA_ERR_CAPACITY and call(scratch=FAKE + 16) == native.VA_ERR_CAPACITY
    assert call(scratch=None) == native.VA_ERR_CAPACITY
    assert call(shape=native.make_shape(8, 2, 64, 16, F32)) < 0
    assert native.lib.va_read_back_bytes(-1, 9, shape) < 0 and native.lib.va_read_back_bytes(16, -1, shape) < 0
    # a plan with items of many rows is for rows that were read back
    if back.launch.counts.n_wide_items:
        assert native.lib.va_attention_q8(FAKE, 512, struct, FAKE, back.launch.header.ctypes.data, FAKE, FAKE, FAKE, 0, FAKE, None, 0,
                                          FAKE, 1 << 30, shape, ROPE, None) < 0


# ---------------------------------------------------------------------------
# plans of chunks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_read_back_plan_names_every_visible_token_once(dtype):
    op, pool = make(dtype=dtype, pages=60)
    op._reads_back = lambda pairs, pages: True
    shared, mine = block([7, 3, 50], 41), block([12], 5)
    specs = [PrefillSpec([shared, mine], torch.tensor([16 * 20, 16 * 21], dtype=torch.int32), 14, 6),
             PrefillSpec([shared], torch.tensor([16 * 33], dtype=torch.int32), 2, 0)]
    launch = op.prepare_prefill_batch(specs).launch
    back = launch.readback
    pages = [3, 7, 12, 20, 21, 33, 50]
    held = {7: 16, 3: 16, 50: 9, 12: 5, 20: 16, 21: 4, 33: 2}
    want = [p * 16 + i if i < held[p] else -1 for p in pages for i in range(16)]
    assert back.slots.tolist() == want
    order = [pages.index(p) for p in (7, 3, 50, 12, 7, 3, 50, 20, 21, 33)]
    assert back.launch.kv_indices.tolist() == order
    assert back.first_row == 0 and back.scratch.numel() >= native.lib.va_read_back_bytes(len(want), 16, op._shape)
    assert back.launch.header is launch.header


def test_pages_that_nobody_sees_are_not_read_back():
    """Lists may name more pages than their tokens fill."""
    op, pool = make(pages=60)
    op._reads_back = lambda pairs, pages: True
    shared = block([7, 3, 50, 1], 32)
    spec = PrefillSpec([shared], torch.tensor([16 * 20, 16 * 2, 16 * 59], dtype=torch.int32), 14, 0)
    back = op.prepare_prefill_batch([spec]).launch.readback
    assert back.slots.tolist() == [*range(48, 64), *range(112, 128), *range(320, 334), -1, -1]  # pages 3, 7 and 20
    seen = back.launch.kv_indices.tolist()
    assert seen[:2] == [1, 0] and 2 in seen and all(0 <= i < 3 for i in seen)


@pytest.mark.parametrize("readers,tokens", [(64, 8192), (5, 300), (33, 70)])
def test_tiles_of_a_plan_over_codes_walk_apart(readers, tokens):
    """Every (row, token) pair once, and no item that another's workgroup would have to serve."""
    op, pool = make(heads=(16, 4, 256), pages=6000)
    shared = block(list(range(-(-tokens // 16))), tokens)
    own = [block([1000 + 2 * i], 1 + i % 15) for i in range(readers)]
    group = WorkerGroup(cache_structure=[[shared, b] for b in own], write_to=own)
    slots = torch.tensor([(1000 + 2 * i) * 16 + 1 + i % 15 for i in range(readers)], dtype=torch.int32)
    meta = op.prepare(group, {id(b): None for b in own}, slots)
    pages, row_of = meta.launch.kv_indices.tolist(), meta.sub_worker.tolist()
    _, items, links, qrefs, *_ = decode_plan(meta.launch.blob.numpy())
    seen = np.zeros((readers, 2), dtype=np.int64)
    for begin, n_links, n_q, _, _, _, partners in items[:, :7].tolist():
        assert partners == 0 and n_q <= 4
        for kv_begin, t0, t1, qref, _, flags in links[begin: begin + n_links, :6].tolist() if n_q else ():
            for i in range(n_q):
                row = row_of[qrefs[qref + i] if flags & 1 else qref + i]
                seen[row, int(pages[kv_begin] >= 1000)] += t1 - t0
    assert (seen[:, 0] == tokens).all() and seen[:, 1].tolist() == [b.num_tokens + 1 for b in own]


def test_a_mixed_plan_keeps_decodes_on_codes():
    op, pool = make(pages=60)
    op._reads_back = lambda pairs, pages: True
    prompt, own = block([7, 3, 50], 41), block([12], 5)
    group = WorkerGroup(cache_structure=[[prompt, own], [prompt]], write_to=[own, prompt])
    spec = PrefillSpec([prompt], torch.tensor([16 * 20], dtype=torch.int32), 14, 0)
    meta = op.prepare_mixed(group, {id(own): None, id(prompt): None}, torch.tensor([12 * 16 + 5, 50 * 16 + 9], dtype=torch.int32), [spec])
    back = meta.launch.readback
    assert back.first_row == 2 and meta.launch.header[9] == 2 and back.launch.header[9] == 14
    assert back.sub_worker.tolist() == [*range(14), *range(14)] and meta.sub_worker.tolist()[back.first_subrow:] == [*range(2, 16)] * 2
    assert not meta.launch.counts.n_wide_items


def test_which_chunks_are_read_back():
    op, _ = make(heads=(32, 8, 128))
    assert op._reads_back(300 * 20000, 20000 // 16) and not op._reads_back(16 * 20000, 20000 // 16)
    assert not op._reads_back(8 * 1_000_000, 1_000_000 // 16)  # few rows over many tokens
    assert not op._reads_back(64 * 500, 500 // 16)
    for other in (make(dtype=F32)[0], make(kernel="generic")[0], make(heads=(6, 2, 64))[0]):
        other._reads_back = lambda pairs, pages: True
        assert other.prepare_prefill_batch([PrefillSpec([], torch.tensor([0], dtype=torch.int32), 9, 0)]).launch.readback is None
    op, _ = make()
    op._reads_back = lambda pairs, pages: True
    op.prepare_workspace([SharedPrefillAttentionBuffers(op, 2, 2, 16, max_pages=8)])
    assert op.prepare_prefill_batch([PrefillSpec([], torch.tensor([0], dtype=torch.int32), 9, 0)]).launch.readback is None
