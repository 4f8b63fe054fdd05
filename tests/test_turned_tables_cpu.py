"""Stored keys are turned by tables of unit length only: with an attention factor every turn would make them longer."""

import pytest
import torch

from async_llm_amd import native
from async_llm_amd.kvcache import MHAKVCache, QuantizedKVCache
from async_llm_amd.shared_cache import BlockKVOps, CacheEviction, QuantizedCacheAttention, SharedCacheAttention

CPU = torch.device("cpu")


class Pages:
    def __init__(self):
        self.taken = 0

    def alloc_pages(self, n):
        got = torch.arange(self.taken, self.taken + n, dtype=torch.int32) * 16
        self.taken += n
        return got


def made(factor, codes=None, mrope=None, rotary=64):
    table = torch.cat([torch.ones(8, 32), torch.zeros(8, 32)], dim=1) * factor
    more = dict(rotary_dim=rotary, **(dict(mrope_section=mrope, rope_base=1e4) if mrope else {}))
    if codes is None:
        pool = MHAKVCache(2, 1, 64, 8, 16, torch.bfloat16, CPU)
        return SharedCacheAttention(pool, table, 4, 2, 64, 16, torch.bfloat16, CPU, **more)
    pool = QuantizedKVCache(2, 1, 64, 8, 16, torch.bfloat16, CPU, codes)
    return QuantizedCacheAttention(pool, table, 4, 2, 64, 16, torch.bfloat16, CPU, **more)


def two_blocks(ops, left, right):
    out = []
    for n in (left, right):
        b = ops.create_block()
        if n:
            b.grow_pages(ops.page_allocator.alloc_pages(b.pages_needed(n)), n)
        b.token_ids = list(range(n))
        out.append(b)
    return out


@pytest.mark.parametrize("codes", [None, torch.int8])
@pytest.mark.parametrize("factor", [1.1386, 0.9, 0.0, float("nan")])
def test_merges_and_appends_are_refused_before_anything_is_taken(factor, codes):
    op = made(factor, codes)
    ops = BlockKVOps(op.kv_cache, op, Pages())
    left, right = two_blocks(ops, 20, 5)
    taken = ops.page_allocator.taken
    for call in (ops.merge_blocks, ops.append_block):
        with pytest.raises(ValueError, match="unit"):
            call(left, right)
    with pytest.raises(ValueError, match="unit"):
        ops._shift_keys_(block=left, start=3, num_tokens=4, position_shift=2)
    assert ops.page_allocator.taken == taken
    assert (left.num_tokens, left.num_pages, left.token_ids) == (20, 2, list(range(20)))
    assert (right.num_tokens, right.num_pages) == (5, 1)


@pytest.mark.parametrize("factor, mrope, rotary", [(1.0, None, 64), (1.2, (8, 12, 12), 64), (1.2, None, 0)])
def test_tables_of_unit_length_and_no_tables_are_not(factor, mrope, rotary):
    """(The copy itself wants a GPU.)"""
    op = made(factor, mrope=mrope, rotary=rotary)
    ops = BlockKVOps(op.kv_cache, op, Pages())
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        ops.merge_blocks(*two_blocks(ops, 20, 5))


def test_what_is_not_turned_is_copied_over_any_table():
    op = made(1.2)
    ops = BlockKVOps(op.kv_cache, op, Pages())
    for left, right in ((20, 0), (0, 5)):
        with pytest.raises(native.ViewAttnError, match="GPU only"):
            ops.merge_blocks(*two_blocks(ops, left, right))


def test_copies_over_codes(monkeypatch):
    called = []
    monkeypatch.setattr(native, "require_device", lambda t, name: None)
    monkeypatch.setattr(native, "current_stream_ptr", lambda device: 0)
    monkeypatch.setattr(native, "call_on", lambda device, function, *a: called.append(function))
    a, b = torch.arange(3), torch.arange(20, 23)
    op = made(1.2, torch.int8)
    with pytest.raises(ValueError, match="unit"):
        op.copy_shifted(a, b, 4)
    assert not called
    op.copy_shifted(a, b)
    made(1.0, torch.int8).copy_shifted(a, b, 4)
    assert len(called) == 2


def test_moves_with_shifts(monkeypatch):
    monkeypatch.setattr(native, "require_device", lambda t, name: None)
    monkeypatch.setattr(native, "call_on", lambda *a: pytest.fail("called"))
    a, b = torch.arange(3), torch.arange(20, 23)
    with pytest.raises(ValueError, match="unit"):
        CacheEviction(made(1.2)).move(a, b, a)


def test_a_table_that_is_filled_after_the_op_was_made():
    op = made(0.0)
    with pytest.raises(ValueError, match="unit"):
        op._check_turns()
    op.cos_sin_cache[:, :32] = 1.0
    op._check_turns()
