"""Plans of chunks that are read back, and the launch over their codes that stands behind them, without a GPU."""

import numpy as np
import pytest
import torch

from async_llm_amd import native
from async_llm_amd.shared_cache import PrefillSpec, WorkerGroup
from tests.test_native_abi_cpu import decode_plan
from tests.test_quant_cpu import BF16, F16, FAKE, ROPE, block, make, pool_struct


def planned(specs_of, heads=(8, 2, 64), pages=4000, page=16, dtype=BF16):
    op, pool = make(heads=heads, pages=pages, page=page, dtype=dtype)
    op._reads_back = lambda pairs, pages: True
    return op, op.prepare_prefill_batch(specs_of(page)).launch.readback


def chunks(new, context):
    """Requests of ``new`` rows over a shared context and blocks of their own, on pages in order."""
    def specs(page):
        held = -(-context // page)
        shared = block(list(range(held)), context, page) if context else None
        out, at = [], held
        for i, n in enumerate(new):
            k = -(-(n + i) // page)
            out.append(PrefillSpec([shared] if shared else [], torch.tensor([p * page for p in range(at, at + k)], dtype=torch.int32), n, i))
            at += k
        return out
    return specs


@pytest.mark.parametrize("heads", [(8, 2, 64), (16, 4, 256), (4, 4, 128), (16, 1, 128), (64, 32, 64)])
@pytest.mark.parametrize("new,context", [([1], 0), ([33], 100), ([1, 2, 3, 4], 9000), ([700, 1, 64], 3000), ([2000], 1)])
def test_the_launch_over_codes_needs_no_merge(heads, new, context):
    """Every (row, token) pair once, in the item that writes the row's result, from the pool's own pages."""
    op, back = planned(chunks(new, context), heads)
    plan = back.codes
    assert not plan.counts.n_partials and not plan.counts.n_wide_items and not plan.header[16]  # (no empty rows)
    _, items, links, qrefs, *_ = decode_plan(plan.blob.numpy())
    pages, row_of = plan.kv_indices.tolist(), back.sub_worker.tolist()
    seen = np.zeros(sum(new), dtype=np.int64)
    for begin, n_links, n_q, part, _, _, partners in items[:, :7].tolist():
        assert not n_q or (part < 0 and partners == 0)
        for kv_begin, t0, t1, qref, causal, flags in links[begin: begin + n_links, :6].tolist() if n_q else ():
            for i in range(n_q):
                row = row_of[qrefs[qref + i] if flags & 1 else qref + i]
                seen[row] += max(0, min(t1, causal + i + 1) - t0)
    want, at = [], 0
    for i, n in enumerate(new):
        want += [context + i + j + 1 for j in range(n)]
    assert seen.tolist() == want
    assert pages[: -(-context // 16)] == list(range(-(-context // 16)))  # pages, not places in the scratch


def test_a_condition_takes_plans_that_one_launch_answers():
    op, back = planned(chunks([33], 100))
    struct, shape = pool_struct(num_pages=4000), op._shape

    def call(condition=FAKE, plan=back.codes.header, shape=shape, q=FAKE):
        return native.lib.va_attention_if_q8(condition, q, 512, struct, FAKE, plan.ctypes.data, FAKE, FAKE, FAKE, 0, FAKE, None, 0, shape,
                                             ROPE, None)

    assert call(condition=None) == native.VA_ERR_ARG and call(q=None) < 0
    shared, own = block([1, 2], 20), [block([5 + i], 3) for i in range(2)]
    many = block(list(range(100, 1100)), 16000)
    step = op.prepare(WorkerGroup(cache_structure=[[many, shared, b] for b in own], write_to=own), {id(b): None for b in own},
                      torch.tensor([5 * 16 + 3, 6 * 16 + 3], dtype=torch.int32))
    assert step.launch.counts.n_partials
    assert call(plan=step.launch.header) == native.VA_ERR_ARG and b"partial states" in native.lib.va_last_error()
    assert call(plan=back.launch.header) < 0 or not back.launch.counts.n_wide_items


def test_float16_activations_are_not_read_back():
    """Whatever the work: float16 operands would cost them as much as the rounding of the result."""
    for dtype in (BF16, F16):
        op, _ = make(heads=(32, 8, 128), dtype=dtype)
        assert op._reads_back(300 * 20000, 20000 // 16) == (dtype == BF16)


def test_only_one_value_sets_the_tiles_of_a_plan_apart():
    """Any other negative number of rows asks for no wide tiles and nothing else."""
    plans = {}
    for rows in (-1, -2, -3, -(2**31) + 1, native.VA_TILES_APART):
        shape = native.make_shape(16, 4, 256, 16, BF16)
        shared = np.arange(512, dtype=np.int32)
        tables = [np.arange(65, dtype=np.int32), np.arange(65, dtype=np.int32) * 512, np.tile(shared, 64), np.full(64, 8192, dtype=np.int32),
                  np.zeros(64, dtype=np.int32), np.full(64, -1, dtype=np.int32)]
        row = np.arange(64, dtype=np.int64)
        subs = native.VaSubRequests(64, 64, 64, *(t.ctypes.data for t in tables), row.ctypes.data)
        params, counts = native.VaPlanParams(native.VA_KERNEL_MFMA, 0, 0, 0, rows), native.VaPlanCounts()
        native.check(native.lib.va_plan_count(subs, shape, params, counts))
        blob = np.zeros(counts.plan_words, dtype=np.int32)
        native.check(native.lib.va_plan_build(subs, shape, params, blob.ctypes.data, blob.size, counts))
        plans[rows] = blob.tobytes()
    assert plans[-1] == plans[-2] == plans[-3] == plans[-(2**31) + 1] != plans[native.VA_TILES_APART]
    assert make()[0].plan_params.wide_tile == native.VA_TILES_APART
