"""Chunks that are read back, where rows of one request, or of one head, are far larger than another's: float16 cannot hold
both, and the step has to answer as the kernel over codes does."""

import pytest
import torch

from tests import quant_util as Q

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16 = torch.bfloat16, torch.float16


def chunk_step(codes, heads=(8, 2, 64), page=16, dtype=BF16, new=(33, 20), context=(120, 90), seed=0):
    """Two requests with a context block each and nothing in common: the op, its step and where the rows of each lie."""
    op, pool, g = Q.make(DEV, heads, page, 80, dtype, codes, seed=seed)
    op._reads_back = lambda pairs, pages: True
    pages = Q.Pages(80, page)
    blocks = [pages.block(DEV, n) for n in context]
    step = Q.prefill_step(op, [([b], pages.block(DEV, 5, room=n), n) for b, n in zip(blocks, new)])
    assert step.meta.launch.readback is not None
    return op, pool, g, step, [Q.slots_of(b) for b in blocks]


def check_as_codes(op, step, q, out, lse, rows=None):
    """Within the bounds of the kernel over codes, for the requests ``rows`` (all)."""
    first = 0
    for r, (segments, n) in enumerate(zip(step.segments, step.new)):
        if rows is None or r in rows:
            part = slice(first, first + n)
            expected = Q.attention64(op, q[part].cpu().view(n, op.num_qo_heads, op.head_dim), segments)
            Q.assert_attends(out[part], lse[part], expected, op.dtype, sum(len(s[0]) for s in segments))
        first += n


@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("which,size", [(0, 1e5), (0, 1e6), (0, 1e12), (0, 1e30), (1, 1e6), (1, 1e12), (1, 1e30)])
@pytest.mark.parametrize("everywhere", [False, True])
def test_large_rows_of_one_request_leave_the_other_as_it_is(codes, which, size, everywhere):
    """One row of the second request (in one kv head, or ``everywhere`` in its context) is ``size`` times as large."""
    op, pool, g, step, contexts = chunk_step(codes)
    slots = contexts[1] if everywhere else contexts[1][40:41]
    x = torch.randn(len(slots), 2, 64, generator=g)
    x[:, 1] *= size
    Q.write(pool, which, 0, slots, *Q.quantised32(x, codes))
    q = torch.randn(53, 512, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check_as_codes(op, step, q, out, lse)


@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_small_values_beside_large_ones_of_another_head(codes):
    op, pool, g, step, contexts = chunk_step(codes)
    for segments in step.segments:
        for slots, _, _ in segments:
            x = torch.randn(len(slots), 2, 64, generator=g)
            x[:, 0] *= 2.0**-50
            Q.write(pool, 1, 0, slots, *Q.quantised32(x, codes))
    q = torch.randn(53, 512, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check_as_codes(op, step, q, out, lse)
    # (the bound counts a value's magnitude by its own row of results: the small head is held to 2^-50 as well)
    assert out[:, :256].abs().max() > 0


@pytest.mark.parametrize("size", [3e4, 1e30])
def test_large_queries_of_one_row(size):
    """A query of the first request is far larger than float16 holds beside these keys; its scores are those of the codes."""
    op, pool, g, step, contexts = chunk_step(E4M3)
    q = torch.randn(53, 512, generator=g)
    q[7] *= size
    q = q.to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    keep = torch.tensor([i for i in range(53) if i != 7])
    expected = [Q.attention64(op, q[a: a + n].cpu().view(n, 8, 64), s) for a, n, s in zip((0, 33), step.new, step.segments)]
    o, l, off, weight, lost = (torch.cat(x) for x in zip(*expected))
    Q.assert_attends(out[keep], lse[keep], (o[keep], l[keep], off[keep], weight[keep], lost[keep]), BF16, 200)
    # scores of up to 1e31: a softmax that is one row's value, where no second score is near the largest
    top = torch.stack([torch.isfinite(out[7]).all(), torch.isfinite(lse[7]).all()])
    assert top.all()
    if size == 3e4:
        Q.assert_attends(out[7:8], lse[7:8], (o[7:8], l[7:8], off[7:8], weight[7:8], lost[7:8]), BF16, 200)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_stays_alone(value):
    op, pool, g, step, contexts = chunk_step(E4M3)
    q = torch.randn(53, 512, generator=g)
    q[7, 64:128] = value  # the second head of a row
    q = q.to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    bad = torch.isnan(out.view(53, 8, 64))
    want = torch.zeros_like(bad)
    want[7, 1] = True
    assert torch.equal(bad, want)
    clean = q.clone()
    clean[7, 64:128] = 0
    rest, _ = op.attend(clean, 0, step.meta, return_lse=True)
    o, l, off, weight, lost = (torch.cat(x) for x in zip(*[Q.attention64(op, clean[a: a + n].cpu().view(n, 8, 64), s, half=True)
                                                            for a, n, s in zip((0, 33), step.new, step.segments)]))
    largest = max(Q.rows64(pool, 1, 0, slots).abs().max().item() for segments in step.segments for slots, _, _ in segments)
    got = torch.where(want.view(53, 512), rest, out)
    Q.assert_attends(got, None, (o, l, off, weight, lost), BF16, 200, torch.full((53,), largest, dtype=torch.float64))


def test_a_recorded_step_follows_its_rows():
    """One graph, replayed over rows that float16 holds and over others in turn; a mixed step's decodes stay as they are."""
    op, pool, g, step, contexts = chunk_step(E4M3)
    q = torch.randn(53, 512, generator=g).to(BF16).to(DEV)
    word = step.meta.launch.readback.scratch[:4].view(torch.int32)
    op.attend(q, 0, step.meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = op.attend(q, 0, step.meta, return_lse=True)
    for size in (1.0, 1e12, 1.0, 1e6, 1e25, 1.0):
        x = torch.randn(2, len(contexts[1]), 2, 64, generator=g)
        x[0, 3] *= size
        for which in range(2):
            Q.write(pool, which, 0, contexts[1], *Q.quantised32(x[which], E4M3))
        graph.replay()
        torch.cuda.synchronize()
        assert word.item() == (size > 1)
        if size > 1:
            check_as_codes(op, step, q, out, lse)
        eager, eager_lse = op.attend(q, 0, step.meta, return_lse=True)
        assert torch.equal(eager, out) and torch.equal(eager_lse, lse)


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("size", [1.0, 1e9])
def test_a_mixed_step_over_a_large_row(page, size):
    op, pool, g = Q.make(DEV, (8, 2, 128), page, 800 // page * 8, BF16, INT8)
    op._reads_back = lambda pairs, pages: True
    pages = Q.Pages(800 // page * 8, page)
    prompt, own = pages.block(DEV, 300), pages.block(DEV, 40, room=1)
    x = torch.randn(1, 2, 128, generator=g) * size
    Q.write(pool, 0, 0, Q.slots_of(prompt)[7:8], *Q.quantised32(x, INT8))
    decode = Q.decode_step(op, pages, [[prompt, own]], [own], g)
    prefill = Q.prefill_step(op, [([prompt], pages.block(DEV, 5, room=70), 70), ([], pages.block(DEV, 9, room=30), 30)])
    meta = op.prepare_mixed(decode.group, decode.pending, decode.slots, prefill.specs)
    q = torch.randn(101, 1024, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, meta, return_lse=True)
    assert meta.launch.readback.scratch[:4].view(torch.int32).item() == (size > 1)
    first = 0
    for segments, n in zip(decode.segments + prefill.segments, [1] + prefill.new):
        half = first > 0 and size == 1
        expected = Q.attention64(op, q[first: first + n].cpu().view(n, 8, 128), segments, half=half)
        largest = max(Q.rows64(pool, 1, 0, s[0]).abs().max().item() for s in segments)
        Q.assert_attends(out[first: first + n], lse[first: first + n], expected, BF16, 500, torch.full((n,), largest * half, dtype=torch.float64))
        first += n


def test_rows_of_zeros_are_no_small_values():
    op, pool, g, step, contexts = chunk_step(E4M3)
    for which in range(2):
        x = torch.randn(len(contexts[0]), 2, 64, generator=g) * 2.0**20
        x[::3] = 0
        x[1::3, :, ::2] = -0.0
        Q.write(pool, which, 0, contexts[0], *Q.quantised32(x, E4M3))
    for slots, _, _ in step.segments[1] + step.segments[0][1:]:
        Q.write(pool, 1, 0, slots, *Q.quantised32(-0.0 * torch.ones(len(slots), 2, 64), E4M3))
    q = (torch.randn(53, 512, generator=g) * 2.0**-20).to(BF16).to(DEV)
    op.attend(q, 0, step.meta)
    assert step.meta.launch.readback.scratch[:4].view(torch.int32).item() == 0
