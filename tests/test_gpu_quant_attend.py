"""View attention over the 8-bit pool on the GPU, against its definition in 64 bits."""

from types import SimpleNamespace

import pytest
import torch

from tests import quant_util as Q

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(op, step, q, first, rows, out, lse, layer=0):
    Hq, D = op.num_qo_heads, op.head_dim
    parts = []
    back = step.meta.launch.readback  # rows from there on ran over float16
    half = torch.zeros(out.shape[0], dtype=torch.float64)
    largest = max([Q.rows64(op.kv_cache, 1, layer, s[0]).abs().max().item() for segments in step.segments for s in segments if len(s[0])])
    for segments, at, n in zip(step.segments, first, rows):
        in_half = back is not None and at >= back.first_row
        parts.append(Q.attention64(op, q[at: at + n].cpu().view(n, Hq, D), segments, layer, in_half))
        if in_half:
            half[at: at + n] = largest
    expected = tuple(torch.cat(x) for x in zip(*parts))
    tokens = max(sum(len(s[0]) for s in segments) for segments in step.segments)
    Q.assert_attends(out, lse, expected, op.dtype, tokens, half)


DECODES = [
    # heads, page, dtype, codes, rotary, mrope, shared, private lengths per request
    ((4, 1, 256), 16, BF16, E4M3, None, None, 0, [[1]]),
    ((4, 1, 256), 16, BF16, E4M3, None, None, 100, [[15], [16, 17], [33]]),
    ((16, 4, 256), 16, F16, INT8, None, None, 515, [[700, 3], [64], [129, 1, 40]]),
    ((8, 2, 128), 16, F32, INT8, None, None, 200, [[300], [77]]),
    ((32, 8, 128), 16, BF16, INT8, None, None, 1000, [[2000], [31, 64], [5], [650], [1, 1, 1]]),
    ((8, 8, 64), 32, F16, E4M3, 32, None, 70, [[200], [95]]),
    ((16, 1, 64), 8, BF16, E4M3, None, None, 50, [[300, 20], [9]]),
    ((6, 2, 128), 16, BF16, E4M3, None, None, 64, [[100], [1]]),  # three q heads a kv head
    ((10, 2, 32), 16, F16, INT8, None, None, 64, [[100], [1]]),
    ((2, 1, 16), 4, F32, E4M3, None, None, 10, [[30], [1]]),
    ((8, 2, 128), 1, BF16, E4M3, None, None, 90, [[120], [1]]),
    ((8, 2, 128), 6, BF16, E4M3, None, None, 90, [[120], [1]]),  # pages that no power of two is
    ((16, 4, 256), 16, BF16, E4M3, 128, (24, 20, 20), 130, [[400, 50], [77]]),
    ((8, 4, 64), 16, F32, E4M3, 18, None, 40, [[50]]),
]


@pytest.mark.parametrize("heads,page,dtype,codes,rotary,mrope,shared,private", DECODES)
def test_decode(heads, page, dtype, codes, rotary, mrope, shared, private):
    total = shared + sum(map(sum, private)) + (3 + sum(map(len, private))) * (page + 1)
    num_pages = -(-total // page) + 8
    op, pool, g = Q.make(DEV, heads, page, num_pages, dtype, codes, rotary, mrope)
    pages = Q.Pages(num_pages, page)
    span = (lambda n: n - n // 3) if mrope else (lambda n: None)
    common = [pages.block(DEV, shared, span=span(shared))] if shared else []
    views = [common + [pages.block(DEV, n, room=1, span=span(n)) for n in lengths] for lengths in private]
    step = Q.decode_step(op, pages, views, [v[-1] for v in views], g)
    q = torch.randn(len(views), heads[0] * heads[2], generator=g).to(dtype).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    n = len(views)
    check(op, step, q, range(n), [1] * n, out, lse)
    assert torch.equal(op.attend(q, 0, step.meta), out)  # the order of sums is fixed


def test_writers_outside_their_view_and_empty_blocks():
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 40, BF16, E4M3, seed=3)
    pages = Q.Pages(40, 16)
    a, b, c, empty = pages.block(DEV, 50), pages.block(DEV, 33, room=1), pages.block(DEV, 16, room=1), pages.block(DEV, 0, room=1)
    other = pages.block(DEV, 20, room=1)
    step = Q.decode_step(op, pages, [[a, b], [a, empty], [a, b], [a]], [b, empty, c, other], g)
    q = torch.randn(4, 8 * 128, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check(op, step, q, range(4), [1] * 4, out, lse)


PREFILLS = [
    # heads, page, dtype, codes, mrope, context lengths, (held, new) per request
    ((4, 1, 256), 16, BF16, E4M3, None, [], [(0, 1)]),
    ((16, 4, 256), 16, BF16, E4M3, None, [100], [(5, 37), (0, 3), (16, 64)]),
    ((32, 8, 128), 16, F16, INT8, None, [300, 17], [(33, 70), (1, 129)]),
    ((8, 2, 128), 16, F32, E4M3, None, [90], [(10, 21)]),
    ((6, 2, 64), 8, BF16, INT8, None, [50], [(3, 11)]),
    ((8, 2, 64), 1, F16, E4M3, None, [50], [(3, 41)]),
    ((16, 4, 256), 16, BF16, E4M3, (24, 20, 20), [200], [(40, 45), (0, 7)]),
    ((16, 4, 256), 32, F16, INT8, None, [777, 40], [(90, 301), (0, 33)]),
    ((32, 8, 128), 64, BF16, E4M3, None, [400], [(0, 200), (77, 1), (100, 65)]),
    ((8, 8, 128), 16, F16, E4M3, None, [100], [(7, 290)]),
    ((16, 1, 64), 16, BF16, INT8, None, [300], [(20, 100)]),
    ((64, 16, 64), 16, F16, E4M3, (12, 10, 10), [120], [(3, 140)]),
]


@pytest.mark.parametrize("heads,page,dtype,codes,mrope,context,requests,back",
                         [(*p, back) for p in PREFILLS for back in (False, True)
                          if not back or (p[2] != F32 and p[0][0] // p[0][1] != 3)])  # (no matrix-core kernel for these)
def test_prefill(heads, page, dtype, codes, mrope, context, requests, back, monkeypatch):
    num_pages = -(-(sum(context) + sum(h + n for h, n in requests)) // page) + 12
    op, pool, g = Q.make(DEV, heads, page, num_pages, dtype, codes, min(heads[2], 128) if mrope else None, mrope)
    pages = Q.Pages(num_pages, page)
    blocks = [pages.block(DEV, n, span=n - n // 4 if mrope else None) for n in context]
    monkeypatch.setattr(op, "_reads_back", lambda pairs, pages: back)
    step = Q.prefill_step(op, [(blocks, pages.block(DEV, h, room=n), n) for h, n in requests], three=mrope is not None)
    assert (step.meta.launch.readback is not None) == back
    new = [n for _, n in requests]
    q = torch.randn(sum(new), heads[0] * heads[2], generator=g).to(dtype).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    check(op, step, q, [sum(new[:r]) for r in range(len(new))], new, out, lse)


def test_large_chunks_are_read_back_and_small_ones_are_not():
    op, pool, g = Q.make(DEV, (32, 8, 128), 16, 260, BF16, E4M3)
    pages = Q.Pages(260, 16)
    context = [pages.block(DEV, 3210)]
    for new, back in ((16, False), (300, True)):
        step = Q.prefill_step(op, [(context, pages.block(DEV, 5, room=new), new)])
        assert (step.meta.launch.readback is not None) == back
        q = torch.randn(new, 32 * 128, generator=g).to(BF16).to(DEV)
        out, lse = op.attend(q, 0, step.meta, return_lse=True)
        check(op, step, q, [0], [new], out, lse)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_chunks_over_a_wide_range(codes, page, back):
    """Keys and values far from one, and among them rows that are far smaller: float16 alone would lose them."""
    op, pool, g = Q.make(DEV, (8, 2, 64), page, 40, BF16, codes)
    pages = Q.Pages(40, page)
    op._reads_back = lambda pairs, pages: back
    for k_size, v_size, q_size in ((2.0**20, 2.0**-40, 2.0**-20), (2.0**-60, 2.0**50, 2.0**55), (2.0**10, 2.0**-100, 2.0**-9)):
        block, own = pages.block(DEV, 100), pages.block(DEV, 3, room=20)
        slots = torch.cat([Q.slots_of(block), Q.slots_of(own, 23)])
        spread = 2.0 ** -torch.randint(0, 12, (123, 1, 1), generator=g)
        k = torch.randn(123, 2, 64, generator=g) * k_size * spread
        v = torch.randn(123, 2, 64, generator=g) * v_size * spread
        for which, x in enumerate((k, v)):
            c, s = Q.quantised32(x, codes)
            Q.write(pool, which, 0, slots, c, s)
        step = Q.prefill_step(op, [([block], own, 20)])
        q = (torch.randn(20, 8 * 64, generator=g) * q_size).to(BF16).to(DEV)
        out, lse = op.attend(q, 0, step.meta, return_lse=True)
        assert (step.meta.launch.readback is not None) == back
        check(op, step, q, [0], [20], out, lse)
        pages = Q.Pages(40, page)


def test_queries_on_rows_apart_and_given_outputs():
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 30, F16, INT8)
    pages = Q.Pages(30, 16)
    views = [[pages.block(DEV, 90, room=1)], [pages.block(DEV, 40, room=1)]]
    step = Q.decode_step(op, pages, views, [v[-1] for v in views], g)
    wide = torch.full((2, 8 * 128 + 64), float("nan"), dtype=F16, device=DEV)
    wide[:, :1024] = torch.randn(2, 1024, generator=g).to(F16).to(DEV)
    plain, base = op.attend(wide[:, :1024].contiguous(), 0, step.meta, return_lse=True)
    out, lse = torch.empty(2, 1024, dtype=F16, device=DEV), torch.empty(2, 8, device=DEV)
    assert op.attend(wide[:, :1024], 0, step.meta, out=out, lse=lse) is out
    assert torch.equal(out, plain) and torch.equal(lse, base)
    _, lse2 = op.attend(wide[:, :1024], 0, step.meta, return_lse=True, lse_base2=True)
    assert torch.allclose(lse2 * 0.6931471805599453, base, rtol=2.0**-22, atol=0)
    odd = torch.cat([torch.zeros(1, dtype=F16, device=DEV), wide[:, :1024].reshape(-1)])[1:].view(2, 1024)  # 2 bytes past 16
    assert torch.equal(op.attend(odd, 0, step.meta), plain)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_row_that_is_not_finite_reaches_those_that_see_it(which, dtype):
    """A key or value row with scale 255 makes NaN of every request that sees it, and of no other."""
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 400, dtype, E4M3)
    pages = Q.Pages(400, 16)
    views = [[pages.block(DEV, 2500, room=1)], [pages.block(DEV, 100, room=1)], [pages.block(DEV, 2000, room=1)]]
    at = slots_row = Q.slots_of(views[0][0])[1234].item()
    codes, scales = (pool.k_codes, pool.v_codes)[which](0), (pool.k_scales, pool.v_scales)[which](0)
    codes.view(torch.uint8)[at // 16, 1, at % 16] = 0
    scales.view(torch.uint8)[slots_row // 16, 1, slots_row % 16] = 255
    # garbage behind the ends of blocks is never visible
    for view in views:
        for s in Q.slots_of(view[0], -(-view[0].num_tokens // 16) * 16)[view[0].num_tokens + 1:].tolist():
            scales.view(torch.uint8)[s // 16, :, s % 16] = 255
            codes.view(torch.uint8)[s // 16, :, s % 16] = 0x7F
    step = Q.decode_step(op, pages, views, [v[-1] for v in views], g)
    q = torch.randn(3, 1024, generator=g).to(dtype).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    out = out.view(3, 8, 128)
    assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1:]).all()
    assert torch.isnan(lse[0, 4:]).all() if which == 0 else torch.isfinite(lse).all()
    assert torch.isfinite(lse[0, :4]).all() and torch.isfinite(lse[1:]).all()


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("which", [0, 1])
def test_a_row_that_is_not_finite_in_a_chunk(which, back):
    """Rows of the chunk in front of it and other requests never see it; those behind it do, in its kv head."""
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 400, BF16, E4M3)
    op._reads_back = lambda pairs, pages: back
    pages = Q.Pages(400, 16)
    context = [pages.block(DEV, 1500)]
    own, other = pages.block(DEV, 7, room=90), pages.block(DEV, 0, room=33)
    step = Q.prefill_step(op, [(context, own, 90), (context, other, 33)])
    at = Q.slots_of(own, 97)[50].item()  # row 43 of the first chunk
    codes, scales = (pool.k_codes, pool.v_codes)[which](0), (pool.k_scales, pool.v_scales)[which](0)
    codes.view(torch.uint8)[at // 16, 1, at % 16] = 0
    scales.view(torch.uint8)[at // 16, 1, at % 16] = 255
    q = torch.randn(123, 1024, generator=g).to(BF16).to(DEV)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    out, seen = out.view(123, 8, 128), torch.zeros(123, 8, dtype=torch.bool, device=DEV)
    seen[43:90, 4:] = True
    assert torch.equal(torch.isnan(out), seen[..., None].expand(out.shape)) and not torch.isinf(out).any()
    assert torch.equal(torch.isnan(lse), seen if which == 0 or back else torch.zeros_like(seen))


def test_a_step_stores_and_attends():
    """``forward`` over two layers: the rows that a step writes are the ones it sees."""
    op, pool, g = Q.make(DEV, (8, 2, 128), 16, 40, BF16, E4M3, layers=2)
    pages = Q.Pages(40, 16)
    views = [[pages.block(DEV, 48, room=1)], [pages.block(DEV, 100, room=1)]]
    step = Q.decode_step(op, pages, views, [v[-1] for v in views], g)
    batch = SimpleNamespace(attn_metadata=step.meta, positions=step.positions, mrope_positions=None, out_loc=step.slots)
    for layer in range(2):
        q, k, v = (torch.randn(2, n, generator=g).to(BF16).to(DEV) for n in (1024, 256, 256))
        out = op.forward(q, k, v, layer, batch)
        both, lse = op.forward_with_lse(q, k, v, layer, batch)
        assert torch.equal(out, both)
        want, _ = Q.quantised32(Q.rotated(op, k.cpu().view(2, 2, 128), step.positions, double=False), E4M3)
        s = step.slots.cpu().long()
        assert torch.equal(pool.k_codes(layer).view(torch.uint8).cpu()[s // 16, :, s % 16], want.view(torch.uint8))
        check(op, step, q, range(2), [1, 1], out, lse, layer)
