"""Rows of the 8-bit pool on the GPU: written, read back and moved, against their definition in 64 bits."""

from types import SimpleNamespace

import pytest
import torch

from tests import quant_util as Q

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def batch(slots, positions, three=None):
    return SimpleNamespace(attn_metadata=None, positions=positions, mrope_positions=three, out_loc=slots)


def raw(pool):
    return pool._codes.view(torch.uint8).cpu().clone(), pool._scales.cpu().clone()


def check_store(op, pool, k, v, where, slots, before, layer=0):
    """The rows of ``slots`` (int64, CPU; -1: skipped) are quantised, every other row is as it was."""
    Hkv, D, P = pool.num_kv_heads, pool.head_dim, pool.page_size
    live = slots >= 0
    page, place = slots[live] // P, slots[live] % P
    codes, scales = raw(pool)
    n = int(live.sum())
    k, v = k.cpu()[live].reshape(n, Hkv, D), v.cpu()[live].reshape(n, Hkv, D)
    where = where.cpu()[..., live]
    for which, x, x64, off in ((0, Q.rotated(op, k, where, double=False), Q.rotated(op, k, where), Q.turn_error(k)),
                               (1, v.float(), v.double(), torch.zeros(v.shape, dtype=torch.float64))):
        c, s = codes[which, layer][page, :, place].view(pool.code_dtype), scales[which, layer][page, :, place]
        finite = torch.isfinite(x64).all(-1)
        Q.assert_quantises(c[finite], s[finite], x64[finite], off[finite], pool.code_dtype)
        assert (s[~finite] == 255).all() and (c.view(torch.uint8)[~finite] == 0).all()
        if op.mrope_section is None or which == 1:  # the same 32-bit arithmetic: code for code
            ec, es = Q.quantised32(x, pool.code_dtype)
            assert torch.equal(s, es) and torch.equal(c.view(torch.uint8)[finite], ec.view(torch.uint8)[finite])
        before[0][which, layer][page, :, place] = c.view(torch.uint8)
        before[1][which, layer][page, :, place] = s
    assert torch.equal(codes, before[0]) and torch.equal(scales, before[1])


STORES = [
    # rows, heads, page, dtype, codes, rotary, mrope
    (1, (4, 2, 256), 16, torch.bfloat16, E4M3, None, None),
    (1, (1, 1, 16), 1, torch.float32, INT8, None, None),
    (77, (8, 4, 128), 16, torch.float16, INT8, None, None),
    (130, (4, 4, 64), 8, torch.bfloat16, INT8, 32, None),
    (65, (6, 3, 32), 7, torch.float32, E4M3, None, None),
    (41, (4, 2, 128), 16, torch.bfloat16, E4M3, 0, None),
    (50, (4, 2, 256), 32, torch.bfloat16, E4M3, 128, (24, 20, 20)),
    (50, (4, 2, 64), 16, torch.float16, INT8, 64, (12, 10, 10)),
    (33, (4, 2, 64), 16, torch.float16, E4M3, 18, None),  # no multiple of 16: element by element
    (33, (2, 2, 256), 5, torch.float32, INT8, 100, None),
]


@pytest.mark.parametrize("rows,heads,page,dtype,codes,rotary,mrope", STORES)
def test_store(rows, heads, page, dtype, codes, rotary, mrope):
    pages = -(-rows // page) + 2
    op, pool, g = Q.make(DEV, heads, page, pages, dtype, codes, rotary, mrope, layers=2)
    width = heads[1] * heads[2]
    k = (torch.randn(rows, width, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    v = torch.randn(rows, width, generator=g).to(dtype)
    slots = torch.randperm(pages * page, generator=g)[:rows]
    slots[3::7] = -1
    where = torch.randint(0, 4000, (rows,), generator=g)
    three = torch.randint(0, 4000, (3, rows), generator=g) if mrope else None
    before = raw(pool)
    fused = torch.cat([k, v, torch.full((rows, 8), float("nan"), dtype=dtype)], dim=1).to(DEV)  # rows lie apart
    op.store_new_kv(fused[:, :width], fused[:, width: 2 * width], 1,
                    batch(slots.to(torch.int32).to(DEV), where.to(DEV), None if three is None else three.to(DEV)))
    check_store(op, pool, k, v, where if three is None else three, slots, before, layer=1)


@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_store_of_unusual_rows(codes):
    """Zeros, the smallest and the largest numbers, maxima on both sides of a scale's edge, infinities and NaN."""
    op, pool, g = Q.make(DEV, (2, 1, 64), 16, 4, torch.float32, codes, 0)
    x = torch.randn(24, 64, generator=g)
    x[0] = 0
    x[1] *= 1e-42
    x[2] *= 2.0**-130
    x[3] = torch.finfo(torch.float32).max
    x[4, 5] = float("inf")
    x[5, 6] = float("nan")
    x[6, 7] = float("-inf")
    top = Q.LARGEST[codes]
    for i, t in enumerate((top, top * (1 + 2.0**-23), top * (1 - 2.0**-24), top / 2, top / 2 * (1 + 2.0**-23))):
        x[8 + i] = x[8 + i].clamp(-1, 1) * (top / 4)
        x[8 + i, 9] = -t
    x[14] = torch.arange(64) * 0.5 - 16  # ties
    x[14, 0] = top / 2 + 1
    x[15] = torch.arange(64) * 2.0**-10  # e4m3's subnormal codes
    x[15, 0] = top
    slots = torch.randperm(64, generator=g)[:24]
    before = raw(pool)
    op.store_new_kv(x.to(DEV), x.flip(0).contiguous().to(DEV), 0, batch(slots.to(DEV), torch.zeros(24, dtype=torch.int64, device=DEV)))
    check_store(op, pool, x, x.flip(0), torch.zeros(24, dtype=torch.int64), slots, before)
    k, _ = pool.load_kv(slots.to(DEV), 0)
    assert torch.isnan(k[4:7]).all() and torch.isfinite(k[:4]).all() and (k[0] == 0).all()


def test_store_without_rotation_alignment_or_room():
    """``store_kv`` as it is, rows on odd addresses, slots past the pool and an empty batch."""
    op, pool, g = Q.make(DEV, (2, 2, 32), 4, 6, torch.bfloat16, E4M3, 0)
    flat = torch.randn(5 * 129 + 3, generator=g).to(torch.bfloat16).to(DEV)
    k = flat[1: 1 + 5 * 129].view(5, 129)[:, :64]
    v = flat[2: 2 + 5 * 129].view(5, 129)[:, 64:128]
    slots = torch.tensor([3, 24, -5, 23, 1 << 40])
    before = raw(pool)
    pool.store_kv(k, v, slots.to(DEV), 0)
    kept = torch.where((slots >= 0) & (slots < 24), slots, -1)
    check_store(op, pool, k.cpu(), v.cpu(), torch.zeros(5, dtype=torch.int64), kept, before)
    pool.store_kv(k[:0], v[:0], slots[:0].to(DEV), 0)


@pytest.mark.parametrize("rows,heads,page,dtype,codes", [
    (1, (1, 1, 16), 1, torch.float32, INT8), (300, (4, 2, 256), 16, torch.bfloat16, E4M3),
    (257, (4, 4, 128), 8, torch.float16, INT8), (99, (3, 3, 64), 5, torch.float32, E4M3),
    (64, (2, 2, 32), 32, torch.float16, E4M3)])
def test_load(rows, heads, page, dtype, codes):
    op, pool, g = Q.make(DEV, heads, page, -(-rows // page) + 1, dtype, codes, 0, layers=2)
    slots = torch.randint(0, rows, (rows,), generator=g)  # some of them twice
    slots[5::9] = -1
    slots[7::31] = pool.num_pages * page
    got = pool.load_kv(slots.to(DEV), 1)
    outside = (slots < 0) | (slots >= pool.num_pages * page)
    for which, x in enumerate(got):
        want = Q.rows64(pool, which, 1, torch.where(outside, 0, slots)).float().to(dtype)
        want[outside] = 0
        assert x.dtype == dtype and torch.equal(x.cpu(), want)
    # rows of the caller's, apart; what lies between them stays
    wide = torch.full((rows, heads[1] + 1, heads[2]), 7.0, dtype=dtype, device=DEV)
    other = wide.clone()
    pool.load_kv(slots.to(DEV), 1, out=(wide[:, :-1], other[:, :-1]))
    assert torch.equal(wide[:, :-1], got[0]) and torch.equal(other[:, :-1], got[1])
    assert (wide[:, -1] == 7).all() and (other[:, -1] == 7).all()


@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_read_back_is_stored_alike(codes, dtype):
    op, pool, g = Q.make(DEV, (2, 2, 128), 16, 12, dtype, codes, 0)
    here, there = torch.arange(96, device=DEV), torch.arange(96, 192, device=DEV)
    first = pool.load_kv(here, 0)
    pool.store_kv(first[0].view(96, -1), first[1].view(96, -1), there, 0)
    again = pool.load_kv(there, 0)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("n,heads,page,codes,rotary,mrope,shift,layers", [
    (1, (1, 1, 16), 1, E4M3, None, None, 5, 1), (100, (4, 2, 256), 16, E4M3, None, None, 77, 3),
    (61, (4, 4, 128), 8, INT8, None, None, 1, 2), (50, (2, 2, 64), 5, INT8, 32, None, 300, 2),
    (47, (4, 2, 256), 16, E4M3, 128, (24, 20, 20), 1234567, 2), (40, (2, 2, 64), 16, E4M3, 18, None, 9, 2),
    (33, (4, 2, 128), 16, INT8, None, None, 0, 2), (33, (4, 2, 128), 16, E4M3, 0, None, 12, 2),
    (29, (3, 3, 32), 4, INT8, None, None, -40, 1), (25, (2, 2, 128), 16, E4M3, None, None, 10**7, 1)])
def test_copy_shifted(n, heads, page, codes, rotary, mrope, shift, layers):
    pages = 2 * (-(-n // page) + 1)
    op, pool, g = Q.make(DEV, heads, page, pages, torch.bfloat16, codes, rotary, mrope, layers=layers)
    perm = torch.randperm(pages * page, generator=g)
    source, target = perm[:n].clone(), perm[n: 2 * n].clone()
    if n > 20:
        source[7], target[11] = -1, pages * page  # skipped
    before = raw(pool)
    op.copy_shifted(source.to(DEV), target.to(DEV), shift)
    live = (source >= 0) & (target < pages * page)
    codes_now, scales_now = raw(pool)
    fp, fs, tp, ts = source[live] // page, source[live] % page, target[live] // page, target[live] % page
    for layer in range(layers):
        c0, s0 = before[0][:, layer], before[1][:, layer]
        k = Q.values64(c0[0][fp, :, fs].view(pool.code_dtype), s0[0][fp, :, fs])
        where = torch.full((int(live.sum()),), shift)
        c, s = codes_now[0, layer][tp, :, ts], scales_now[0, layer][tp, :, ts]
        if shift == 0 or op.rotary_dim == 0:
            assert torch.equal(c, c0[0][fp, :, fs]) and torch.equal(s, s0[0][fp, :, fs])
        else:
            Q.assert_quantises(c.view(pool.code_dtype), s, Q.rotated(op, k, where), Q.turn_error(k), pool.code_dtype)
            if mrope is None:
                ec, es = Q.quantised32(Q.rotated(op, k.float(), where, double=False), pool.code_dtype)
                assert torch.equal(c, ec.view(torch.uint8)) and torch.equal(s, es)
        before[0][0, layer][tp, :, ts], before[1][0, layer][tp, :, ts] = c, s
        before[0][1, layer][tp, :, ts] = c0[1][fp, :, fs]
        before[1][1, layer][tp, :, ts] = s0[1][fp, :, fs]
    assert torch.equal(codes_now, before[0]) and torch.equal(scales_now, before[1])


@pytest.mark.parametrize("rotary", [None, 18])
def test_keys_shift_in_place(rotary):
    op, pool, g = Q.make(DEV, (4, 2, 64), 16, 6, torch.bfloat16, E4M3, rotary, layers=2)
    slots = torch.randperm(96, generator=g)[:50]
    want = torch.randperm(96, generator=g)
    spare = torch.tensor([s for s in want.tolist() if s not in set(slots.tolist())])[:46]
    before = raw(pool)
    op.copy_shifted(slots.to(DEV), slots.to(DEV), 31)
    codes, scales = raw(pool)
    assert torch.equal(codes[1], before[0][1]) and torch.equal(scales[1], before[1][1])
    where = torch.full((50,), 31)
    for layer in range(2):
        k = Q.values64(before[0][0, layer][slots // 16, :, slots % 16].view(E4M3), before[1][0, layer][slots // 16, :, slots % 16])
        ec, es = Q.quantised32(Q.rotated(op, k.float(), where, double=False), E4M3)
        assert torch.equal(codes[0, layer][slots // 16, :, slots % 16], ec.view(torch.uint8))
        assert torch.equal(scales[0, layer][slots // 16, :, slots % 16], es)
        assert torch.equal(codes[0, layer][spare // 16, :, spare % 16], before[0][0, layer][spare // 16, :, spare % 16])
