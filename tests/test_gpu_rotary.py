"""Rotation of queries and keys against complex products in 64 bits, and the table of the same frequencies."""

import pytest
import torch

from async_llm_amd.rotary import RotaryEmbedding
from async_llm_amd.shared_cache import apply_rope_correction

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def turned(r, x, positions):
    """``x [n, heads, d]`` in 64 bits, and the sum of the magnitudes that a result is made of."""
    x, h = x.double(), r.rotary_dim // 2
    angle = positions.cpu().double()[:, None] * r.inv_freq.cpu()
    unit = torch.polar(torch.full_like(angle, r.attention_factor), angle)[:, None]
    y, size = x.clone(), x.abs()
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if r.interleaved else (slice(0, h), slice(h, 2 * h))
    z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * unit
    y[..., a], y[..., b] = z.real, z.imag
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * r.attention_factor
    return y, size


def check(r, x, positions, got):
    exact, size = turned(r, x.cpu(), positions)
    # the turn: cosine within 3 units (reduction, polynomial, factor), product and sum one each; positions times frequencies
    # are off by 2^-53 of their number of turns, which is under a unit up to 2^28 turns; then the one rounding
    slack = 6 * 2.0**-24 * size
    off = (got.cpu().double() - exact).abs()
    small = 2.0**-25 if got.dtype == F16 else 0.0  # steps of the smallest float16 numbers
    assert bool((off <= slack + HALF[got.dtype] * (exact.abs() + slack) + small).all()), float((off / (slack + 1e-30)).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [(128, 128), (256, 64), (64, 16), (80, 80), (96, 24), (6, 2), (64, 10), (192, 64)])
@pytest.mark.parametrize("n", [1, 7, 5000])
def test_rotations(dev, dtype, interleaved, dims, n):
    gen = torch.Generator().manual_seed(n)
    r = RotaryEmbedding(dims[0], dims[1], 1e6, interleaved, YARN if n == 7 else None, dev)
    hq, hkv = (5, 1) if n == 5000 else (6, 2)
    qkv = torch.randn(n, (hq + 2 * hkv) * dims[0], generator=gen).to(dtype)
    positions = torch.randint(-100, 3_000_000, (n,), generator=gen)
    device = qkv.to(dev)
    q, k = device[:, : hq * dims[0]], device[:, hq * dims[0]: (hq + hkv) * dims[0]]
    out_q, out_k = r(positions.to(dev), q, k)
    assert out_q.shape == q.shape and out_q.is_contiguous() and out_k.is_contiguous()
    for x, y, heads in ((q, out_q, hq), (k, out_k, hkv)):
        check(r, x.reshape(n, heads, dims[0]), positions, y.view(n, heads, dims[0]))
    assert torch.equal(device.cpu(), qkv)
    # in place, with 32-bit positions and rows of heads
    r(positions.int().to(dev), q.view(n, hq, dims[0]) if n == 1 else q, k.view(n, hkv, dims[0]) if n == 1 else k,
      out=(q.view(n, hq, dims[0]) if n == 1 else q, k.view(n, hkv, dims[0]) if n == 1 else k))
    assert torch.equal(q, out_q) and torch.equal(k, out_k)
    assert torch.equal(device[:, (hq + hkv) * dims[0]:].cpu(), qkv[:, (hq + hkv) * dims[0]:])


def test_rows_at_odd_places_and_no_keys(dev):
    gen = torch.Generator().manual_seed(2)
    r = RotaryEmbedding(64, device=dev)
    wide = torch.randn(9, 3 + 4 * 64, generator=gen).to(dev, BF16)
    positions = torch.arange(9, device=dev)
    got, none = r(positions, wide[:, 3:])
    assert none is None
    assert torch.equal(got, r(positions, wide[:, 3:].contiguous())[0])
    check(r, wide[:, 3:].reshape(9, 4, 64), positions, got.view(9, 4, 64))
    flipped = wide[:, 3:].t().contiguous().t()  # neither rows nor elements adjacent
    assert torch.equal(r(positions, flipped)[0], got)
    assert r(positions[:0], wide[:0, 3:])[0].shape == (0, 256)


def test_far_positions(dev):
    """The angle at position 2^30 is as good as at 1."""
    r = RotaryEmbedding(64, device=dev)
    positions = torch.tensor([2**30, 2**30 + 1, -(2**30), 2**40 // 3, 0])
    x = torch.ones(5, 1, 64)
    got = r(positions.to(dev), x.to(dev))[0]
    far = positions.abs() < 2**31
    check(r, x[far], positions[far], got[far])


@pytest.mark.parametrize("scaling", [None, YARN])
def test_table(dev, scaling):
    r = RotaryEmbedding(128, 64, 1e6, scaling=scaling, device=dev)
    table = r.cos_sin_cache(70001)
    angle = torch.arange(70001, dtype=torch.float64)[:, None] * r.inv_freq.cpu()
    exact = torch.cat([angle.cos(), angle.sin()], dim=1) * r.attention_factor
    # a cosine is off by the angle's rounding (under a unit of pi / 4) and a unit and a half of its own, then the factor's
    assert float((table.cpu().double() - exact).abs().max()) <= 4 * 2.0**-24 * r.attention_factor
    unit = r.cos_sin_cache(70001, unit=True)
    assert float((unit.cpu().double() - exact / r.attention_factor).abs().max()) <= 4 * 2.0**-24
    # what takes the table turns as the rotation does
    k = torch.randn(50, 2, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    small = RotaryEmbedding(64, 64, 1e6, scaling=scaling, device=dev)
    at = torch.arange(1000, 1050, device=dev)
    torch.testing.assert_close(apply_rope_correction(k, at, small.cos_sin_cache(2000)), small(at, k)[0], rtol=0, atol=4e-6)


def test_recorded_and_on_another_stream(dev):
    gen = torch.Generator().manual_seed(3)
    r = RotaryEmbedding(128, device=dev)
    q, positions = torch.randn(300, 1024, generator=gen).to(dev, BF16), torch.arange(300, device=dev)
    want = r(positions, q)[0]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = r(positions, q)[0]
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph):
        out = r(positions, q)[0]
    for _ in range(3):
        positions += 17
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(out, r(positions, q)[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_that_no_cache_holds(dev, interleaved):
    """What is rotated in one call is what is rotated row by row, past 256 MB too, and of a few narrow rows a workgroup."""
    r = RotaryEmbedding(256, interleaved=interleaved, device=dev)
    q = torch.randn(13000, 5120, dtype=torch.bfloat16, device=dev)
    at = torch.arange(13000, device=dev) * 7
    got, _ = r(at, q)
    for first in (0, 6000, 12900):
        part = slice(first, first + 100)
        assert torch.equal(got[part], r(at[part], q[part])[0])
    narrow = q[:, 512:1024]
    assert torch.equal(r(at, narrow)[0], got[:, 512:1024])


def test_refusals(dev):
    r = RotaryEmbedding(64, device=dev)
    q, at = torch.zeros(4, 128, device=dev), torch.arange(4, device=dev)
    for args in ((at[:3], q), (at.float(), q), (at[None], q), (at.cpu(), q), (at, q[:, :100]), (at, q, q.half()), (at, q, q[:3]),
                 (at, q.view(4, 1, 128))):
        with pytest.raises(ValueError):
            r(*args)
    for out in ((q.half(), None), (q[:, :64], None), (q.t().contiguous().t(), None), (None, None)):
        with pytest.raises(ValueError, match="out"):
            r(at, q, out=out)
    with pytest.raises(ValueError, match="overlap"):
        r(at, q, out=(torch.zeros(200, device=dev).as_strided((4, 128), (10, 1)), None))
    both = torch.randn(5, 300, device=dev)
    for bad in (both[1:, :128], both[:4, 8:136]):  # results over rows that are still to be read
        with pytest.raises(ValueError, match="apart"):
            r(at, both[:4, :128], out=(bad, None))
    want = r(at, both[:4, :128].clone())[0]
    r(at, both[:4, :128], out=(both[:4, 140: 268], None))  # beside them
    assert torch.equal(both[:4, 140: 268], want)
    # q and k of one array: what becomes of either lies apart from the other
    qkv = torch.randn(5, 192 + 64, device=dev)
    q, k = qkv[:4, :128], qkv[:4, 128: 192]
    want = r(at, q.clone(), k.clone())
    for bad in ((k, q), (q, qkv[1:, 128: 192]), (qkv[:4, 64: 192], k), (torch.empty(4, 128, device=dev), qkv[:4, 64: 128])):
        with pytest.raises(ValueError):
            r(at, q, k, out=bad)
    one = torch.empty(4, 128, device=dev)
    with pytest.raises(ValueError, match="apart"):
        r(at, q, k, out=(one, one[:, :64]))
    r(at, q, k, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    with pytest.raises(ValueError, match="max_position"):
        r.cos_sin_cache(0)
