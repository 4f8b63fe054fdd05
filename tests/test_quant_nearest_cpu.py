"""The check of codes itself: it takes the nearest ones and no others."""

import pytest
import torch

from tests import quant_util as Q
from tests.quant_nearest import assert_nearest, spacing

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def rows(codes, seed=0):
    x = torch.randn(200, 2, 64, generator=torch.Generator().manual_seed(seed))
    x *= torch.exp(2 * torch.randn(200, 2, 1, generator=torch.Generator().manual_seed(seed + 1)))
    c, s = Q.quantised32(x, codes)
    return x.double(), c, s, torch.pow(2.0, s.double() - 127)[..., None]


@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_nearest_codes_pass(codes):
    x, c, s, _ = rows(codes)
    assert_nearest(c, s, x, torch.zeros_like(x), codes)
    # ... of rows that 32 bits have moved by a little, up to what is said
    moved = x * (1 + 2.0**-22 * torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(5)).clamp(-1, 1))
    assert_nearest(c, s, moved, 2.0**-21 * x.abs().amax(-1, keepdim=True).expand(x.shape), codes)


@pytest.mark.parametrize("off", [0.0, 2.0**-20])
@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_truncated_codes_do_not(codes, off):
    x, c, s, step = rows(codes)
    y = x / step
    gap = spacing(y, codes)
    cut = torch.trunc(y / gap) * gap
    cut = cut.to(torch.int8) if codes == INT8 else cut.float().to(E4M3)
    assert (cut.float() != c.float()).double().mean() > 0.3
    with pytest.raises(AssertionError, match="further from its element"):
        assert_nearest(cut, s, x, off * x.abs().amax(-1, keepdim=True).expand(x.shape), codes)


@pytest.mark.parametrize("codes", [E4M3, INT8])
def test_one_code_that_is_off_by_one_does_not(codes):
    x, c, s, _ = rows(codes)
    off = 2.0**-20 * x.abs().amax(-1, keepdim=True).expand(x.shape)
    for at, by in (((0, 0, 3), 1), ((57, 1, 60), -1), ((199, 1, 0), 1)):
        raw = c.view(torch.uint8).clone()
        raw[at] = (int(raw[at]) + by) % 256
        with pytest.raises(AssertionError):
            assert_nearest(raw.view(codes), s, x, off, codes)
