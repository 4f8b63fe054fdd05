"""Slots that nobody sees stay as they are where lists name single slots of a page with others between them."""

import numpy as np
import pytest
import torch

from async_llm_amd import native
from tests.test_weigh_plan_cpu import expected, plan_of

pytestmark = pytest.mark.gpu
SLOTS, CAUSAL = native.VA_SUB_SLOTS, native.VA_SUB_CAUSAL


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("subs", [
    [(1, [3, 8, 9, 40], 4, SLOTS), (1, [2], 1, 0), (2, [41, 44], 2, SLOTS)],
    [(9, [4], 1, CAUSAL), (40, [70, 66, 79], 3, SLOTS), (1, [1, 0], 2, 0)],  # tile items
])
def test_unseen_slots_are_left(dtype, page, subs):
    dev, gen, pages, (hq, hkv, D) = torch.device("cuda:0"), torch.Generator().manual_seed(page), 80 // page + 1, (8, 2, 64)
    kind = native.dtype_id(dtype)
    rc, words, counts = plan_of(subs, (hq, hkv, D), page, pages, dtype=kind)
    assert rc == 0, native.lib.va_last_error()
    rows, slots = sum(n for n, *_ in subs), pages * page
    k = torch.randn(slots, hkv, D, generator=gen).to(dtype)
    q = torch.randn(rows, hq, D, generator=gen).to(dtype)
    lse = 3.0 + torch.rand(rows, hq, generator=gen)
    weights, out = torch.rand(2, hkv, slots, generator=gen)
    device = {name: t.to(dev) for name, t in dict(k=k, q=q, lse=lse, weights=weights, out=out, plan=torch.from_numpy(words[: counts.plan_words]),
                                                  worker=torch.arange(rows), loc=torch.zeros(rows, dtype=torch.int64)).items()}
    scratch = torch.empty(counts.workspace_bytes, dtype=torch.uint8, device=dev)
    at = {name: t.data_ptr() for name, t in device.items()}
    header = np.ascontiguousarray(words[:24])
    native.call_on(dev, native.lib.va_weigh, at["q"], hq * D, at["k"], hkv * D, pages, at["plan"], header.ctypes.data, at["worker"], at["loc"], 0,
                   at["lse"], 0, at["weights"], at["out"], scratch.data_ptr(), scratch.numel(), native.VaShape(hq, hkv, D, page, kind),
                   native.VaRope(native.VA_ROPE_TABLE, 0, None, 0, 0, 0, None), native.current_stream_ptr(dev))
    want, slack, seen = weights.double(), torch.zeros(hkv, slots, dtype=torch.float64), torch.zeros(slots, dtype=torch.bool)
    score = torch.einsum("rhgd,nhd->rhgn", q.double().view(rows, hkv, -1, D), k.double()) / D**0.5
    size = torch.einsum("rhgd,nhd->rhgn", q.double().abs().view(rows, hkv, -1, D), k.double().abs()) / D**0.5
    l = lse.double().view(rows, hkv, -1, 1)
    p = torch.exp(score - l)
    # a score loses a unit for each of its D products and a few for its query's parts and scale, a log-sum two; exp2 two of its own
    error = p * ((D + 8) * size + 2 * (score.abs() + l.abs()) + 4) * 2.0**-24
    pairs = expected(subs, hq // hkv, page, 0)
    for (row, slot), times in pairs.items():
        n = times // (hq // hkv)
        want[:, slot] += n * p[row, :, :, slot].sum(-1)
        slack[:, slot] += n * error[row, :, :, slot].sum(-1)
        seen[slot] = True
    slack = slack + (len(pairs) * hq // hkv + 2) * 2.0**-24 * want
    got = device["out"].cpu()
    assert torch.equal(got[:, ~seen], out[:, ~seen])
    assert bool(((got.double() - want).abs() <= slack)[:, seen].all())
    assert torch.equal(device["weights"].cpu(), weights)
