"""Chunks that are read back, where one key has nearly all of the weight and very many have the rest: each of their weights is
under what float16 holds beside 1, their sum is not."""

import pytest
import torch

from async_llm_amd.kvcache import QuantizedKVCache
from async_llm_amd.shared_cache import QuantizedCacheAttention
from tests import quant_util as Q


@pytest.mark.gpu
@pytest.mark.parametrize("new", [4098, 3])  # rows in wide tiles and a few behind them; narrow tiles alone
@pytest.mark.parametrize("at", [0, 30000])  # where the large one lies
def test_many_small_weights_count(new, at):
    dev, tokens, heads, D = torch.device("cuda"), 65536, 16, 64
    n_pages = tokens // 16 + -(-new // 16)
    codes = torch.zeros(2, 1, n_pages, heads, 16, D, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    scales = torch.full((2, 1, n_pages, heads, 16), 127, dtype=torch.uint8, device=dev)
    pool = QuantizedKVCache.from_buffers(codes, scales, torch.bfloat16)
    op = QuantizedCacheAttention(pool, torch.zeros(1, 1), 4 * heads, heads, D, 16, torch.bfloat16, dev, rotary_dim=0)
    op._reads_back = lambda pairs, pages: True
    # scores 18 (times log2(e): 25.97) for one token, whose value is 0, and 0 for the others, whose values are 1
    one = codes.view(torch.uint8)
    value = lambda x: torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8).item()
    one[1, 0, : tokens // 16] = value(1.0)
    one[0, 0, at // 16, :, at % 16] = value(2.25)
    one[1, 0, at // 16, :, at % 16] = 0
    context, own = Q.Pages(1, 16).block(dev, 0), Q.Pages(1, 16).block(dev, 0)
    context.page_starts, context.num_tokens = [16 * i for i in range(tokens // 16)], tokens
    own.page_starts, own.spare = [], [tokens + 16 * i for i in range(-(-new // 16))]
    step = Q.prefill_step(op, [([context], own, new)])
    assert step.meta.launch.readback is not None
    q = torch.ones(new, 4 * heads * D, dtype=torch.bfloat16, device=dev)
    out, lse = op.attend(q, 0, step.meta, return_lse=True)
    row = torch.arange(new, dtype=torch.float64)
    small = torch.exp(torch.tensor(-18.0, dtype=torch.float64))
    total = 1 + small * (tokens - 1 + row + 1)  # (the row's own block has keys of score 0 and values of 0)
    want = (small * (tokens - 1) / total)[:, None]
    # The result is rounded to float16 (2^-11) and bf16 (2^-8), its sums to 32 bits; a weight loses 2^-33 of the largest (2^-25 where the
    # largest is 2^8) or 2^-11 of itself, its exponent of 26 in 32 bits 26 * 2^-23.
    room = want * (2.0**-8 + 2 * 2.0**-11 + (tokens + 64) * 2.0**-24 + 2.0**-16) + tokens * 2.0**-33
    error = (out.cpu().double() - want).abs()
    assert (error <= room).all(), f"{out.min().item()} to {out.max().item()} where {want.min().item()} to {want.max().item()} was expected"
    assert (lse.cpu().double() - (18 + total.log())[:, None]).abs().max() <= 18 * 2.0**-22 + (tokens + 64) * 2.0**-23
