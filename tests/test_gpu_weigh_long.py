"""Attention weights of views so long that a wave writes the sums it holds several times on its way."""

import pytest
import torch

from async_llm_amd.shared_cache import CacheBlock, CacheEviction, WorkerGroup
from tests.eviction_util import UNIT, make_op, turned64, turned64_abs

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


def fill(op, gen):
    """Random keys of every slot, made on the GPU; a few e4m3 codes are NaN (elements over 464)."""
    pool = op.kv_cache
    if not hasattr(pool, "k_codes"):
        for page in pool.k_cache(0).split(256):
            page.copy_(torch.randn(page.shape, device=op.device, generator=gen))
        return
    for codes, scales in zip(pool.k_codes(0).split(256), pool.k_scales(0).split(256)):
        x = torch.randn(codes.shape, device=op.device, generator=gen)
        codes.view(torch.uint8).copy_((x * 100 if pool.code_dtype == E4M3 else (x * 30).round().clamp(-127, 127)).to(pool.code_dtype).view(torch.uint8))
        scales.view(torch.uint8).copy_(torch.randint(119, 122, scales.shape, device=op.device, generator=gen))


def keys64(op, slots, heads):
    """``[n, heads, d]`` on the GPU."""
    pool, page, place = op.kv_cache, slots // op.page_size, slots % op.page_size
    if not hasattr(pool, "k_codes"):
        return pool.k_cache(0)[page, place, heads].double()
    codes = pool.k_codes(0).view(torch.uint8)[page, heads, place].view(pool.code_dtype).double()
    return codes * torch.pow(2.0, pool.k_scales(0).view(torch.uint8)[page, heads, place].double() - 127)[..., None]


# tokens of a strip that a wave holds: 2048, half of that of tokens looked up one by one, 512 of rows of 1 KB
@pytest.mark.parametrize("dtype, codes, hkv, D, page, tokens, held", [
    (BF16, None, 256, 64, 16, 24007, 2048),
    (BF16, None, 256, 64, 1, 12011, 1024),
    (F16, None, 256, 64, 5, 20003, 1024),
    (F32, None, 128, 256, 16, 10005, 512),
    (BF16, E4M3, 256, 64, 16, 24007, 2048),
    (F16, INT8, 256, 64, 1, 20003, 1024),
])
def test_sums_are_written_on_the_way(dtype, codes, hkv, D, page, tokens, held):
    dev, gen = torch.device("cuda:0"), torch.Generator(device="cuda").manual_seed(tokens)
    pages = -(-tokens // page) + 8
    op = make_op(dev, hkv, hkv, D, page, dtype, pages, codes, positions=tokens + 100)
    fill(op, gen)
    order = torch.randperm(pages, device=dev, generator=gen)
    starts = (order * page).tolist()
    block, own = CacheBlock(dev, page), CacheBlock(dev, page)
    for b, n in ((block, tokens), (own, 0)):
        b.page_starts, b.num_tokens = [starts.pop() for _ in range(-(-n // page))], n
    opened = starts.pop()
    meta = op.prepare(WorkerGroup(cache_structure=[[block, own]], write_to=[own]), {id(own): opened}, torch.tensor([opened], dtype=torch.int32, device=dev))
    e = CacheEviction(op)
    plan = e.plan(meta)
    words = plan.refs[0].numpy()
    items, strips = words[words[6]: words[6] + 8 * words[1]].reshape(-1, 8), words[words[21]: words[21] + words[20] + 1]
    longest = max(int(items[a: b, 2].sum()) for a, b in zip(strips, strips[1:]))
    assert longest > held + 64  # (four heads a workgroup: a wave has all tokens of its strip)

    q = torch.randn(1, hkv * D, generator=torch.Generator().manual_seed(1)).to(dtype)
    loc = meta.sub_loc.cpu()
    x = [turned64(op, q.double().view(1, hkv, D), loc[i: i + 1]).to(dev) for i in range(2)]
    mixed = turned64_abs(op, q.double().view(1, hkv, D)).to(dev)
    arrays = meta.launch.host_tables[0]
    slots = []
    for i in range(2):
        at = torch.from_numpy(arrays[2][arrays[1][i]: arrays[1][i + 1]]).long()
        slots.append((at[:, None] * page + torch.arange(page)).reshape(-1)[: arrays[3][i]].to(dev))
    every = torch.cat(slots)
    assert len(every) == tokens + 1
    score, size = torch.empty(2, hkv, tokens + 1, dtype=torch.float64, device=dev)
    for h in range(0, hkv, 16):
        heads = slice(h, h + 16)
        k = keys64(op, every, heads)
        y = torch.cat([part[:, heads].expand(len(s), -1, -1) for part, s in zip(x, slots)])
        score[heads] = (k * y).sum(-1).T / D**0.5
        size[heads] = (k.abs() * mixed[:, heads]).sum(-1).T / D**0.5
    strange = score.isnan()  # (sums of these tokens alone are not numbers)
    assert bool(strange.any()) == (codes == E4M3)
    lse = torch.logsumexp(score.masked_fill(strange, float("-inf")), -1).float()[None].contiguous()
    p = torch.exp(score - lse.double().T)
    weights = torch.rand(hkv, e.num_slots, device=dev, generator=gen) / tokens
    want, slack = weights.double(), torch.zeros(hkv, e.num_slots, dtype=torch.float64, device=dev)
    want[:, every] += p
    slack[:, every] = p * ((D + 16) * size + 2 * (score.abs() + lse.double().T.abs()) + 4) * UNIT + 3 * UNIT * p
    slack += UNIT * want
    before = weights.clone()
    apart = torch.full_like(weights, 9.0)
    e.accumulate(q.to(dev), lse, 0, plan, weights, out=apart)
    assert torch.equal(weights, before)
    off = (apart.double() - want).abs()[:, every] / slack[:, every]
    assert torch.equal(apart[:, every].isnan(), strange)
    assert float(off[~strange].max()) <= 1.0
    unseen = torch.ones(e.num_slots, dtype=torch.bool, device=dev)
    unseen[every] = False
    assert bool((apart[:, unseen] == 9.0).all())
    e.accumulate(q.to(dev), lse, 0, plan, weights)
    assert torch.equal(weights[:, every].nan_to_num(7.0), apart[:, every].nan_to_num(7.0)) and torch.equal(weights[:, unseen], before[:, unseen])
