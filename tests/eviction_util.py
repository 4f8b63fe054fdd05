"""Attention weights of a step from their definition, in 64 bits on the CPU, and the bound of what rounding may do."""

from __future__ import annotations

import math

import torch

from async_llm_amd.kvcache import MHAKVCache, QuantizedKVCache
from async_llm_amd.shared_cache import CacheBlock, QuantizedCacheAttention, SharedCacheAttention
from tests.quant_util import quantised32, rows64, turns, write

UNIT = 2.0**-24  # half a step of 32 bits, relative


def make_op(dev, hq, hkv, d, page, dtype, pages, codes=None, rotary=None, mrope=None, positions=4096, layers=1):
    rotary = d if rotary is None else rotary
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    table = torch.cat([angle.cos(), angle.sin()], dim=1).float().to(dev)
    more = dict(rotary_dim=rotary)
    if mrope:
        more.update(mrope_section=mrope, rope_base=1e4)
    if codes is None:
        return SharedCacheAttention(MHAKVCache(hkv, layers, d, pages, page, dtype, dev), table, hq, hkv, d, page, dtype, dev, **more)
    pool = QuantizedKVCache(hkv, layers, d, pages, page, dtype, dev, codes)
    return QuantizedCacheAttention(pool, table, hq, hkv, d, page, dtype, dev, **more)


def fill(op, gen, layer=0, garbage=None):
    """Random rows in every slot; ``garbage``: what slots that nobody reads hold instead (set by the caller)."""
    pool = op.kv_cache
    if isinstance(pool, QuantizedKVCache):
        slots = torch.arange(pool.num_pages * pool.page_size)
        for which in (0, 1):
            x = torch.randn(len(slots), op.num_kv_heads, op.head_dim, generator=gen)
            write(pool, which, layer, slots, *quantised32(x, pool.code_dtype))
    else:
        for x in (pool.k_cache(layer), pool.v_cache(layer)):
            x.copy_(torch.randn(x.shape, generator=gen))


def keys64(op, layer, slots):
    if isinstance(op.kv_cache, QuantizedKVCache):
        return rows64(op.kv_cache, 0, layer, slots)
    flat = op.kv_cache.k_cache(layer).cpu().double().reshape(-1, op.num_kv_heads, op.head_dim)
    return flat[torch.as_tensor(slots, dtype=torch.int64)]


def turned64(op, x, where):
    """``x [n, heads, d]`` in 64 bits, rotated to ``where [n]`` or ``[3, n]``."""
    half = op.rotary_dim // 2
    if half == 0:
        return x
    if op.mrope_section is None:
        c, s = turns(op, where)
    else:
        where = where if where.dim() == 2 else torch.stack([where] * 3)
        c, s = turns(op, where)
    a, b = x[..., :half], x[..., half: 2 * half]
    return torch.cat([c[:, None] * a - s[:, None] * b, c[:, None] * b + s[:, None] * a, x[..., 2 * half:]], dim=-1)


def weights64(op, q, lse, meta, weights, layer=0, window=0):
    """``weights`` with what a step adds, in 64 bits, and how far 32 bits may be off it.

    A score is a sum of D products of a key (exact) and a query element, which the rotation (two products, a sum and the cosine's
    own rounding), the scale and its split leave within 8 units; sums of D terms in any order stay within D units of the sum
    of magnitudes A.  Cosines of mRoPE angles are within two units more.  exp2 of its argument, a score less a log-sum, loses a
    unit of each of those (times log2 e and back) and two of its own; n weights added up lose n units at most."""
    arrays, sub_worker, _ = meta.launch.host_tables
    qo, kvp, kvi, lens, flags = (torch.from_numpy(a).long() for a in arrays[:5])
    P, G, hkv, D = op.page_size, op.num_qo_heads // op.num_kv_heads, op.num_kv_heads, op.head_dim
    q, lse, out = q.cpu().double().view(-1, op.num_qo_heads, D), lse.cpu().double(), weights.cpu().double().clone()
    total, slack = torch.zeros_like(out), torch.zeros_like(out)
    count = torch.zeros(out.shape[1], dtype=torch.float64)
    loc, worker = meta.sub_loc.cpu(), meta.sub_worker.cpu()
    for s in range(len(lens)):
        n, rows = int(lens[s]), range(int(qo[s]), int(qo[s + 1]))
        entries = kvi[kvp[s]: kvp[s + 1]]
        if flags[s] & 2:
            slots = entries[:n]
        else:
            slots = (entries[:, None] * P + torch.arange(P)).reshape(-1)[:n]
        if n == 0 or not len(rows):
            continue
        k = keys64(op, layer, slots)  # [n, hkv, D]
        index = torch.tensor(list(rows))
        x = turned64(op, q[worker[index]], loc[..., index]).view(-1, hkv, G, D)
        # rotating mixes two elements: both magnitudes count
        mixed = turned64_abs(op, q[worker[index]]).view(-1, hkv, G, D)
        score = torch.einsum("rhgd,nhd->rhgn", x, k) / math.sqrt(D)
        size = torch.einsum("rhgd,nhd->rhgn", mixed, k.abs()) / math.sqrt(D)
        l = lse[worker[index]].view(-1, hkv, G, 1)
        p = torch.exp(score - l)
        seen = torch.ones(len(rows), n, dtype=torch.bool)
        if flags[s] & 1:
            seen = torch.arange(n)[None] <= n - len(rows) + torch.arange(len(rows))[:, None]
        if window:
            seen = seen & (torch.arange(len(rows))[:, None] >= len(rows) - window)
        dead = (l == -math.inf).expand_as(p)
        hidden = dead | ~seen[:, None, None, :]
        p = p.masked_fill(hidden, 0.0)
        error = ((D + 16) * size + 2 * (score.abs() + l.abs()) + 4) * UNIT
        error = (p * error).masked_fill(hidden, 0.0)
        total.index_add_(1, slots, p.sum((0, 2)))
        slack.index_add_(1, slots, error.sum((0, 2)))
        count.index_add_(0, slots, torch.full((n,), float(len(rows) * G), dtype=torch.float64))
    out += total
    return out, slack + (count + 2) * UNIT * total + UNIT * out.abs()


def turned64_abs(op, x):
    half, x = op.rotary_dim // 2, x.abs()
    if half == 0:
        return x
    a, b = x[..., :half], x[..., half: 2 * half]
    return torch.cat([a + b, a + b, x[..., 2 * half:]], dim=-1)


def blocks_of(op, r, lengths, pages):
    """Blocks of these lengths over pages taken from the list ``pages``."""
    out = []
    for n in lengths:
        b = CacheBlock(op.device, op.page_size)
        b.num_tokens = n
        b.page_starts = [pages.pop() * op.page_size for _ in range(-(-n // op.page_size))]
        b.token_ids = [r.randrange(1000) for _ in range(n)]
        out.append(b)
    return out
