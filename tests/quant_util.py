"""The 8-bit pool's operators from their definition, in 64 bits on the CPU, and the bounds of what rounding may do."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from async_llm_amd.kvcache import QuantizedKVCache
from async_llm_amd.shared_cache import CacheBlock, QuantizedCacheAttention

LIMIT = {torch.float8_e4m3fn: 1.875 * 2.0**127, torch.int8: 127 * 2.0**121}  # what a code may stand for in 32 bits
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
EPS = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step, of the value
OPERAND = {False: 2.0**-17, True: 2.0**-11}  # of queries and weights: sums of two bf16 numbers, or float16
HALF_KEY = {torch.float8_e4m3fn: -1, torch.int8: 1}  # log2 of what a code of the largest scale counts as float16 key


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
def scale_bytes(x: torch.Tensor, code_dtype) -> torch.Tensor:
    """Smallest byte b >= 1 with max|x| <= largest * 2^(b - 127), by comparison; 255 for rows that are not finite."""
    top = x.double().abs().amax(-1).clamp(max=LIMIT[code_dtype])
    b = torch.arange(1, 255, dtype=torch.float64)
    edges = LARGEST[code_dtype] * torch.pow(2.0, b - 127)
    out = torch.searchsorted(edges, top.nan_to_num(0.0, 0.0, 0.0).contiguous()) + 1
    return torch.where(torch.isfinite(x).all(-1), out, 255).to(torch.uint8)


def quantised32(x: torch.Tensor, code_dtype):
    """Codes and scale bytes of 32-bit rows: the scaled row is exact, the rounding torch's."""
    b = scale_bytes(x, code_dtype)
    y = x.double().clamp(-LIMIT[code_dtype], LIMIT[code_dtype]) / torch.pow(2.0, b.double() - 127)[..., None]
    y = torch.where((b == 255)[..., None], 0.0, y).float()
    return (y.to(code_dtype) if code_dtype == torch.float8_e4m3fn else y.round().to(torch.int8)), b


def values64(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    b = scales.view(torch.uint8).double()
    v = codes.float().double() * torch.pow(2.0, b - 127)[..., None]
    return torch.where((b == 255)[..., None], math.nan, v)


def write(pool: QuantizedKVCache, which: int, layer: int, slots, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Put ``codes [n, kv_heads, head_dim]`` and their scale bytes into slots."""
    s = torch.as_tensor(slots, dtype=torch.int64)
    page, place = s // pool.page_size, s % pool.page_size
    for tensor, x in (((pool.k_codes, pool.v_codes)[which](layer), codes), ((pool.k_scales, pool.v_scales)[which](layer), scales)):
        held = tensor.view(torch.uint8).cpu()
        held[page, :, place] = x.view(torch.uint8)
        tensor.view(torch.uint8).copy_(held)


def scales_of(pool: QuantizedKVCache, which: int, layer: int, slots) -> torch.Tensor:
    scales = (pool.k_scales, pool.v_scales)[which](layer).cpu().view(torch.uint8)
    s = torch.as_tensor(slots, dtype=torch.int64)
    page, place = s // pool.page_size, s % pool.page_size
    return scales[page, :, place]


def rows64(pool: QuantizedKVCache, which: int, layer: int, slots) -> torch.Tensor:
    """``[n, kv_heads, head_dim]`` values of slots, on the CPU."""
    codes = (pool.k_codes, pool.v_codes)[which](layer).cpu().view(torch.uint8)
    scales = (pool.k_scales, pool.v_scales)[which](layer).cpu().view(torch.uint8)
    s = torch.as_tensor(slots, dtype=torch.int64)
    page, place = s // pool.page_size, s % pool.page_size
    return values64(codes[page, :, place].view(pool.code_dtype), scales[page, :, place])


def turns(op, where: torch.Tensor, double=True):
    """Cosines and sines ``[n, pairs]`` of ``where [n]`` or ``[3, n]`` (angles: 32-bit products, by definition)."""
    where = where.cpu()
    if op.mrope_section is None:
        table = op.cos_sin_cache.cpu()
        rows = table[where.abs().clamp(max=table.shape[0] - 1)]
        c, s = rows[:, : op.rotary_dim // 2], rows[:, op.rotary_dim // 2: op.rotary_dim]
        s = torch.where((where < 0)[:, None], -s, s)
        return (c.double(), s.double()) if double else (c, s)
    if where.dim() == 1:
        where = where.expand(3, -1)
    pair = torch.arange(op.rotary_dim // 2)
    _, h, w = op.mrope_section
    axis = torch.where((pair % 3 == 1) & (pair < 3 * h), 1, torch.where((pair % 3 == 2) & (pair < 3 * w), 2, 0))
    angle = (where.float()[axis].T * op._mrope_inv_freq.cpu()).double()
    return (angle.cos(), angle.sin()) if double else (angle.cos().float(), angle.sin().float())


def rotated(op, x: torch.Tensor, where: torch.Tensor, double=True) -> torch.Tensor:
    """``x [n, heads, d]`` rotated row by row; in 32 bits every product and sum is rounded by itself."""
    if op.rotary_dim == 0:
        return x.double() if double else x.float()
    c, s = (t[:, None] for t in turns(op, where, double))
    x = x.double() if double else x.float()
    h = op.rotary_dim // 2
    a, b = x[..., :h], x[..., h: 2 * h]
    return torch.cat([c * a - s * b, c * b + s * a, x[..., 2 * h:]], dim=-1)


def assert_quantises(codes: torch.Tensor, scales: torch.Tensor, x64: torch.Tensor, off: torch.Tensor, code_dtype):
    """Every finite row's scale is the smallest that holds it, every code the nearest, where ``off`` (elements) is how
    far the 32-bit row may be from the 64-bit one."""
    L = LARGEST[code_dtype]
    x64 = x64.clamp(-LIMIT[code_dtype], LIMIT[code_dtype])
    b = scales.view(torch.uint8).double()
    step = torch.pow(2.0, b - 127)
    top, slack = x64.abs().amax(-1), off.amax(-1)
    assert (top <= L * step + slack).all(), "a scale is too small for its row"
    assert ((top > L * step / 2 - slack) | (b == 1)).all(), "a scale is larger than its row needs"
    y = x64 / step[..., None]
    if code_dtype == torch.int8:
        gap = torch.ones_like(y)
    else:  # spacing of e4m3 codes around y: 2^(exponent - 3), from 2^-9 on
        gap = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    err = (codes.float().double() - y).abs()
    room = gap / 2 + off / step[..., None]
    # (over the upper edge of a binade the spacing is twice as large: a 32-bit row just above it has rounded there)
    assert (err <= room * (1 + 1e-9)).all() or (err <= torch.where(err <= room * (1 + 1e-9), err, gap + off / step[..., None])).all()


def turn_error(x: torch.Tensor) -> torch.Tensor:
    """How far a pair rotated in 32 bits may be from its 64-bit value: sines and cosines to 1.5 units in the last place
    (2^-24 each, at most), two products, a sum: under 8 * 2^-24 of the two magnitudes together."""
    return 8 * 2.0**-24 * 2 * x.double().abs().amax(-1, keepdim=True).expand(x.shape)


# ---------------------------------------------------------------------------
# a pool, an op, blocks
# ---------------------------------------------------------------------------
def make(device, heads, page, num_pages, dtype=torch.bfloat16, code_dtype=torch.float8_e4m3fn, rotary=None, mrope=None,
         layers=1, max_pos=4096, seed=0, base=10000.0, kernel=None):
    """An op over a pool with random content."""
    Hq, Hkv, D = heads
    g = torch.Generator().manual_seed(seed)
    pool = QuantizedKVCache(Hkv, layers, D, num_pages, page, dtype, device, code_dtype)
    for layer in range(layers):
        for codes, scales in ((pool.k_codes, pool.k_scales), (pool.v_codes, pool.v_scales)):
            x = torch.randn(num_pages, Hkv, page, D, generator=g) * torch.exp(torch.randn(num_pages, Hkv, page, 1, generator=g))
            c, b = quantised32(x, code_dtype)
            codes(layer).view(torch.uint8).copy_(c.view(torch.uint8))
            scales(layer).view(torch.uint8).copy_(b)
    rotary = D if rotary is None else rotary
    table = torch.zeros(1, max(rotary, 1))
    if rotary and mrope is None:
        angle = torch.arange(max_pos, dtype=torch.float64)[:, None] / base ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
        table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    op = QuantizedCacheAttention(pool, table.to(device), Hq, Hkv, D, page, dtype, pool.device, rotary_dim=rotary,
                                 mrope_section=mrope, rope_base=base if mrope else None, kernel=kernel)
    return op, pool, g


class Pages:
    """Pages of a pool in scattered order."""

    def __init__(self, num_pages, page, seed=0):
        self.order = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.page = page

    def block(self, device, tokens, room=0, span=None):
        """A block of ``tokens`` on pages that hold ``room`` more; what is past its own pages is ``block.spare``."""
        b = CacheBlock(device, self.page)
        n, total = -(-tokens // self.page), -(-(tokens + room) // self.page)
        starts = [self.order.pop() * self.page for _ in range(total)]
        b.page_starts, b.spare, b.num_tokens, b.mrope_span_override = starts[:n], starts[n:], tokens, span
        return b


def slots_of(block, tokens=None):
    starts = torch.tensor(list(block.page_starts) + list(getattr(block, "spare", [])), dtype=torch.int64)
    grid = (starts[:, None] + torch.arange(block.page_size)).reshape(-1)
    return grid[: block.num_tokens if tokens is None else tokens]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attention64(op, q: torch.Tensor, segments, layer=0, half=False):
    """One request: ``q [rows, Hq, D]``; ``segments``: ``(slots, positions [rows] or [3, rows], first)`` where token t of
    a segment is visible to row i iff t <= first + i.  Returns out ``[rows, Hq * D]``, lse ``[rows, Hq]`` and the bound of
    score errors, where a query element is off by 2^-17 of itself or, ``half``, by a rounding to float16, the weighted
    values, and what underflow may lose."""
    S, Hq, D = q.shape
    Hkv = op.num_kv_heads
    G = Hq // Hkv
    operand, least = OPERAND[half], 0.0
    if half:
        # q' = q 2^(top - 127 - shift) with the largest scale byte of the keys among the rows; below 2^-14 its steps are
        # even, and it is rounded twice (as it is, and rotated)
        sizes_of = torch.cat([scales_of(op.kv_cache, 0, layer, slots).flatten() for slots, _, _ in segments]).int()
        top = max([1] + sizes_of[sizes_of != 255].tolist())
        least = 2.0 ** (-13 - (top - 127 - HALF_KEY[op.kv_cache.code_dtype]))
    scores, sizes, values = [], [], []
    for slots, where, first in segments:
        k, v = rows64(op.kv_cache, 0, layer, slots), rows64(op.kv_cache, 1, layer, slots)
        r = rotated(op, q, where).view(S, Hkv, G, D)
        x = torch.einsum("shgd,thd->hsgt", r, k) / math.sqrt(D)
        size = torch.einsum("shgd,thd->hsgt", r.abs().clamp(min=least), k.abs()) / math.sqrt(D)
        hidden = torch.arange(len(slots))[None, :] > first + torch.arange(S)[:, None]
        scores.append(x.masked_fill(hidden[None, :, None], -math.inf))
        sizes.append(size.masked_fill(hidden[None, :, None], 0.0))
        values.append(v)
    x, size, v = torch.cat(scores, -1), torch.cat(sizes, -1), torch.cat(values)
    lse = torch.logsumexp(x, -1)
    p = torch.where(torch.isinf(lse)[..., None], 0.0, torch.exp(x - torch.where(torch.isinf(lse), 0.0, lse)[..., None]))
    out = torch.einsum("hsgt,thd->shgd", p, v).reshape(S, Hq * D)
    weight = torch.einsum("hsgt,thd->shgd", p, v.abs()).reshape(S, Hq * D)
    # A score is off by its query's rounding (two bf16 numbers hold 16 bits: 2^-17; float16 for many new tokens: 2^-11) and
    # that of D products in 32 bits (D * 2^-24), both of the magnitudes' sum, its exponent by 2^-23 of itself.
    off = (size.amax(-1) * (operand + D * 2.0**-24) + x.abs().masked_fill(torch.isinf(x), 0.0).amax(-1) * 2.0**-22) if x.shape[-1] else torch.zeros_like(lse)
    off = off.permute(1, 0, 2).reshape(S, Hq)
    # Weights under 2^-126, and low parts of weights under 2^-117, are no normal 32-bit (bf16) numbers and may become zero:
    # less than 2^-125 of a value for each token.
    lost = (v.abs().amax() * len(v) * 2.0**-125 if len(v) else torch.zeros(())).double().expand(S, 1)
    return out, lse.permute(1, 0, 2).reshape(S, Hq), off, weight, lost


def assert_attends(out, lse, expected, dtype, tokens, half=None):
    """|out - out64| <= rounding of the result + (2 * score error + rounding of a weight + sums of 32 bits) * sum p|v|.

    ``half`` marks the rows [rows] that ran in float16 (a number: the largest value's magnitude; 0 others): results are
    rounded to that first, by 2^-11 of themselves or 2^-39 of that, and weights by 2^-11 of themselves or 2^-25 each."""
    o, l, off, weight, lost = expected
    half = (torch.zeros(o.shape[0]) if half is None else half)[:, None]
    operand = torch.where(half > 0, OPERAND[True], OPERAND[False])
    got = out.detach().cpu().double()
    relative = (2 * off + operand + (tokens + 64) * 2.0**-24).repeat_interleave(o.shape[1] // off.shape[1], dim=1)
    room = EPS[dtype] * o.abs() + weight * relative * (1 + EPS[dtype]) + lost + (2.0**-24 if dtype == torch.float16 else 2.0**-126)
    room = room + (half > 0) * 2.0**-11 * o.abs() * (1 + EPS[dtype]) + half * (2.0**-39 + tokens * 2.0**-25)
    assert got.shape == o.shape
    worst = ((got - o).abs() - room).max().item()
    assert worst <= 0, f"out is {worst:.3e} further off than rounding explains"
    if lse is not None:
        seen = torch.isfinite(l)
        have = lse.detach().cpu().double()
        assert torch.equal(torch.isfinite(have), seen)
        slack = off + l.abs().masked_fill(~seen, 0) * 2.0**-22 + (tokens + 64) * 2.0**-23
        assert ((have - l).abs()[seen] <= slack[seen]).all(), "lse"


def decode_step(op, pages, views, writers, gen, buffers=None):
    """Plan a decode step over ``views`` (lists of blocks) whose requests write ``writers``: metadata, and each
    request's segments for :func:`attention64`."""
    from async_llm_amd.shared_cache import WorkerGroup

    P = op.page_size
    group = WorkerGroup(cache_structure=views, write_to=writers)
    pending, slots = {}, []
    for b in writers:
        opened = b.spare[0] if b.num_tokens % P == 0 else None
        pending[id(b)] = opened
        slots.append((b.page_starts[-1] if opened is None else opened) + b.num_tokens % P)
    slots = torch.tensor(slots, dtype=torch.int32, device=op.device)
    meta = op.prepare(group, pending, slots, **({} if buffers is None else {"graph_buffers": buffers}))
    segments = []
    for w, view in enumerate(views):
        grown = [b.num_tokens + (id(b) in pending) for b in view]
        spans = [b.mrope_span + (id(b) in pending) for b in view]
        rows = []
        for j, b in enumerate(view):
            if grown[j]:
                rows.append((slots_of(b, grown[j]), torch.tensor([sum(spans[j:]) - 1]), 1 << 40))
        if writers[w] not in view:
            rows.append((slots[w: w + 1].cpu().long(), torch.tensor([writers[w].mrope_span]), 1 << 40))
        segments.append(rows)
    positions = torch.tensor([b.mrope_span for b in writers], dtype=torch.int64, device=op.device)
    return SimpleNamespace(meta=meta, segments=segments, slots=slots, positions=positions, group=group, pending=pending)


def prefill_step(op, requests, three=False, buffers=None):
    """``requests``: ``(context blocks, own block with room, new)``."""
    from async_llm_amd.shared_cache import PrefillSpec

    specs, segments, slots, positions = [], [], [], []
    for context, own, new in requests:
        rel = torch.stack([torch.arange(new) // 3, torch.arange(new) % 5, torch.arange(new) // 2]) if three else None
        starts = torch.tensor(list(own.page_starts) + list(own.spare), dtype=torch.int32)
        starts = starts[: -(-(own.num_tokens + new) // op.page_size)]
        specs.append(PrefillSpec(context, starts, new, own.num_tokens, own.mrope_span, rel))
        rel = torch.arange(new) if rel is None else rel
        spans = [b.mrope_span for b in context] + [own.mrope_span]
        rows = [(slots_of(b), rel + sum(spans[j:]), 1 << 40) for j, b in enumerate(context)]
        rows.append((slots_of(own, own.num_tokens + new), rel + own.mrope_span, own.num_tokens))
        segments.append(rows)
        slots.append(slots_of(own, own.num_tokens + new)[own.num_tokens:])
        positions.append(rel + own.mrope_span)
    meta = op.prepare_prefill_batch(specs, **({} if buffers is None else {"graph_buffers": buffers}))
    return SimpleNamespace(meta=meta, segments=segments, specs=specs, slots=torch.cat(slots).to(op.device),
                           positions=torch.cat(positions, dim=-1).to(op.device), new=[n for _, _, n in requests])
