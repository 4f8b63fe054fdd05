"""The operators of an 8-bit key-value cache, as measurable cases.

A program that keeps its paged cache in 8 bits writes each step's keys and values into it
(``store``: the key rotated to its block-relative position, both quantised with a scale for every
token and kv head), attends to views of it (``attend``: one new token a request; ``chunk``: many
new tokens of a request, causal among themselves), reads rows of it back (``load``) and moves runs
of tokens to other slots, the keys rotated by a shift on the way (``merge``).

A row of one token and kv head is ``code * 2**e``: codes are float8 (e4m3) or int8, and ``e`` is the
smallest whole number for which the row's largest magnitude is at most 448 (127) times ``2**e``.
Codes lie as ``[layers, pages, kv heads, page size, head dim]``, scales as float8_e8m0 without the
last axis.  Rotations are by a 32-bit cos|sin table, or by angles that are the 32-bit products of
positions on three axes and 32-bit frequencies.

Ragged lengths come from a case's ``shape`` number, so that ``work`` knows them; values and the order
of pages come from the seed.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
SECTIONS = {64: (12, 10, 10), 128: (24, 20, 20)}  # by rotary width: pair dims of time, height and width


def _model(hq, hkv, d, dtype="bf16", codes="e4m3", rope="table", page=16):
    return dict(hq=hq, hkv=hkv, d=d, dtype=dtype, codes=codes, rope=rope, page=page)


def listed():
    wide, usual = (16, 4, 256), (32, 8, 128)
    return [
        # the new tokens of a full decode batch, some rows of it padding: the smallest write there is
        dict(name="store_step", kind="store", rows=64, shape=1, **_model(*wide)),
        # the new tokens of a prefill batch
        dict(name="store_chunk", kind="store", rows=4099, shape=2, **_model(*usual, "f16", "int8")),
        # one agent with a short view, float32 activations: the smallest step
        dict(name="attend_one", kind="attend", workers=1, shared=256, views=2, private_lo=512, private_hi=1024, shape=3,
             **_model(8, 2, 128, "f32", "int8")),
        # a few cooperating agents over one prompt and each other's notes
        dict(name="attend_agents", kind="attend", workers=4, shared=1500, views=3, private_lo=64, private_hi=2048,
             shape=4, **_model(*usual, "f16", "int8")),
        # a full decode batch over a long shared prompt
        dict(name="attend_batch", kind="attend", workers=64, shared=8192, views=3, private_lo=256, private_hi=8192,
             shape=5, **_model(*wide)),
        # eight long-context requests with images in their blocks
        dict(name="attend_long", kind="attend", workers=8, shared=0, views=8, private_lo=16384, private_hi=16384,
             shape=6, **_model(*wide, rope="mrope")),
        # one request takes in a tool result with an image
        dict(name="chunk_image", kind="chunk", requests=1, new_lo=333, new_hi=333, prefix_lo=100, prefix_hi=400,
             prompt=2048, views=2, private_lo=200, private_hi=1500, shape=7, **_model(*wide, rope="mrope")),
        # ragged writes of ordinary length over a long prompt and some blocks
        dict(name="chunk_ragged", kind="chunk", requests=4, new_lo=300, new_hi=1500, prefix_lo=0, prefix_hi=1000,
             prompt=8000, views=2, private_lo=50, private_hi=3000, shape=8, **_model(*usual)),
        # a short note is read back
        dict(name="load_note", kind="load", rows=717, shape=9, **_model(64, 16, 64, "f16", "int8")),
        # a whole view is read back
        dict(name="load_view", kind="load", rows=41237, shape=10, **_model(*wide)),
        # a short note is appended to another
        dict(name="merge_notes", kind="merge", rows=517, shift=203, layers=2, shape=11,
             **_model(64, 16, 64, "bf16", "int8")),
        # a block of odd length goes behind another in all of the layers
        dict(name="merge_blocks", kind="merge", rows=12556, shift=7001, layers=4, shape=12, **_model(*wide)),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _span(rng, lo, hi):
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return min(a, b), max(a, b)


def _draw_once(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "attend", "chunk", "chunk", "load", "merge"])
    hq, hkv, d = rng.choice([(16, 4, 256), (16, 4, 256), (32, 8, 128), (32, 8, 128), (8, 2, 128), (64, 16, 64)])
    rope, codes = rng.choice(["table", "table", "mrope"]), rng.choice(["e4m3", "e4m3", "int8"])
    if kind in ("store", "merge") and codes == "int8":
        rope = "table"  # whole codes have to be equal: no sines whose last bit is free
    case = dict(kind=kind, shape=rng.randrange(1 << 20),
                **_model(hq, hkv, d, rng.choice(["bf16", "bf16", "f16"]), codes, rope, rng.choice([16, 16, 16, 32, 64, 1])))
    if kind == "store":
        case.update(rows=_log(rng, 1, 16384))
    elif kind == "load":
        case.update(rows=_log(rng, 1, 65536))
    elif kind == "merge":
        case.update(rows=_log(rng, 1, 16384), shift=_log(rng, 1, 16384), layers=rng.choice([1, 2, 4]))
    elif kind == "attend":
        lo, hi = _span(rng, 64, 16384)
        case.update(workers=_log(rng, 1, 64), shared=_log(rng, 64, 8192), views=rng.randint(1, 4), private_lo=lo,
                    private_hi=hi)
        if rng.random() < 0.15:  # 32-bit activations: short steps
            case.update(dtype="f32", workers=min(case["workers"], 8), shared=min(case["shared"], 1024),
                        private_lo=min(lo, 1024), private_hi=min(hi, 1024))
    else:
        n, c, p = _span(rng, 2, 1500), _span(rng, 16, 3000), _span(rng, 1, 1000)
        case.update(requests=_log(rng, 1, 4), new_lo=n[0], new_hi=n[1], prefix_lo=p[0], prefix_hi=p[1],
                    prompt=_log(rng, 64, 8192), views=rng.randint(0, 2), private_lo=c[0], private_hi=c[1])
    return case


def draw(rng):
    limits = {c["kind"]: work(c) for c in listed()}  # the dearest listed case of each kind
    limits["attend"] = work(next(c for c in listed() if c["name"] == "attend_long"))
    while True:
        case = _draw_once(rng)
        w = work(case)
        if all(w[k] <= max(x[k] for x in limits.values()) for k in w) and w["flops"] <= limits["chunk"]["flops"]:
            return case


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
def _views(case):
    """What each request reads: ``[(block name, tokens)]`` in view order, and its new rows.  Its own block, which
    holds the new rows, comes last; block 0 is the one that all share."""
    r = random.Random(case["shape"])
    if case["kind"] == "attend":
        full = case["workers"] == 1 or case["views"] > 4
        out, name = [], 1
        for _ in range(case["workers"]):
            lengths = [r.randint(case["private_lo"], case["private_hi"])
                       for _ in range(case["views"] if full else r.randint(1, case["views"]))]
            lengths[-1] += 1  # the new token
            view = ([(0, case["shared"])] if case["shared"] else []) + [(name + i, n) for i, n in enumerate(lengths)]
            out.append((view, 1))
            name += len(lengths)
        return out
    out, name = [], 1
    for _ in range(case["requests"]):
        new, prefix = r.randint(case["new_lo"], case["new_hi"]), r.randint(case["prefix_lo"], case["prefix_hi"])
        lengths = [r.randint(case["private_lo"], case["private_hi"]) for _ in range(case["views"])] + [prefix + new]
        out.append(([(0, case["prompt"])] + [(name + i, n) for i, n in enumerate(lengths)], new))
        name += len(lengths)
    return out


def _blocks(case):
    """Tokens of every distinct block, by name."""
    return dict(b for view, _ in _views(case) for b in view)


def _seen(new, tokens):
    """(query row, key) pairs of a view."""
    return new * sum(tokens) - new * (new - 1) // 2


def work(case):
    """Codes and scales of every distinct token read (or written) once, activations once; 4 * D * Hq operations per
    visible (query row, key) pair."""
    row, width, size = case["hkv"] * 2 * (case["d"] + 1), case["hkv"] * 2 * case["d"], SIZES[case["dtype"]]
    if case["kind"] == "store":
        return {"bytes": case["rows"] * (width * size + row + 12), "flops": 0}
    if case["kind"] == "load":
        return {"bytes": case["rows"] * (width * size + row + 8), "flops": 0}
    if case["kind"] == "merge":
        return {"bytes": case["rows"] * (2 * case["layers"] * row + 16), "flops": 0}
    views, q = _views(case), case["hq"] * case["d"]
    rows = sum(new for _, new in views)
    return {"bytes": sum(_blocks(case).values()) * row + rows * (2 * q * size + 4 * case["hq"]),
            "flops": 4 * q * sum(_seen(new, [n for _, n in view]) for view, new in views)}


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------
def _power(e):
    """2**e in 32 bits, e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x, kind):
    """Codes and scales of the rows (last axis) of 32-bit ``x``."""
    part, power = torch.frexp(x.abs().amax(-1))
    edge, bits = (0.875, 9) if kind == "e4m3" else (0.9921875, 7)
    power = torch.where(part == 0, -126, (power - bits + (part > edge)).clamp(-126, 127))
    y = x * _power(-power)[..., None]
    codes = y.to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().to(torch.int8)
    return codes, (power + 127).to(torch.uint8)


def _values(codes, scales):
    """32-bit values of codes and scales (``uint8`` exponents)."""
    return codes.float() * _power(scales.int() - 127)[..., None]


def _pool(case, gen, pages, layers):
    """Codes ``[2, layers, pages, hkv, page, d]`` and exponents of a pool with content: keys with strong and weak
    channels, values whose size differs from token to token."""
    hkv, d, page, dev = case["hkv"], case["d"], case["page"], gen.device
    codes = torch.empty(2, layers, pages, hkv, page, d, dtype=CODES[case["codes"]], device=dev)
    scales = torch.empty(2, layers, pages, hkv, page, dtype=torch.uint8, device=dev)
    gain = torch.exp(0.5 * torch.randn(hkv, 1, d, device=dev, generator=gen))
    step = max(1, (1 << 27) // (hkv * page * d))
    for layer in range(layers):
        for at in range(0, pages, step):
            n = min(step, pages - at)
            k = torch.randn(n, hkv, page, d, device=dev, generator=gen) * gain
            v = torch.randn(n, hkv, page, d, device=dev, generator=gen)
            v *= torch.exp(0.5 * torch.randn(n, hkv, page, 1, device=dev, generator=gen))
            for which, x in enumerate((k, v)):
                c, e = _quantised(x, case["codes"])
                codes[which, layer, at: at + n], scales[which, layer, at: at + n] = c, e
    return codes, scales


def _rotation(case, dev, positions):
    """What the op's constructor takes: the cos|sin table for positions below ``positions``, or frequencies."""
    rotary = case["d"] if case["rope"] == "table" else min(case["d"], 128)
    inv = 1.0 / (1e7 ** (torch.arange(0, rotary, 2, dtype=torch.float32, device=dev) / rotary))
    if case["rope"] == "mrope":
        pair = torch.arange(rotary // 2, device=dev)
        _, h, w = SECTIONS[rotary]
        axis = torch.where((pair % 3 == 1) & (pair < 3 * h), 1, torch.where((pair % 3 == 2) & (pair < 3 * w), 2, 0))
        return dict(rotary=rotary, inv=inv, axis=axis, table=None)
    angle = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * inv.double()
    return dict(rotary=rotary, inv=None, axis=None, table=torch.cat([angle.cos(), angle.sin()], dim=1).float())


def _span_of(case, tokens):
    """How far positions move over a block: an image of a quarter of it moves them by its side only."""
    if case["rope"] == "table" or tokens < 16:
        return tokens
    side = math.isqrt(tokens // 4)
    return tokens - side * side + side


def _image_positions(new):
    """Positions of text, one image of a quarter of the tokens, text, in three axes."""
    side = math.isqrt(new // 4)
    lead = (new - side * side) // 2
    square = torch.arange(side * side)
    grid = torch.stack([0 * square, square // max(1, side), square % max(1, side)]) + lead
    tail = torch.arange(new - lead - side * side) + lead + side
    return torch.cat([torch.arange(lead).expand(3, -1), grid, tail.expand(3, -1)], dim=1)


def _handles(s):
    """The cache and the op that a program builds once."""
    from async_llm_amd.kvcache import QuantizedKVCache
    from async_llm_amd.shared_cache import QuantizedCacheAttention

    c, r = s.case, s.rope
    s.cache = QuantizedKVCache.from_buffers(s.codes, s.scales, s.dtype)
    more = dict(rotary_dim=r["rotary"])
    if r["table"] is None:
        more.update(mrope_section=SECTIONS[r["rotary"]], rope_base=1e7)
    table = r["table"] if r["table"] is not None else torch.zeros(1, r["rotary"], device=s.dev)
    s.op = QuantizedCacheAttention(s.cache, table, c["hq"], c["hkv"], c["d"], c["page"], s.dtype, s.dev, **more)


def prepare(case, seed):
    s = SimpleNamespace(case=case, dev=torch.device("cuda"), dtype=DTYPES[case["dtype"]])
    s.gen = torch.Generator(device=s.dev).manual_seed(seed)
    if case["kind"] in ("attend", "chunk"):
        _prepare_views(s)
    else:
        _prepare_rows(s)
    if own:
        _handles(s)
        if case["kind"] in ("attend", "chunk"):
            _plan(s)
    return s


def _prepare_rows(s):
    c = s.case
    n, page = c["rows"], c["page"]
    half = -(-n // page) + 1
    pages = half * (2 if c["kind"] == "merge" else 1)
    s.codes, s.scales = _pool(c, s.gen, pages, c.get("layers", 1))
    s.rope = _rotation(c, s.dev, n + c.get("shift", 0) + 64)
    order = torch.randperm(pages, device=s.dev, generator=s.gen)
    slots = (order[:, None] * page + torch.arange(page, device=s.dev)).reshape(-1)  # runs of scattered pages
    if c["kind"] == "merge":
        s.source, s.shift = slots[:n].contiguous(), c["shift"]
        s.target = slots[half * page + 1: half * page + 1 + n].contiguous()  # behind a token that is there
    elif c["kind"] == "load":
        s.slots = slots[:n].contiguous()
    else:
        width, hkv = (c["hq"] + 2 * c["hkv"]) * c["d"], c["hkv"] * c["d"]
        qkv = torch.randn(n, width, device=s.dev, generator=s.gen)  # the fused projection that k and v are slices of
        qkv = (qkv * torch.exp(0.5 * torch.randn(width, device=s.dev, generator=s.gen))).to(s.dtype)
        s.k, s.v = qkv[:, -2 * hkv: -hkv], qkv[:, -hkv:]
        out_loc = slots[:n].to(torch.int32)
        out_loc[12::13] = -1  # rows of padding
        positions = torch.arange(n, device=s.dev)
        mrope = _image_positions(n).to(s.dev).contiguous() if c["rope"] == "mrope" else None
        s.batch = SimpleNamespace(attn_metadata=None, positions=positions, mrope_positions=mrope, out_loc=out_loc)


def _prepare_views(s):
    c, page, dev = s.case, s.case["page"], s.dev
    s.views, s.tokens = _views(c), _blocks(c)
    pages = sum(-(-n // page) for n in s.tokens.values())
    s.codes, s.scales = _pool(c, s.gen, pages, 1)
    order = torch.randperm(pages, device=dev, generator=s.gen)
    s.pages, at = {}, 0  # pages of every block, in its order
    for name, n in s.tokens.items():
        s.pages[name] = order[at: at + -(-n // page)]
        at += -(-n // page)
    s.new = [new for _, new in s.views]
    depth, rows, width = max(len(view) for view, _ in s.views), max(s.new), c["hq"] * c["d"]
    # the distance of every query row from the start of every block of its view
    s.rel = []
    starts = torch.zeros(depth, len(s.views), dtype=torch.int64)
    for r, (view, new) in enumerate(s.views):
        three = c["rope"] == "mrope" and c["kind"] == "chunk"
        s.rel.append(_image_positions(new) if three else torch.arange(new))
        held = view[-1][1] - new  # tokens of its own block before this step
        spans = [_span_of(c, n) for _, n in view[:-1]] + [_span_of(c, held)]
        for j in range(len(view)):
            starts[j, r] = sum(spans[j:])
    axes = s.rel[0].dim() == 2
    s.where = torch.zeros((3,) * axes + (depth, len(s.views), rows), dtype=torch.int64)
    for r, rel in enumerate(s.rel):
        s.where[..., r, : s.new[r]] = rel.unsqueeze(-2) + starts[:, r, None]
    s.starts, s.where = starts, s.where.to(dev)
    s.rope = _rotation(c, dev, int(starts.max()) + rows + 64)
    s.q = torch.randn(sum(s.new), width, device=dev, generator=s.gen).to(s.dtype)
    # the same tables padded, for the plain form: slots, lengths and the first row's last visible token
    base = torch.arange(page, device=dev)
    s.index, s.length, s.causal = [], [], []
    for j in range(depth):
        index = torch.zeros(len(s.views), max(view[j][1] if j < len(view) else 1 for view, _ in s.views), dtype=torch.int64, device=dev)
        length, causal = torch.zeros(2, len(s.views), dtype=torch.int64)
        for r, (view, new) in enumerate(s.views):
            if j < len(view):
                name, n = view[j]
                index[r, :n] = (s.pages[name][:, None] * page + base).reshape(-1)[:n]
                length[r], causal[r] = n, n - new if j == len(view) - 1 else n
        s.index.append(index)
        s.length.append(length.to(dev))
        s.causal.append(causal.to(dev))
    place = torch.zeros(len(s.views), rows, dtype=torch.int64)
    firsts = [sum(s.new[:r]) for r in range(len(s.new))]
    for r, n in enumerate(s.new):
        place[r, :n] = firsts[r] + torch.arange(n)
    s.place = place.to(dev)
    s.valid = (torch.arange(rows)[None, :] < torch.tensor(s.new)[:, None]).to(dev)


def _plan(s):
    """The plan of the step, made once for all of its layers."""
    from async_llm_amd.shared_cache import CacheBlock, PrefillSpec, WorkerGroup

    c, page = s.case, s.case["page"]
    starts = {name: [int(p) * page for p in pages.tolist()] for name, pages in s.pages.items()}
    blocks, opened = {}, {}
    for view, new in s.views:
        for at, (name, n) in enumerate(view):
            if name in blocks:
                continue
            b = blocks[name] = CacheBlock(s.dev, page)
            b.num_tokens = n - new if at == len(view) - 1 else n
            held = -(-b.num_tokens // page)
            b.page_starts = starts[name][:held]
            b.mrope_span_override = _span_of(c, b.num_tokens)
            opened[name] = starts[name][held] if held < len(starts[name]) else None
    if c["kind"] == "attend":
        group = WorkerGroup(cache_structure=[[blocks[name] for name, _ in view] for view, _ in s.views])
        pending = {id(blocks[view[-1][0]]): opened[view[-1][0]] for view, _ in s.views}
        slots = torch.tensor([starts[view[-1][0]][(view[-1][1] - 1) // page] + (view[-1][1] - 1) % page
                              for view, _ in s.views], dtype=torch.int32, device=s.dev)
        s.meta = s.op.prepare(group, pending, slots)
        return
    specs = []
    for r, (view, new) in enumerate(s.views):
        name = view[-1][0]
        specs.append(PrefillSpec([blocks[b] for b, _ in view[:-1]], torch.tensor(starts[name], dtype=torch.int32), new,
                                 blocks[name].num_tokens, blocks[name].mrope_span,
                                 s.rel[r] if s.rel[r].dim() == 2 else None))
    s.meta = s.op.prepare_prefill_batch(specs)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return {"store": _run_store, "load": _run_load, "merge": _run_merge, "attend": _run_views,
            "chunk": _run_views}[s.case["kind"]](s)


def _turns(rope, where):
    """32-bit cosines and sines ``[..., pairs]`` of whole positions: ``[...]``, or ``[3, ...]`` for three axes."""
    if rope["table"] is not None:
        rows = rope["table"][where.abs().clamp(max=rope["table"].shape[0] - 1)]
        cos, sin = rows.chunk(2, dim=-1)
        return cos, torch.where(where[..., None] < 0, -sin, sin)
    angle = (where.float().movedim(0, -1)[..., rope["axis"]] * rope["inv"]).double()
    return angle.cos().float(), angle.sin().float()


def _turned(x, cos, sin):
    """32-bit ``x [..., d]`` rotated: pairs are dims i and i + pairs, the rest passes through."""
    pairs = cos.shape[-1]
    a, b = x[..., :pairs], x[..., pairs: 2 * pairs]
    return torch.cat([cos * a - sin * b, cos * b + sin * a, x[..., 2 * pairs:]], dim=-1)


def _rows_of(s, slots):
    """Pages and places of slots, as the pool is indexed."""
    return slots // s.case["page"], slots % s.case["page"]


def _pools(s):
    return {"codes": s.codes, "scales": s.scales.view(torch.float8_e8m0fnu)}


def _run_store(s):
    c, b = s.case, s.batch
    if own:
        s.op.store_new_kv(s.k, s.v, 0, b)
        return _pools(s)
    live = b.out_loc >= 0
    page, place = _rows_of(s, b.out_loc[live].long())
    shape = (-1, c["hkv"], c["d"])
    where = b.positions if b.mrope_positions is None else b.mrope_positions
    cos, sin = _turns(s.rope, where[..., live])
    k = _turned(s.k[live].float().reshape(shape), cos[:, None], sin[:, None])
    for which, x in enumerate((k, s.v[live].float().reshape(shape))):
        codes, scales = _quantised(x, c["codes"])
        s.codes[which, 0].view(torch.uint8)[page, :, place] = codes.view(torch.uint8)
        s.scales[which, 0][page, :, place] = scales
    return _pools(s)


def _run_load(s):
    if own:
        k, v = s.cache.load_kv(s.slots, 0)
        return {"k": k, "v": v}
    page, place = _rows_of(s, s.slots)
    k, v = (_values(s.codes[w, 0].view(torch.uint8)[page, :, place].view(s.codes.dtype), s.scales[w, 0][page, :, place]).to(s.dtype)
            for w in (0, 1))
    return {"k": k, "v": v}


def _run_merge(s):
    if own:
        s.op.copy_shifted(s.source, s.target, s.shift)
        return _pools(s)
    page, place = _rows_of(s, s.source)
    to_page, to_place = _rows_of(s, s.target)
    raw = s.codes.view(torch.uint8)
    codes, scales = raw[:, :, page, :, place], s.scales[:, :, page, :, place]  # [rows, 2, layers, hkv, d]
    k = _values(codes[:, 0].contiguous().view(s.codes.dtype), scales[:, 0])
    at = torch.tensor(s.shift, device=s.dev)
    cos, sin = _turns(s.rope, at if s.rope["table"] is not None else at.expand(3))
    turned, e = _quantised(_turned(k, cos, sin), s.case["codes"])
    raw[:, :, to_page, :, to_place] = torch.stack([turned.view(torch.uint8), codes[:, 1]], dim=1)
    s.scales[:, :, to_page, :, to_place] = torch.stack([e, scales[:, 1]], dim=1)
    return _pools(s)


def _run_views(s):
    c = s.case
    if own:
        if c["kind"] == "attend":
            out, lse = s.op.attend(s.q, 0, s.meta, return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": s.op.attend(s.q, 0, s.meta)}
    hkv, g, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    keys, values = (_values(s.codes[w, 0], s.scales[w, 0]).transpose(1, 2).reshape(-1, hkv, d) for w in (0, 1))
    q = s.q[s.place].float().view(*s.place.shape, hkv, g, d)  # [requests, rows, hkv, g, d]
    row = torch.arange(q.shape[1], device=s.dev)
    scores = []
    for j, index in enumerate(s.index):  # the blocks of a view, one after the other
        where = s.where[..., j, :, :]
        if s.rope["axis"] is not None and where.dim() == 2:
            where = where.expand(3, -1, -1)
        cos, sin = _turns(s.rope, where)
        turned = _turned(q, cos[:, :, None, None], sin[:, :, None, None]).permute(0, 2, 1, 3, 4).reshape(len(s.new), hkv, -1, d)
        x = torch.matmul(turned, keys[index].permute(0, 2, 3, 1).contiguous()) * d ** -0.5
        x = x.view(len(s.new), hkv, q.shape[1], g, -1)
        t = torch.arange(index.shape[1], device=s.dev)
        seen = (t < s.length[j][:, None])[:, None, :] & (t <= (s.causal[j][:, None] + row)[..., None])
        scores.append(x.masked_fill(~seen[:, None, :, None, :], -math.inf))
    top = torch.stack([x.amax(-1) for x in scores]).amax(0)
    weights = [torch.exp(x - top[..., None]) for x in scores]
    total = sum(w.sum(-1) for w in weights)
    out = sum(torch.matmul(w.view(len(s.new), hkv, -1, w.shape[-1]), values[index].permute(0, 2, 1, 3).contiguous())
              for w, index in zip(weights, s.index))
    out = out.view(len(s.new), hkv, q.shape[1], g, d) / total[..., None]
    out = out.permute(0, 2, 1, 3, 4)[s.valid].reshape(-1, c["hq"] * d).to(s.dtype)
    if c["kind"] == "chunk":
        return {"out": out}
    return {"out": out, "lse": (top + total.log()).permute(0, 2, 1, 3)[s.valid].reshape(-1, c["hq"])}


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(s, which, layer, slots):
    """``[n, hkv, d]``"""
    page, place = slots // s.case["page"], slots % s.case["page"]
    codes = s.codes[which, layer].view(torch.uint8)[page, :, place].view(s.codes.dtype).double()
    return codes * torch.pow(2.0, s.scales[which, layer][page, :, place].double() - 127)[..., None]


def _exact_turn(s, x, where):
    """``x [n, heads, d]`` as complex pairs times the turns of ``where [n]`` or ``[3, n]``."""
    r = s.rope
    if r["table"] is not None:
        entry = r["table"][where].double()
        unit = torch.complex(entry[:, : entry.shape[1] // 2], entry[:, entry.shape[1] // 2:])
    else:
        where = where if where.dim() == 2 else torch.stack([where] * 3)
        product = where.float()[r["axis"]] * r["inv"][:, None]  # angles are 32-bit products by definition
        unit = torch.polar(torch.ones_like(product, dtype=torch.float64), product.double()).T
    h = unit.shape[1]
    z = torch.complex(x[..., :h].contiguous(), x[..., h: 2 * h].contiguous()) * unit[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * h:]], dim=-1)


def _exact_codes(s, x):
    part, power = torch.frexp(x.abs().amax(-1) / LARGEST[s.case["codes"]])
    power = torch.where(part == 0.5, power - 1, power).clamp(min=-126).double()
    y = x / torch.pow(2.0, power)[..., None]
    if s.case["codes"] == "int8":
        return torch.round(y), torch.pow(2.0, power)
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, torch.pow(2.0, power)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "load":
        return {"k": _exact_values(s, 0, 0, s.slots), "v": _exact_values(s, 1, 0, s.slots)}
    if case["kind"] in ("store", "merge"):
        codes, scales = s.codes.float().double(), torch.pow(2.0, s.scales.double() - 127)
        for layer in range(case.get("layers", 1)):
            if case["kind"] == "store":
                live = torch.nonzero(s.batch.out_loc >= 0)[:, 0]
                slots, shape = s.batch.out_loc[live].long(), (len(live), case["hkv"], case["d"])
                where = s.batch.positions if s.batch.mrope_positions is None else s.batch.mrope_positions
                rows = [_exact_codes(s, _exact_turn(s, s.k[live].double().reshape(shape), where[..., live])),
                        _exact_codes(s, s.v[live].double().reshape(shape))]
            else:
                slots = s.target
                where = torch.full_like(s.source, s.shift)
                rows = [_exact_codes(s, _exact_turn(s, _exact_values(s, 0, layer, s.source), where))]
                page, place = s.source // case["page"], s.source % case["page"]
                rows.append((codes[1, layer][page, :, place], scales[1, layer][page, :, place]))
            for which, (c, e) in enumerate(rows):
                codes[which, layer][slots // case["page"], :, slots % case["page"]] = c
                scales[which, layer][slots // case["page"], :, slots % case["page"]] = e
        return {"codes": codes if case["codes"] == "e4m3" else None, "scales": scales}
    g, outs, sums, first = case["hq"] // case["hkv"], [], [], 0
    for r, (view, new) in enumerate(s.views):
        q = s.q[first: first + new].double().view(new, case["hq"], case["d"])
        first += new
        scores, values = [], []
        for j, (name, n) in enumerate(view):
            slots = (s.pages[name][:, None] * case["page"] + torch.arange(case["page"], device=s.dev)).reshape(-1)[:n]
            k, v = _exact_values(s, 0, 0, slots), _exact_values(s, 1, 0, slots)
            turned = _exact_turn(s, q, s.rel[r].to(s.dev) + int(s.starts[j, r]))
            turned = turned.view(new, case["hkv"], g, case["d"]).transpose(0, 1).reshape(case["hkv"], new * g, case["d"])
            x = torch.bmm(turned.contiguous(), k.permute(1, 2, 0).contiguous()).view(case["hkv"], new, g, n) / math.sqrt(case["d"])
            if j == len(view) - 1:
                ahead = torch.arange(n, device=s.dev) - (n - new) > torch.arange(new, device=s.dev)[:, None]
                x.masked_fill_(ahead[None, :, None], -math.inf)
            scores.append(x)
            values.append(v)
        x = torch.cat(scores, dim=-1)
        lse = torch.logsumexp(x, dim=-1)  # [hkv, new, g]
        p = torch.exp(x - lse[..., None]).view(case["hkv"], new * g, -1)
        o = torch.bmm(p, torch.cat(values).permute(1, 0, 2).contiguous()).view(case["hkv"], new, g, case["d"])
        outs.append(o.transpose(0, 1).reshape(new, -1))
        sums.append(lse.transpose(0, 1).reshape(new, -1))
    return {"out": torch.cat(outs)} if case["kind"] == "chunk" else {"out": torch.cat(outs), "lse": torch.cat(sums)}
