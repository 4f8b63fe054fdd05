"""The operators that let a cache outlive its room, as measurable cases.

A program whose views outgrow its pool keeps count of what attention looks at, drops the tokens that
nobody looks at and moves the others together.  Its layers add the weight that a step's queries gave
to every cached token (``weigh``); from those sums it chooses what stays of a block (``select``) and
moves that to other slots, keys turned to the positions they have there (``move``).  What makes
positions in the first place, in models of either layout and of scaled frequencies, is ``rotate``.

* ``weigh``: ``w[hk, t] += sum over the rows and q heads of hk that see token t of
  exp(q_turned . k_t / sqrt(d) - lse)``, the log-sum of each row and head given; a query is turned by its
  distance from the start of the block that holds the token.  Many new tokens of a request see each
  other causally, and only the last ``window`` of them are counted where that is not 0.
* ``select``: of each block of n tokens the first and the last few stay, and of the others the
  heaviest (weights summed over kv heads, ties to the lower position) until ``keep`` are together.
  Results are positions, in rising order, and slots.
* ``move``: rows of K, V and weights to other slots in all layers, keys turned by
  ``new position - old position``.
* ``rotate``: q and k of a step, slices of a fused projection, rotated by position; pairs are (i, i + h)
  or (2 i, 2 i + 1), over the head or its first part.

Pools are ``[pages, page size, kv heads, head dim]`` in 16 or 32 bits, or codes ``[pages, kv heads, page size,
head dim]`` with a scale ``2**e`` for each row.  Ragged lengths come from a case's ``shape`` number, so that
``work`` knows them; values, positions and the order of pages come from the seed.
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
SECTIONS = {64: (12, 10, 10), 128: (24, 20, 20)}  # by rotary width: pair dims of time, height and width
SCALINGS = {
    "none": None,
    "linear": dict(rope_type="linear", factor=4.0),
    "llama3": dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192),
    "yarn": dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
}


def _model(hq, hkv, d, dtype="bf16", codes="", rope="table", page=16):
    return dict(hq=hq, hkv=hkv, d=d, dtype=dtype, codes=codes, rope=rope, page=page)


def listed():
    wide, usual = (16, 4, 256), (32, 8, 128)
    return [
        # the queries and keys of a full decode batch, a quarter of each head rotated: the smallest rotation
        dict(name="rotate_step", kind="rotate", rows=64, hq=16, hkv=4, d=256, dtype="bf16", rotary=64, layout="half",
             scaling="none", far=131072, run=False),
        # a prefill batch of odd length at the far end of a long context, neighbouring pairs
        dict(name="rotate_chunk", kind="rotate", rows=4099, hq=32, hkv=8, d=128, dtype="f16", rotary=128, layout="pairs",
             scaling="llama3", far=1000003, run=True),
        # many small heads in 32 bits, frequencies scaled by parts
        dict(name="rotate_wide", kind="rotate", rows=16384, hq=64, hkv=16, d=64, dtype="f32", rotary=64, layout="half",
             scaling="yarn", far=131072, run=True),
        # one agent with a short view, 32-bit activations: the smallest step that is weighed
        dict(name="weigh_one", kind="weigh", workers=1, shared=256, views=2, private_lo=512, private_hi=1024, window=0,
             shape=1, **_model(8, 2, 128, "f32")),
        # a few cooperating agents over one prompt and each other's notes, cached in 8 bits
        dict(name="weigh_agents", kind="weigh", workers=4, shared=1500, views=3, private_lo=64, private_hi=2048, window=0,
             shape=2, **_model(*usual, "f16", "e4m3")),
        # a full decode batch over a long shared prompt
        dict(name="weigh_batch", kind="weigh", workers=64, shared=8192, views=3, private_lo=256, private_hi=8192,
             window=0, shape=3, **_model(*wide)),
        # eight long-context requests with images in their blocks
        dict(name="weigh_long", kind="weigh", workers=8, shared=0, views=8, private_lo=16384, private_hi=16384, window=0,
             shape=4, **_model(*wide, rope="mrope")),
        # ragged writes of ordinary length over a long prompt and some blocks, every new token counted
        dict(name="weigh_chunk", kind="weigh_chunk", requests=4, new_lo=300, new_hi=1500, prefix_lo=0, prefix_hi=1000,
             prompt=8000, views=2, private_lo=50, private_hi=3000, window=0, shape=5, **_model(*usual)),
        # one short note loses half of its tokens
        dict(name="select_note", kind="select", blocks=1, lo=1500, hi=1500, hkv=8, keep=50, first=4, last=64, page=16,
             shape=6),
        # long contexts are cut to an eighth
        dict(name="select_long", kind="select", blocks=8, lo=60000, hi=131072, hkv=4, keep=12, first=4, last=256, page=16,
             shape=7),
        # what is left of a short note moves together
        dict(name="move_note", kind="move", rows=517, of=1100, layers=2, shape=8, **_model(64, 16, 64, "f16")),
        # what is left of a long block moves together in all of the layers
        dict(name="move_block", kind="move", rows=12556, of=40000, layers=4, shape=9, **_model(*wide)),
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
    kind = rng.choice(["rotate", "rotate", "weigh", "weigh", "weigh", "weigh_chunk", "weigh_chunk", "select", "move"])
    hq, hkv, d = rng.choice([(16, 4, 256), (16, 4, 256), (32, 8, 128), (32, 8, 128), (8, 2, 128), (64, 16, 64)])
    if kind == "rotate":
        return dict(kind=kind, rows=_log(rng, 1, 16384), hq=hq, hkv=hkv, d=d, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    rotary=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["half", "pairs"]),
                    scaling=rng.choice(list(SCALINGS)), far=_log(rng, 20000, 4000000), run=rng.random() < 0.5)
    if kind == "select":
        lo, hi = _span(rng, 1, 131072)
        return dict(kind=kind, blocks=_log(rng, 1, 64), lo=lo, hi=hi, hkv=hkv, keep=rng.randint(1, 99),
                    first=rng.choice([0, 1, 4]), last=_log(rng, 1, 512), page=16, shape=rng.randrange(1 << 20))
    codes = rng.choice(["", "", "", "e4m3", "int8"])
    rope = "table" if kind == "move" else rng.choice(["table", "table", "mrope"])
    case = dict(kind=kind, shape=rng.randrange(1 << 20),
                **_model(hq, hkv, d, rng.choice(["bf16", "bf16", "f16"]), codes, rope, rng.choice([16, 16, 16, 32, 64, 1])))
    if kind == "move":
        rows = _log(rng, 1, 16384)
        case.update(rows=rows, of=rows + _log(rng, 1, 32768), layers=rng.choice([1, 2, 4]))
    elif kind == "weigh":
        lo, hi = _span(rng, 64, 16384)
        case.update(workers=_log(rng, 1, 64), shared=_log(rng, 64, 8192), views=rng.randint(1, 4), private_lo=lo,
                    private_hi=hi, window=0)
        if rng.random() < 0.15:  # 32-bit activations: short steps
            case.update(dtype="f32", codes="", workers=min(case["workers"], 8), shared=min(case["shared"], 1024),
                        private_lo=min(lo, 1024), private_hi=min(hi, 1024))
    else:
        n, c, p = _span(rng, 2, 1500), _span(rng, 16, 3000), _span(rng, 1, 1000)
        case.update(requests=_log(rng, 1, 4), new_lo=n[0], new_hi=n[1], prefix_lo=p[0], prefix_hi=p[1],
                    prompt=_log(rng, 64, 8192), views=rng.randint(0, 2), private_lo=c[0], private_hi=c[1],
                    window=rng.choice([0, 0, 32, 64]))
    return case


def draw(rng):
    most = {}  # of each kind of pass, the dearest listed one
    for c in listed():
        for k, v in work(c).items():
            most[c["kind"], k] = max(v, most.get((c["kind"], k), 0))
    while True:
        case = _draw_once(rng)
        if all(v <= most[case["kind"], k] for k, v in work(case).items()):
            return case


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
def _views(case):
    """What each request reads: ``[(block name, tokens)]`` in view order, and its new rows.  Its own block, which
    holds the new rows, comes last; block 0 is the one that all share."""
    r = random.Random(case["shape"])
    out, name = [], 1
    if case["kind"] == "weigh":
        full = case["workers"] == 1 or case["views"] > 4
        for _ in range(case["workers"]):
            lengths = [r.randint(case["private_lo"], case["private_hi"])
                       for _ in range(case["views"] if full else r.randint(1, case["views"]))]
            lengths[-1] += 1  # the new token
            view = ([(0, case["shared"])] if case["shared"] else []) + [(name + i, n) for i, n in enumerate(lengths)]
            out.append((view, 1))
            name += len(lengths)
        return out
    for _ in range(case["requests"]):
        new, prefix = r.randint(case["new_lo"], case["new_hi"]), r.randint(case["prefix_lo"], case["prefix_hi"])
        lengths = [r.randint(case["private_lo"], case["private_hi"]) for _ in range(case["views"])] + [prefix + new]
        out.append(([(0, case["prompt"])] + [(name + i, n) for i, n in enumerate(lengths)], new))
        name += len(lengths)
    return out


def _blocks(case):
    """Tokens of every distinct block, by name."""
    return dict(b for view, _ in _views(case) for b in view)


def _counted(case, new):
    """Rows of a request that are counted: its last ones."""
    return min(new, case["window"]) if case["window"] else new


def _lengths(case):
    r = random.Random(case["shape"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["blocks"])]


def _kept(case, n):
    """Tokens that stay of a block of n."""
    return max(1, n * case["keep"] // 100)


def work(case):
    """Each operand once: keys of every distinct token, queries and log-sums, weights read and written; 2 * d * hq operations
    per counted (query row, key) pair."""
    if case["kind"] == "rotate":
        return {"bytes": case["rows"] * ((case["hq"] + case["hkv"]) * case["d"] * 2 * SIZES[case["dtype"]] + 8), "flops": 0}
    if case["kind"] == "select":
        lengths = _lengths(case)
        return {"bytes": sum(n * (4 * case["hkv"] + 8) + 16 * _kept(case, n) for n in lengths), "flops": 0}
    size = SIZES[case["dtype"]]
    row = case["d"] + 1 if case["codes"] else case["d"] * size  # of a token and kv head, keys alone
    if case["kind"] == "move":
        return {"bytes": case["rows"] * (4 * case["layers"] * case["hkv"] * row + 8 * case["hkv"] + 24), "flops": 0}
    views, q = _views(case), case["hq"] * case["d"]
    rows = sum(_counted(case, new) for _, new in views)
    pairs = 0
    for view, new in views:
        c = _counted(case, new)
        pairs += c * sum(n for _, n in view) - c * (c - 1) // 2
    return {"bytes": sum(_blocks(case).values()) * case["hkv"] * (row + 8) + rows * (q * size + 4 * case["hq"]),
            "flops": 2 * q * pairs}


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------
def _power(e):
    """2**e in 32 bits, e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x, kind):
    """Codes and scales of the rows (last axis) of 32-bit ``x``: the smallest power of two that holds a row's largest magnitude
    as 448 (127)."""
    part, power = torch.frexp(x.abs().amax(-1))
    edge, bits = (0.875, 9) if kind == "e4m3" else (0.9921875, 7)
    power = torch.where(part == 0, -126, (power - bits + (part > edge)).clamp(-126, 127))
    y = x * _power(-power)[..., None]
    codes = y.to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().to(torch.int8)
    return codes, (power + 127).to(torch.uint8)


def _values(codes, scales):
    """32-bit values of codes and scales (``uint8`` exponents)."""
    return codes.float() * _power(scales.int() - 127)[..., None]


def _fill(case, gen, kv, pages):
    """One layer's K or V: keys with strong and weak channels, values whose size differs from token to token.  Rows as the pool
    holds them, or codes and scales."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    coded = bool(case["codes"])
    shape = (pages, hkv, page, d) if coded else (pages, page, hkv, d)
    out = torch.empty(shape, dtype=CODES[case["codes"]] if coded else DTYPES[case["dtype"]], device=gen.device)
    scales = torch.empty(shape[:-1], dtype=torch.uint8, device=gen.device) if coded else None
    gain = torch.exp(0.5 * torch.randn(hkv, d, device=gen.device, generator=gen))
    step = max(1, (1 << 27) // (hkv * page * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn(n, page, hkv, d, device=gen.device, generator=gen)
        x *= gain if kv == 0 else torch.exp(0.5 * torch.randn(n, page, hkv, 1, device=gen.device, generator=gen))
        if coded:
            out[at: at + n], scales[at: at + n] = _quantised(x.transpose(1, 2), case["codes"])
        else:
            out[at: at + n] = x
    return out, scales


def _pool(s, pages, layers, values=True):
    """The pool with content: ``s.kv [2, layers, ...]`` and ``s.scales``, or only the keys' half filled."""
    c = s.case
    coded = bool(c["codes"])
    shape = (pages, c["hkv"], c["page"], c["d"]) if coded else (pages, c["page"], c["hkv"], c["d"])
    if own and not coded:
        from async_llm_amd.kvcache import MHAKVCache

        s.cache = MHAKVCache(c["hkv"], layers, c["d"], pages, c["page"], s.dtype, s.dev)
        s.kv = [[s.cache.k_cache(i) for i in range(layers)], [s.cache.v_cache(i) for i in range(layers)]]
    else:
        kind = CODES[c["codes"]] if coded else s.dtype
        s.kv = torch.zeros(2, layers, *shape, dtype=torch.uint8 if coded else kind, device=s.dev).view(kind)
    s.scales = torch.full((2, layers, *shape[:-1]), 127, dtype=torch.uint8, device=s.dev) if coded else None
    for kv in range(2 if values else 1):
        for layer in range(layers):
            x, e = _fill(c, s.gen, kv, pages)
            s.kv[kv][layer].copy_(x)
            if coded:
                s.scales[kv, layer] = e
    s.num_slots = pages * c["page"]


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
    """The op over the pool and what evicts from it, built once."""
    from async_llm_amd.kvcache import QuantizedKVCache
    from async_llm_amd.shared_cache import CacheEviction, QuantizedCacheAttention, SharedCacheAttention

    c, r = s.case, s.rope
    more = dict(rotary_dim=r["rotary"])
    if r["table"] is None:
        more.update(mrope_section=SECTIONS[r["rotary"]], rope_base=1e7)
    table = r["table"] if r["table"] is not None else torch.zeros(1, r["rotary"], device=s.dev)
    kind = SharedCacheAttention
    if c["codes"]:
        kind, s.cache = QuantizedCacheAttention, QuantizedKVCache.from_buffers(s.kv, s.scales, s.dtype)
    s.op = kind(s.cache, table, c["hq"], c["hkv"], c["d"], c["page"], s.dtype, s.dev, **more)
    s.eviction = CacheEviction(s.op)


def prepare(case, seed):
    s = SimpleNamespace(case=case, dev=torch.device("cuda"), dtype=DTYPES.get(case.get("dtype")))
    s.gen = torch.Generator(device=s.dev).manual_seed(seed)
    {"rotate": _prepare_rotate, "select": _prepare_select, "move": _prepare_move, "weigh": _prepare_views,
     "weigh_chunk": _prepare_views}[case["kind"]](s)
    return s


def _frequencies(case):
    """64-bit frequencies of the pairs, and the factor on cosines and sines."""
    base, spec = 1e6, SCALINGS[case["scaling"]]
    f = 1.0 / base ** (torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
    if spec is None:
        return f, 1.0
    factor = spec["factor"]
    if case["scaling"] == "linear":
        return f / factor, 1.0
    original = spec["original_max_position_embeddings"]
    if case["scaling"] == "llama3":  # long waves are stretched, short ones stay, in between a blend
        turns = original * f / (2 * math.pi)
        blend = ((turns - spec["low_freq_factor"]) / (spec["high_freq_factor"] - spec["low_freq_factor"])).clamp(0, 1)
        return f / factor * (1 - blend) + f * blend, 1.0
    # by the number of turns within the original length: 32 and more stay, one and fewer are stretched
    at = lambda turns: case["rotary"] * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), case["rotary"] - 1)
    ramp = ((torch.arange(len(f), dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1


def _prepare_rotate(s):
    c = s.case
    n, q, k = c["rows"], c["hq"] * c["d"], c["hkv"] * c["d"]
    qkv = torch.randn(n, q + 2 * k, device=s.dev, generator=s.gen)  # the fused projection that q and k are slices of
    qkv = (qkv * torch.exp(0.5 * torch.randn(q + 2 * k, device=s.dev, generator=s.gen))).to(s.dtype)
    s.q, s.k = qkv[:, :q], qkv[:, q: q + k]
    if c["run"]:
        s.positions = torch.arange(n, device=s.dev) + torch.randint(c["far"] - n, (1,), device=s.dev, generator=s.gen)
    else:
        s.positions = torch.randint(c["far"], (n,), device=s.dev, generator=s.gen)
    f, s.factor = _frequencies(c)
    s.inv = f.to(s.dev)
    if own:
        from async_llm_amd.rotary import RotaryEmbedding

        s.rotary = RotaryEmbedding(c["d"], rotary_dim=c["rotary"], base=1e6, interleaved=c["layout"] == "pairs",
                                   scaling=SCALINGS[c["scaling"]], device=s.dev)


def _weights(s, num_slots):
    """Sums of former steps: few tokens with most of the weight, and some that nobody ever saw."""
    w = torch.exp(2 * torch.randn(s.case["hkv"], num_slots, device=s.dev, generator=s.gen) - 6)
    return w * (torch.rand(num_slots, device=s.dev, generator=s.gen) > 0.3)


def _prepare_select(s):
    c, page = s.case, s.case["page"]
    s.counts = _lengths(c)
    s.keep = [_kept(c, n) for n in s.counts]
    pages = [-(-n // page) for n in s.counts]
    order = torch.randperm(sum(pages), device=s.dev, generator=s.gen)
    at, rows = 0, []
    for n, p in zip(s.counts, pages):
        rows.append((order[at: at + p, None] * page + torch.arange(page, device=s.dev)).reshape(-1)[:n])
        at += p
    s.slots = torch.cat(rows)
    s.weights = _weights(s, sum(pages) * page)
    # the same padded, for the plain form
    s.padded = torch.zeros(len(rows), max(s.counts), dtype=torch.int64, device=s.dev)
    for i, r in enumerate(rows):
        s.padded[i, : len(r)] = r
    s.length, s.stay = (torch.tensor(x, device=s.dev)[:, None] for x in (s.counts, s.keep))
    if own:
        from async_llm_amd.shared_cache import CacheEviction

        s.select = CacheEviction.select


def _prepare_move(s):
    c, page = s.case, s.case["page"]
    n, of = c["rows"], c["of"]
    pages = -(-of // page) + -(-n // page)
    _pool(s, pages, c["layers"])
    order = torch.randperm(pages, device=s.dev, generator=s.gen)
    slots = (order[:, None] * page + torch.arange(page, device=s.dev)).reshape(-1)  # runs of scattered pages
    kept = torch.randperm(of, device=s.dev, generator=s.gen)[:n].sort().values
    s.source, s.target = slots[kept].contiguous(), slots[-(-of // page) * page:][:n].contiguous()
    s.shifts = torch.arange(n, device=s.dev) - kept
    s.rope = _rotation(c, s.dev, of + 1)
    s.weights = _weights(s, s.num_slots)
    if own:
        _handles(s)


def _prepare_views(s):
    c, page, dev = s.case, s.case["page"], s.dev
    s.views, s.tokens = _views(c), _blocks(c)
    pages = sum(-(-n // page) for n in s.tokens.values())
    _pool(s, pages, 1, values=False)
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
        three = c["rope"] == "mrope" and c["kind"] == "weigh_chunk"
        s.rel.append(_image_positions(new) if three else torch.arange(new))
        spans = [_span_of(c, n) for _, n in view[:-1]] + [_span_of(c, view[-1][1] - new)]
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
    s.place, row = place.to(dev), torch.arange(rows)[None, :]
    s.valid = (row < torch.tensor(s.new)[:, None]).to(dev)
    s.counted = ((row >= torch.tensor([new - _counted(c, new) for new in s.new])[:, None])).to(dev) & s.valid
    # the log-sums that the step's attention left behind
    top = torch.full((len(s.new), c["hkv"], rows, c["hq"] // c["hkv"]), -math.inf, device=dev)
    for j in range(depth):
        top = torch.logaddexp(top, torch.logsumexp(_scores(s, j), dim=-1))
    s.lse = torch.empty(sum(s.new), c["hq"], device=dev)
    s.lse[s.place[s.valid]] = top.permute(0, 2, 1, 3)[s.valid].reshape(-1, c["hq"])
    # (as much as this step adds, as after one step or two)
    s.weights = _weights(s, s.num_slots) * (50 * sum(_counted(c, new) for new in s.new) * c["hq"] / c["hkv"] / s.num_slots)
    if own:
        _handles(s)
        s.sums = s.weights.clone()
        _plan(s)


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
    if c["kind"] == "weigh":
        group = WorkerGroup(cache_structure=[[blocks[name] for name, _ in view] for view, _ in s.views])
        pending = {id(blocks[view[-1][0]]): opened[view[-1][0]] for view, _ in s.views}
        slots = torch.tensor([starts[view[-1][0]][(view[-1][1] - 1) // page] + (view[-1][1] - 1) % page
                              for view, _ in s.views], dtype=torch.int32, device=s.dev)
        s.meta = s.op.prepare(group, pending, slots)
    else:
        specs = []
        for r, (view, new) in enumerate(s.views):
            name = view[-1][0]
            specs.append(PrefillSpec([blocks[b] for b, _ in view[:-1]], torch.tensor(starts[name], dtype=torch.int32), new,
                                     blocks[name].num_tokens, blocks[name].mrope_span,
                                     s.rel[r] if s.rel[r].dim() == 2 else None))
        s.meta = s.op.prepare_prefill_batch(specs)
    s.plan = s.eviction.plan(s.meta, window=c["window"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return {"rotate": _run_rotate, "select": _run_select, "move": _run_move, "weigh": _run_weigh,
            "weigh_chunk": _run_weigh}[s.case["kind"]](s)


def _run_rotate(s):
    if own:
        q, k = s.rotary(s.positions, s.q, s.k)
        return {"q": q, "k": k}
    c = s.case
    angle = s.positions.double()[:, None] * s.inv
    cos, sin = ((f * s.factor).float()[:, None] for f in (angle.cos(), angle.sin()))
    pairs = c["rotary"] // 2
    out = {}
    for name, x in (("q", s.q), ("k", s.k)):
        x = x.float().view(c["rows"], -1, c["d"])
        a, b = (x[..., :pairs], x[..., pairs: 2 * pairs]) if c["layout"] == "half" else (x[..., 0: 2 * pairs: 2], x[..., 1: 2 * pairs: 2])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.cat([a, b], dim=-1) if c["layout"] == "half" else torch.stack([a, b], dim=-1).flatten(-2)
        out[name] = torch.cat([turned, x[..., 2 * pairs:]], dim=-1).view(c["rows"], -1).to(s.dtype)
    return out


def _run_select(s):
    c = s.case
    if own:
        kept = s.select(s.weights, s.slots, s.counts, s.keep, first=c["first"], last=c["last"])
        return {"positions": kept.positions, "slots": kept.slots}
    score = s.weights.double().sum(0).float()[s.padded]
    at = torch.arange(score.shape[1], device=s.dev)
    always = (at < c["first"]) | (at >= s.length - c["last"])
    score = torch.where(always, math.inf, score).masked_fill(at >= s.length, -math.inf)
    order = score.sort(dim=1, descending=True, stable=True).indices
    stays = torch.zeros_like(score, dtype=torch.bool).scatter_(1, order, at < s.stay)
    return {"positions": torch.nonzero(stays)[:, 1], "slots": s.padded[stays]}


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


def _pools(s):
    out = {"weights": s.weights}
    for name, rows in zip("kv", s.kv):
        out[name] = list(rows)
    if s.scales is not None:
        out["scales"] = s.scales.view(torch.float8_e8m0fnu)
    return out


def _run_move(s):
    c = s.case
    if own:
        s.eviction.move(s.source, s.target, s.shifts, weights=s.weights)
        return _pools(s)
    (page, place), (to_page, to_place) = ((x // c["page"], x % c["page"]) for x in (s.source, s.target))
    cos, sin = _turns(s.rope, s.shifts)
    s.weights[:, s.target] = s.weights[:, s.source]
    if c["codes"]:
        raw = s.kv.view(torch.uint8)
        codes, scales = raw[:, :, page, :, place], s.scales[:, :, page, :, place]  # [rows, 2, layers, hkv, d]
        k = _values(codes[:, 0].contiguous().view(s.kv.dtype), scales[:, 0])
        turned, e = _quantised(_turned(k, cos[:, None, None], sin[:, None, None]), c["codes"])
        # (a row that keeps its position is moved code for code)
        still = (s.shifts == 0)[:, None, None]
        turned = torch.where(still[..., None], codes[:, 0], turned.view(torch.uint8))
        e = torch.where(still, scales[:, 0], e)
        raw[:, :, to_page, :, to_place] = torch.stack([turned, codes[:, 1]], dim=1)
        s.scales[:, :, to_page, :, to_place] = torch.stack([e, scales[:, 1]], dim=1)
        return _pools(s)
    k = _turned(s.kv[0][:, page, place].float(), cos[:, None], sin[:, None])  # [layers, rows, hkv, d]
    s.kv[0][:, to_page, to_place] = k.to(s.dtype)
    s.kv[1][:, to_page, to_place] = s.kv[1][:, page, place]
    return _pools(s)


def _keys(s):
    """32-bit keys by slot, ``[slots, hkv, d]``."""
    c = s.case
    k = _values(s.kv[0][0], s.scales[0, 0]).transpose(1, 2) if c["codes"] else s.kv[0][0].float()
    return k.reshape(-1, c["hkv"], c["d"])


def _scores(s, j, keys=None):
    """Scores of all rows over the tokens of the j-th block of their views, ``[requests, hkv, rows, g, tokens]``; -inf where a
    row does not see a token."""
    c = s.case
    hkv, g, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    keys = _keys(s) if keys is None else keys
    q = s.q[s.place].float().view(*s.place.shape, hkv, g, d)  # [requests, rows, hkv, g, d]
    where = s.where[..., j, :, :]
    if s.rope["axis"] is not None and where.dim() == 2:
        where = where.expand(3, -1, -1)
    cos, sin = _turns(s.rope, where)
    turned = _turned(q, cos[:, :, None, None], sin[:, :, None, None]).permute(0, 2, 1, 3, 4).reshape(len(s.new), hkv, -1, d)
    x = torch.matmul(turned, keys[s.index[j]].permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    x = x.view(len(s.new), hkv, q.shape[1], g, -1)
    t, row = torch.arange(x.shape[-1], device=s.dev), torch.arange(q.shape[1], device=s.dev)
    seen = (t < s.length[j][:, None])[:, None, :] & (t <= (s.causal[j][:, None] + row)[..., None])
    return x.masked_fill_(~seen[:, None, :, None, :], -math.inf)


def _run_weigh(s):
    c = s.case
    if own:
        return {"weights": s.eviction.accumulate(s.q, s.lse, 0, s.plan, s.weights, out=s.sums)}
    out, keys = s.weights.clone(), _keys(s)
    lse = s.lse[s.place].view(*s.place.shape, c["hkv"], -1).permute(0, 2, 1, 3)
    lse = lse.masked_fill(~s.counted[:, None, :, None], math.inf)
    for j, index in enumerate(s.index):  # the blocks of a view, one after the other
        p = torch.exp(_scores(s, j, keys) - lse[..., None])
        out.index_add_(1, index.reshape(-1), p.sum((2, 3)).transpose(0, 1).reshape(c["hkv"], -1))
    return {"weights": out}


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(s, kv, layer, slots):
    """``[n, hkv, d]``"""
    page, place = slots // s.case["page"], slots % s.case["page"]
    if not s.case["codes"]:
        return s.kv[kv][layer][page, place].double()
    codes = s.kv[kv][layer].view(torch.uint8)[page, :, place].view(s.kv.dtype).double()
    return codes * torch.pow(2.0, s.scales[kv, layer][page, :, place].double() - 127)[..., None]


def _exact_turn(s, x, where):
    """``x [n, heads, d]`` as complex pairs times the turns of ``where [n]`` or ``[3, n]``."""
    r = s.rope
    if r["table"] is not None:
        entry = r["table"][where.abs()].double()
        unit = torch.complex(entry[:, : entry.shape[1] // 2], entry[:, entry.shape[1] // 2:] * where.sign()[:, None])
    else:
        where = where if where.dim() == 2 else torch.stack([where] * 3)
        product = where.float()[r["axis"]] * r["inv"][:, None]  # angles are 32-bit products by definition
        unit = torch.polar(torch.ones_like(product, dtype=torch.float64), product.double()).T
    h = unit.shape[1]
    z = torch.complex(x[..., :h].contiguous(), x[..., h: 2 * h].contiguous()) * unit[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * h:]], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "select": lambda s: None, "move": _exact_move, "weigh": _exact_weigh,
            "weigh_chunk": _exact_weigh}[case["kind"]](s)


def _exact_rotate(s):
    c = s.case
    h, out = c["rotary"] // 2, {}
    unit = torch.polar(torch.full((c["rows"], h), s.factor, dtype=torch.float64, device=s.dev),
                       torch.outer(s.positions.double(), s.inv))[:, None]
    for name, x in (("q", s.q), ("k", s.k)):
        x = x.double().view(c["rows"], -1, c["d"])
        y = x.clone()
        if c["layout"] == "pairs":
            z = torch.view_as_complex(x[..., : 2 * h].unflatten(-1, (h, 2)).contiguous()) * unit
            y[..., : 2 * h] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :h].contiguous(), x[..., h: 2 * h].contiguous()) * unit
            y[..., :h], y[..., h: 2 * h] = z.real, z.imag
        out[name] = y.view(c["rows"], -1)
    return out


def _exact_move(s):
    c = s.case
    weights = s.weights.double()
    weights[:, s.target] = s.weights[:, s.source].double()
    if c["codes"]:  # (codes and scales are rounded: which values they are is for the plain form to say)
        return {"weights": weights}
    page, place = s.target // c["page"], s.target % c["page"]
    out = {"weights": weights, "k": [], "v": []}
    for layer in range(c["layers"]):
        for kv, name in enumerate("kv"):
            rows, moved = s.kv[kv][layer].double(), _exact_rows(s, kv, layer, s.source)
            rows[page, place] = moved if kv else _exact_turn(s, moved, s.shifts)
            out[name].append(rows)
    return out


def _exact_weigh(s):
    c = s.case
    hkv, g, d = c["hkv"], c["hq"] // c["hkv"], c["d"]
    out, first = s.weights.double(), 0
    for r, (view, new) in enumerate(s.views):
        skip = new - _counted(c, new)
        q = s.q[first + skip: first + new].double().view(new - skip, c["hq"], d)
        lse = s.lse[first + skip: first + new].double().view(-1, hkv, g).transpose(0, 1).reshape(hkv, -1, 1)
        first += new
        for j, (name, n) in enumerate(view):
            slots = (s.pages[name][:, None] * c["page"] + torch.arange(c["page"], device=s.dev)).reshape(-1)[:n]
            k = _exact_rows(s, 0, 0, slots)
            turned = _exact_turn(s, q, (s.rel[r].to(s.dev) + int(s.starts[j, r]))[..., skip:])
            turned = turned.view(new - skip, hkv, g, d).transpose(0, 1).reshape(hkv, -1, d)
            p = torch.exp(torch.bmm(turned.contiguous(), k.permute(1, 2, 0).contiguous()) / math.sqrt(d) - lse)
            if j == len(view) - 1:
                ahead = torch.arange(n, device=s.dev) - (n - new) > torch.arange(skip, new, device=s.dev)[:, None]
                p = p.view(hkv, new - skip, g, n).masked_fill(ahead[None, :, None], 0.0).view(hkv, -1, n)
            out[:, slots] += p.sum(1)
    return {"weights": out}
