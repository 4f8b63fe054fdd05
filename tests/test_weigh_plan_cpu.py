"""Plans of attention weights without a GPU: every visible (query row, token) pair is counted once, every token has one
owner, and what no plan is made of is refused."""

import random

import numpy as np
import pytest
import torch

from async_llm_amd import native
from async_llm_amd.shared_cache import CacheEviction, SharedCacheAttention
from async_llm_amd.kvcache import MHAKVCache


def plan_of(subs, heads=(8, 2, 64), page=4, pages=64, window=0, capacity=None, dtype=native.VA_BF16, codes=False):
    """``subs``: (rows, entries, seq_len, flags)."""
    arrays = [np.concatenate([[0], np.cumsum([r for r, *_ in subs])]), np.concatenate([[0], np.cumsum([len(e) for _, e, *_ in subs])]),
              np.concatenate([np.asarray(e) for _, e, *_ in subs] or [[]]), [n for _, _, n, _ in subs], [f for *_, f in subs]]
    a = [np.ascontiguousarray(x, dtype=np.int32) for x in arrays]
    s = native.VaSubRequests(len(subs), int(a[0][-1]), int(a[0][-1]), a[0].ctypes.data, a[1].ctypes.data,
                             a[2].ctypes.data if a[2].size else None, a[3].ctypes.data, a[4].ctypes.data, None, None)
    shape, counts = native.VaShape(*heads, page, dtype), native.VaWeighCounts()
    words = np.zeros(1 << 20 if capacity is None else capacity, dtype=np.int32)
    return native.lib.va_weigh_plan(s, shape, int(codes), pages, window, words.ctypes.data, words.size, counts), words, counts


def counted(words, heads, page, dtype=native.VA_BF16):
    """{(sub-row, slot): times} of what the plan's items count, and {slot: owners}."""
    h = words[:24]
    n_items, n_rows, n_joins, n_partials, off = h[1], h[2], h[3], h[4], h[6:10]
    items = words[off[0]: off[0] + 8 * n_items].reshape(-1, 8)
    joins = words[off[1]: off[1] + 8 * n_joins].reshape(-1, 8)
    pages = words[off[2]:]
    sub, lo, hi = (words[off[3] + i * n_rows: off[3] + (i + 1) * n_rows] for i in range(3))
    g = heads[0] // heads[1]
    n_tile_items, n_tile_rows, n_strips = h[18], h[19], h[20]
    strips = words[h[21]: h[21] + n_strips + 1]
    assert n_rows * g % 16 == 0 and n_tile_items % 8 == 0 and n_tile_rows * g % 32 == 0
    if n_items > n_tile_items:  # strips hold every other item once
        assert n_strips % 8 == 0 and strips[0] == n_tile_items and strips[-1] == n_items and (np.diff(strips) >= 0).all()
    pairs, owners, parts = {}, {}, {}
    for k, (first_page, first, n, begin, end, partial) in enumerate(items[:, :6]):
        if n == 0:
            assert k < n_tile_items
            continue
        of_tile = 32 if k < n_tile_items else 16  # (row, q head) pairs
        assert end * 32 <= n_tile_rows * g and n <= 256 if k < n_tile_items else begin * 16 >= n_tile_rows * g
        if k >= n_tile_items and dtype != native.VA_F32 and heads[2] == 64:
            assert end == begin + 1
        assert 0 < n and 0 <= begin < end <= n_rows * g // of_tile
        slots = [int(pages[first_page + t // page]) * page + t % page for t in range(first, first + n)]
        if partial >= 0:
            parts[int(partial)] = (int(first_page), int(first), int(n))
            assert partial + n <= n_partials
        else:
            for s in slots:
                owners[s] = owners.get(s, 0) + 1
        # (q heads of a row may lie in two tiles of an item that splits: count them)
        for p in range(begin * of_tile, end * of_tile):
            r = p // g
            if sub[r] >= 0:
                for t, s in zip(range(first, first + n), slots):
                    if lo[r] <= t < hi[r]:
                        key = (int(sub[r]), s)
                        pairs[key] = pairs.get(key, 0) + 1
    for first_page, first, n, partial, count in joins[:, :5]:
        for i in range(count):
            assert parts.pop(int(partial + i * n)) == (first_page, first, n)
        for t in range(first, first + n):
            s = int(pages[first_page + t // page]) * page + t % page
            owners[s] = owners.get(s, 0) + 1
    assert not parts
    assert all(v == 1 for v in owners.values()), "a token has several owners"
    return pairs, owners


def expected(subs, g, page, window):
    out, row = {}, 0
    for rows, entries, n, flags in subs:
        for i in range(rows):
            if window and i < rows - window:
                continue
            seen = max(0, n - rows + i + 1) if flags & native.VA_SUB_CAUSAL else n
            for t in range(seen):
                slot = int(entries[t]) if flags & native.VA_SUB_SLOTS else int(entries[t // page]) * page + t % page
                out[row + i, slot] = out.get((row + i, slot), 0) + g
        row += rows
    return out


def random_subs(r, page, pages):
    free = list(range(pages))
    r.shuffle(free)
    blocks = []
    while len(free) > 3 and len(blocks) < 6:
        n = r.randint(1, min(len(free), 9))
        blocks.append([free.pop() for _ in range(n)])
    subs = []
    for _ in range(r.randint(1, 6)):
        b = r.choice(blocks)
        kind = r.random()
        if kind < 0.5:  # a reader, not of the last tokens maybe, or of a page list that is longer than it reads
            subs.append((r.choice([0, 1, 1, 3]), b, r.randint(0, len(b) * page), 0))
        elif kind < 0.75:  # many new tokens
            n = r.randint(1, len(b) * page)
            subs.append((r.randint(1, n + 2), b, n, native.VA_SUB_CAUSAL))
        elif kind < 0.8:  # pages that a list names twice
            subs.append((1, b + b[:2], r.randint(0, (len(b) + len(b[:2])) * page), 0))
        elif kind < 0.9:  # single slots
            subs.append((1, [r.choice(b) * page + r.randrange(page)], 1, native.VA_SUB_SLOTS))
        else:  # a list that shares some pages only
            mixed = b[::2] + r.choice(blocks)[1:]
            subs.append((r.randint(1, 2), mixed, r.randint(0, len(mixed) * page), 0))
    return subs


@pytest.mark.parametrize("heads", [(8, 2, 64), (3, 1, 64), (16, 16, 64), (40, 2, 64)])
@pytest.mark.parametrize("page", [1, 3, 16])
def test_every_pair_is_counted_once(heads, page):
    r = random.Random(heads[0] * 100 + page)
    for _ in range(25):
        subs, window = random_subs(r, page, 40), r.choice([0, 0, 1, 2])
        rc, words, counts = plan_of(subs, heads, page, 40, window)
        assert rc == 0, native.lib.va_last_error()
        pairs, owners = counted(words, heads, page)
        want = expected(subs, heads[0] // heads[1], page, window)
        assert pairs == want
        assert set(s for _, s in want) <= set(owners)


def test_readers_of_a_block_share_its_tokens():
    """A prompt that many read is one span, cut into chunks; a request's own block another."""
    prompt, own = list(range(100)), [[200 + 10 * i + k for k in range(10)] for i in range(4)]
    subs = [s for i in range(4) for s in ((1, prompt, 1600, 0), (1, own[i], 150, 0))]
    rc, words, counts = plan_of(subs, (8, 8, 64), 16, 300)
    assert rc == 0 and counts.n_spans == 5
    assert counts.n_rows == 16 * 5  # a row an q head: whole tiles of 16
    assert counts.n_joins == 0
    strips = np.diff(words[words[21]: words[21] + words[20] + 1])
    tokens = words[words[6]: words[6] + 8 * counts.n_items].reshape(-1, 8)[:, 2]
    assert tokens.sum() == 1600 + 4 * 150 and (strips <= 3).all()  # few items: workgroups for all


def test_lists_that_are_alike_and_lists_that_are_almost():
    """Readers of one list make one run of it, whatever they see of it; a list that goes on shares what is the same."""
    a, longer = list(range(10)), list(range(12))
    subs = [(1, a, 160, 0), (1, a, 150, 0), (0, a, 160, 0), (2, a, 159, native.VA_SUB_CAUSAL), (1, [20, 21], 32, 0)]
    rc, words, counts = plan_of(subs, (8, 8, 64), 16, 30)
    assert rc == 0 and counts.n_spans == 2
    rc, words, counts = plan_of([*subs, (1, longer, 192, 0)], (8, 8, 64), 16, 30)
    assert rc == 0 and counts.n_spans == 3
    pairs, _ = counted(words, (8, 8, 64), 16)
    assert pairs == expected([*subs, (1, longer, 192, 0)], 1, 16, 0)
    # a bad page is found in the first of two lists that are alike
    rc, _, _ = plan_of([(1, [3, 30], 20, 0), (1, [3, 30], 20, 0)], (8, 8, 64), 16, 30)
    assert rc == native.VA_ERR_ARG and b"page 30 lies outside" in native.lib.va_last_error()


def test_strips_cost_the_same():
    """Long and short blocks, some with many readers, over as many workgroups as the GPU holds."""
    r = random.Random(1)
    free = list(range(20000))
    prompt = [free.pop() for _ in range(512)]
    subs = []
    for _ in range(64):
        subs.append((1, prompt, 8192, 0))
        n = r.randint(20, 400)
        subs.append((1, [free.pop() for _ in range(n)], n * 16 - r.randint(0, 15), 0))
    rc, words, counts = plan_of(subs, (16, 4, 256), 16, 20000)
    counted_strips = words[words[21]: words[21] + words[20] + 1]
    items = words[words[6]: words[6] + 8 * counts.n_items].reshape(-1, 8)
    cost = [sum(n * (3 + b - a) for _, _, n, a, b, *_ in items[s: e]) for s, e in zip(counted_strips, counted_strips[1:])]
    cost = [c for c in cost if c]
    assert words[18] == 32  # the prompt: tiles
    assert rc == 0 and 480 <= len(cost) <= 512 and max(cost) < 1.05 * sum(cost) / len(cost)


def test_rows_are_split_where_tokens_are_few():
    for dtype in (native.VA_BF16, native.VA_F32):  # tile items; strips, of parts of the rows
        rc, words, counts = plan_of([(500, list(range(40)), 640, native.VA_SUB_CAUSAL)], (8, 2, 64), 16, 64, dtype=dtype)
        assert rc == 0 and counts.n_joins >= 2 and counts.n_items >= 16
        counted(words, (8, 2, 64), 16, dtype)


@pytest.mark.parametrize("subs, message", [
    ([(1, [64], 4, 0)], "page 64 lies outside"),
    ([(1, [-1], 1, 0)], "page -1 lies outside"),
    ([(1, [256], 1, native.VA_SUB_SLOTS)], "slot 256 lies outside"),
    ([(1, [0], 5, 0)], "5 tokens in 1 entries"),
    ([(1, [0], -1, 0)], "must not fall"),
])
def test_refusals(subs, message):
    rc, _, _ = plan_of(subs)
    assert rc == native.VA_ERR_ARG and message in native.lib.va_last_error().decode()


def test_no_rows_and_no_tokens_make_an_empty_plan():
    for subs in ([], [(0, [3], 4, 0)], [(1, [], 0, 0)], [(3, [5], 1, native.VA_SUB_CAUSAL), (1, [], 0, native.VA_SUB_SLOTS)]):
        rc, words, counts = plan_of(subs)
        assert rc == 0 and counts.n_spans <= 1
    rc, words, counts = plan_of([])
    assert counts.n_items == 0 and counts.workspace_bytes == 0


def test_a_small_buffer_says_how_large_it_has_to_be():
    subs = [(1, list(range(20)), 80, 0)]
    rc, _, counts = plan_of(subs, capacity=30)
    assert rc == native.VA_ERR_CAPACITY and counts.plan_words > 30
    rc, _, again = plan_of(subs, capacity=counts.plan_words)
    assert rc == 0 and again.plan_words == counts.plan_words


def test_heads_that_do_not_divide_and_negative_windows_are_refused():
    assert plan_of([(1, [0], 1, 0)], heads=(3, 2, 64))[0] == native.VA_ERR_ARG
    assert plan_of([(1, [0], 1, 0)], window=-1)[0] == native.VA_ERR_ARG
    assert plan_of([(1, [0], 1, 0)], pages=1 << 30, page=4)[0] == native.VA_ERR_ARG


def eviction_on_the_cpu(hq=4, hkv=2):
    pool = MHAKVCache(hkv, 1, 64, 8, 4, torch.bfloat16, torch.device("cpu"))
    op = SharedCacheAttention(pool, torch.zeros(8, 64), hq, hkv, 64, 4, torch.bfloat16, torch.device("cpu"))
    return CacheEviction(op)


def test_calls_without_a_gpu_are_refused():
    e = eviction_on_the_cpu()
    weights = e.new_weights()
    assert weights.shape == (2, 32)
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        CacheEviction.select(weights, one, [1], 1)
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        e.move(one, one)
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        e.clear(weights, one)
    for slots in (one.float(), one[None], one.bool()):
        with pytest.raises(ValueError, match="slots must be"):
            e.clear(weights, slots)
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        e.accumulate(torch.zeros(1, 256), None, 0, None, weights)
    with pytest.raises(ValueError, match="no multiple"):
        eviction_on_the_cpu(3, 2)


def test_selection_entry_refuses():
    n, k = np.array([5], dtype=np.int64), np.array([6], dtype=np.int64)
    call = lambda counts, keep, ws=0: native.lib.va_select_tokens(  # noqa: E731
        None, 1, 8, None, 1, counts.ctypes.data, keep.ctypes.data, 0, 0, None, None, None, None, ws, None)
    assert call(n, k) == native.VA_ERR_ARG and b"cannot stay" in native.lib.va_last_error()
    assert call(n, n) == native.VA_ERR_ARG and b"null pointer" in native.lib.va_last_error()
    assert call(-n, n) == native.VA_ERR_ARG
    assert call(n, 0 * n) == 0  # nothing stays: nothing to do
    long = np.array([50000], dtype=np.int64)
    need = native.lib.va_select_workspace_bytes(1, long.ctypes.data)
    assert need >= 4 * 50000 and native.lib.va_select_workspace_bytes(1, (-long).ctypes.data) == -1
    assert native.lib.va_select_workspace_bytes(1, n.ctypes.data) == 0
    clear = native.lib.va_clear_weights
    assert clear(None, -1, 4, None, 1, None) == native.VA_ERR_ARG and clear(None, 2, 4, None, 1, None) == native.VA_ERR_ARG
    assert clear(None, 0, 4, None, 1, None) == 0 and clear(None, 2, 4, None, 0, None) == 0
