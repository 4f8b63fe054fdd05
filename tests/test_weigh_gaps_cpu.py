"""Plans of attention weights own the tokens that somebody sees and no others, for keys of 16 and 32 bits: also where lists name
single slots of a page with others between them."""

import random

import pytest

from async_llm_amd import native
from tests.test_weigh_plan_cpu import counted, expected, plan_of, random_subs

SLOTS, CAUSAL = native.VA_SUB_SLOTS, native.VA_SUB_CAUSAL


def check(subs, heads, page, pages, dtype, window=0):
    rc, words, counts = plan_of(subs, heads, page, pages, window, dtype=dtype)
    assert rc == 0, native.lib.va_last_error()
    pairs, owners = counted(words, heads, page, dtype)
    want = expected(subs, heads[0] // heads[1], page, window)
    assert pairs == want
    assert set(owners) == set(s for _, s in want)
    return counts


@pytest.mark.parametrize("dtype", [native.VA_BF16, native.VA_F32])
def test_slots_with_others_between_them(dtype):
    heads = (8, 2, 64)
    for subs, spans in (
        ([(1, [0, 5], 2, SLOTS)], 2),
        ([(1, [5, 0, 1, 15], 4, SLOTS)], 3),
        ([(1, [16], 1, SLOTS), (2, [19], 1, SLOTS), (1, [17], 1, SLOTS)], 2),
        ([(1, [2], 5, 0), (1, [32 + 9], 1, SLOTS)], 2),  # the page's first five tokens, and one behind
        ([(1, [2], 9, 0), (1, [32 + 9], 1, SLOTS)], 1),
        ([(9, [2], 12, CAUSAL), (40, [32 + 14], 1, SLOTS)], 2),  # tile items
        ([(1, [3, 4, 3], 2, SLOTS)], 1),  # (only two of its entries count)
        ([(1, [7, 7, 9], 3, SLOTS)], 2),  # one twice
    ):
        assert check(subs, heads, 16, 8, dtype).n_spans == spans


def slot_lists(r, page, pages):
    out = []
    for _ in range(r.randint(1, 4)):
        base = r.randrange(pages)
        near = [min(pages * page - 1, base * page + r.randrange(2 * page)) for _ in range(r.randint(1, 6))]
        out.append((r.choice([1, 1, 2, 9]), near, r.randint(0, len(near)), SLOTS | r.choice([0, 0, CAUSAL])))
    return out


@pytest.mark.parametrize("dtype", [native.VA_BF16, native.VA_F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (3, 1, 96), (16, 16, 128), (40, 2, 256)])
@pytest.mark.parametrize("page", [1, 3, 16])
def test_owners_are_who_is_seen(dtype, heads, page):
    r = random.Random(heads[0] * 100 + page + dtype)
    for _ in range(25):
        subs = random_subs(r, page, 40) + slot_lists(r, page, 40)
        r.shuffle(subs)
        check(subs, heads, page, 40, dtype, r.choice([0, 0, 1, 2]))


@pytest.mark.parametrize("dtype", [native.VA_BF16, native.VA_F32])
@pytest.mark.parametrize("rows", [5, 500])
def test_split_rows_count_every_pair_once(dtype, rows):
    """Few tokens under many rows: items of parts of the rows, joined."""
    subs = [(rows, list(range(40)), 640, CAUSAL), (rows, [50, 51, 52], 41, 0), (2, [900, 905, 908], 3, SLOTS)]
    counts = check(subs, (8, 2, 64), 16, 64, dtype)
    assert counts.n_joins >= 2 or rows == 5
