"""A plan of attention weights holds its pool's pages and slots: over a pool of another size it is refused, before anything is
launched."""

import ctypes

import numpy as np
import pytest

from async_llm_amd import native
from tests.test_weigh_plan_cpu import plan_of

NOWHERE = ctypes.c_void_p(1 << 20)  # (an address that a refused call does not look at)


def weigh(words, pages, codes):
    shape, rope = native.VaShape(8, 2, 64, 4, native.VA_BF16), native.VaRope(native.VA_ROPE_TABLE, 0, None, 0, 0, 0, None)
    tables = (NOWHERE, words.ctypes.data, NOWHERE, NOWHERE, 0, NOWHERE, 0, NOWHERE, NOWHERE, None, 0, shape, rope, None)
    if codes:
        pool = native.VaQuantPool(NOWHERE, NOWHERE, NOWHERE, NOWHERE, native.VA_CODE_E4M3, pages)
        return native.lib.va_weigh_q8(NOWHERE, 512, pool, *tables)
    return native.lib.va_weigh(NOWHERE, 512, NOWHERE, 128, pages, *tables)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("pages", [0, 1, 99, 101, 200])
def test_a_plan_of_another_pool_is_refused(codes, pages):
    rc, words, _ = plan_of([(1, [99, 3], 7, 0)], pages=100, codes=codes)
    assert rc == 0
    assert weigh(words, pages, codes) == native.VA_ERR_ARG
    assert b"another shape or pool" in native.lib.va_last_error()
    # over its own pool the call goes on to the workspace, which is missing here
    assert weigh(words, 100, codes) == native.VA_ERR_CAPACITY
