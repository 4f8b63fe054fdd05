"""The entry that moves tokens, with no layers: weights alone, and what it refuses."""

import ctypes

from async_llm_amd import native

NOWHERE = ctypes.c_void_p(1 << 20)  # (an address that these calls do not look at)


def test_no_layers():
    shape = native.VaShape(4, 2, 64, 16, native.VA_BF16)
    move = lambda src, n, weights, slots=160: native.lib.va_move_kv(  # noqa: E731
        None, None, 0, 0, 0, slots, src, src, None, n, weights, shape, None, None)
    assert move(None, 5, None) == 0  # neither rows nor weights
    assert move(None, 0, NOWHERE) == 0 and move(NOWHERE, 5, NOWHERE, 0) == 0
    assert move(None, 5, NOWHERE) == native.VA_ERR_ARG and b"null pointer" in native.lib.va_last_error()
    assert move(NOWHERE, -1, NOWHERE) == native.VA_ERR_ARG
    assert move(NOWHERE, 1 << 40, NOWHERE) == native.VA_ERR_ARG and b"too many tokens" in native.lib.va_last_error()
    # layers want a pool
    assert native.lib.va_move_kv(None, None, 128, 0, 1, 160, NOWHERE, NOWHERE, None, 5, None, shape, None, None) == native.VA_ERR_ARG
