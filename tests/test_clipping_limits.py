"""Clipped updates at the ends of what their calls allow."""
import ctypes
import resource

import pytest

from geeps_amd import native


def create(sizes, types):
    n = len(sizes)
    at = [(1 + 2 * i) << 54 for i in range(2 * n)]  # addresses that nothing is read from
    h = ctypes.c_void_p()
    rc = native.lib().gp_grad_plan_create(
        ctypes.byref(h), n, (ctypes.c_void_p * n)(*at[:n]), (ctypes.c_int * n)(*types), (ctypes.c_void_p * n)(*at[n:]),
        (ctypes.c_int * n)(*types), (ctypes.c_size_t * n)(*sizes))
    assert h.value is None
    return rc, native.lib().gp_last_error()


@pytest.mark.parametrize("sizes,word", [
    ([1 << 41], b"too many values"), ([1 << 52], b"too many values"), ([5, 1 << 40, 1 << 40], b"too many values"),
    ([1 << 61], b"too long"), ([(1 << 61) - 1, 1 << 60], b"too long")])
@pytest.mark.parametrize("kind", [0, 1])
def test_lists_past_any_memory_are_refused(sizes, word, kind):
    """Before a table of them is built on the host: 2^52 values would take 2^37 entries of 32 bytes."""
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    rc, message = create(sizes, [kind] * len(sizes))
    assert rc == native.GP_ERR_INVALID and word in message, message
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 16  # KiB
