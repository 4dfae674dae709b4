"""Shared host memory on a machine that may refuse to page-lock it: the rows are
the same either way, and a refusal is over when the call has returned."""
import ctypes
import mmap

import pytest
import torch

from geeps_amd import native, rowops
from test_hostshare import Owner, _open, pytestmark as needs_app


@pytest.mark.gpu
@needs_app
@pytest.mark.parametrize("floats", [1, 1000 * 128 + 7, 1 << 22])
def test_peer_reads_what_the_owner_wrote_beside_a_gpu(floats):
    o = Owner(floats)
    try:
        assert o.pinned in ("0", "1")
        assert _open(o.args()) == (0, "ok")
    finally:
        o.close()


@pytest.mark.gpu
def test_a_refused_registration_fails_no_later_call(dev):
    L = native.lib()
    memory = mmap.mmap(-1, 1 << 20)
    at = ctypes.addressof(ctypes.c_char.from_buffer(memory))
    rc = L.gp_host_register(at, 1 << 20)
    assert rc in (native.GP_OK, native.GP_ERR_HIP)
    y, x = torch.full((128 * 1000,), 2.0, device=dev), torch.full((128 * 1000,), 3.0, device=dev)
    rowops.apply_updates(y, [x])
    assert bool((y == 5.0).all())
    assert bool((x + 1 == 4.0).all())
    if rc == native.GP_OK:
        assert L.gp_host_unregister(at) == native.GP_OK
