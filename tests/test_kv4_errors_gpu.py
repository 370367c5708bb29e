"""Errors of the q4_0 cache's calls: a refused call leaves nothing behind that a later one would report."""
import ctypes as ct

import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu


def test_a_failed_call_does_not_fail_the_next(dev):
    """A cache larger than any memory."""
    import torch
    L = tsrc.lib()
    kv = dev.kv4_create(511, 64, 10)
    try:
        h = ct.c_void_p()
        assert L.tsrc_kv4_create(dev.handle, 511, 64, 1 << 30, ct.byref(h)) == tsrc.E_NOMEM
        x = torch.randn(4, 511 * 64, device="cuda")
        kv.set_rows(x, x)
        out = torch.empty_like(x)
        kv.get_rows(out, None)
        dev.sync()
        want = P.unpack(P.pack(*P.quantise(x.cpu().numpy())))
        np.testing.assert_array_equal(out.cpu().numpy(), want.astype(np.float32))
    finally:
        kv.free()


def test_all_that_went_wrong_is_reported(dev):
    """Bad indexes of three calls before one synchronisation: the report names the three, and is then cleared."""
    import torch
    kv = dev.kv4_create(1, 64, 10)
    try:
        x = torch.randn(2, 64, device="cuda")
        at = torch.tensor([3, 10], device="cuda")
        kv.set_rows(x, None, cells=at)
        kv.get_rows(x, None, cells=at)
        kv.reorder(torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 1, 2, 5, 5)
        with pytest.raises(tsrc.TsrcError) as e:
            dev.sync()
        assert e.value.code == tsrc.E_ARG and all(n in str(e.value) for n in ("set_rows", "get_rows", "reorder"))
        dev.sync()
    finally:
        kv.free()
