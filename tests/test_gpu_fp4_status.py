"""Failure detection of the fp4 product: a wait that runs out is reported, once, and what follows runs as before."""
import ctypes
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def status(L):
    v = ctypes.c_int32(-1)
    L.call("duq4_last_device_status", L.current_stream(), ctypes.byref(v))
    return v.value


def test_a_wait_that_runs_out_is_reported_once():
    import duqlinear4bitcuda_b200.lib as L
    import duqlinear4bitcuda_b200.nn as nn
    layer = nn.LinearFP4.from_linear(torch.nn.Linear(512, 300).half().cuda())
    x = torch.randn(200, 512, device="cuda").half()
    want = layer(x)
    assert status(L) == 0
    result = torch.zeros(1, dtype=torch.int32, device="cuda")
    t0 = time.monotonic()
    L.call("duq4_fp4_wait_selftest", L.ptr(result), L.current_stream())
    after = layer(x)                      # queued behind it
    assert status(L) == 414               # the wait's code 14, in the product's range
    took = time.monotonic() - t0
    assert result.item() == 3 and 0.9 < took < 5
    assert status(L) == 0
    assert torch.equal(after, want) and torch.equal(layer(x), want) and status(L) == 0


def test_run_outs_do_not_add_up():
    """The first code stays until it is read; a second run-out of the same kind is one report."""
    import duqlinear4bitcuda_b200.lib as L
    result = torch.zeros(2, dtype=torch.int32, device="cuda")
    for i in range(2):
        L.call("duq4_fp4_wait_selftest", result[i:].data_ptr(), L.current_stream())
    assert status(L) == 414 and result.tolist() == [3, 3] and status(L) == 0
