"""Paged attention after a bounded wait that ran out: what the block has in flight lands before it leaves
(without a GPU fault: a barrier that expects bytes which nothing sends)."""
import ctypes as C
import time

import pytest
import torch

import timestral_b200 as tb

pytestmark = pytest.mark.gpu


def test_copies_in_flight_land_and_the_wait_for_them_is_bounded():
    assert torch.cuda.is_available()
    err, landed = C.c_int32(0), C.c_int32(0)
    t0 = time.time()
    rc = tb.lib().tsb_test_wait_expiry(2, C.byref(err), C.byref(landed))
    assert rc == tb.TSB_ERR_DEVICE and err.value == 5, (rc, err.value)
    assert landed.value == 1, "the copies in flight were not waited for"
    assert time.time() - t0 < 60
    x = torch.arange(1000, device="cuda")
    assert x.sum().item() == 499500                       # the context is usable
