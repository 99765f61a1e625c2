"""The bounded waits of the 8-bit projection's tensor-core kernels: with a budget of one cycle the first wait that has
not completed gives up, the kernel drains what is in flight and ends, the device status reports it, and the next call
is right again.  No wait is made to hang."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ats_v2_b200 import _lib
from ats_v2_b200.quantization import int8_linear, quantize_int8
from tests.bounds import INT8_SLACK, assert_within, int8_exact

pytestmark = pytest.mark.gpu


def status():
    code = ctypes.c_int(0)
    return _lib.query("ats_device_status", ctypes.byref(code)), code.value


@pytest.mark.parametrize("M,N,K", [(40, 512, 4096), (200, 2048, 2048), (2304, 4096, 2048)])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(M, N, K):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).cuda().bfloat16()
    w, s = quantize_int8(torch.randn(N, K, generator=g).cuda())
    torch.cuda.synchronize()
    _lib.check_device_status("before the timeout test")
    _lib.call("ats_set_wait_budget", 1)
    try:
        int8_linear(x, w, s)
        torch.cuda.synchronize()
    finally:
        _lib.call("ats_set_wait_budget", 0)
    st, code = status()
    assert st == _lib.ATS_ETIMEOUT and 30 < code < 50
    assert status() == (_lib.ATS_OK, 0)  # reading cleared it
    y = int8_linear(x, w, s)
    torch.cuda.synchronize()
    assert status() == (_lib.ATS_OK, 0)
    e, mag = int8_exact(x, w, s)
    assert_within(y, e, INT8_SLACK * mag)
