"""The 8-bit projection's clusters leave nothing behind: CTAs that read one another's shared memory, or signal one
another's barriers, run many times in a row with other kernels on the same SMs right after them, at the shares, sizes
and numbers of blocks where some warps have nothing to read or some barriers are passed once."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ats_v2_b200 import _lib
from ats_v2_b200.quantization import int8_linear, quantize_int8
from tests.bounds import INT8_SLACK, assert_within, int8_exact

pytestmark = pytest.mark.gpu


def repeated(M, N, K, calls=60):
    """The same call many times, with a kernel that fills shared memory (the quantisation of odd rows) between."""
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).cuda().bfloat16()
    w, s = quantize_int8(torch.randn(N, K, generator=g).cuda())
    odd = torch.randn(600, 2047, generator=g).cuda()
    held = []
    for _ in range(calls):
        held.append(int8_linear(x, w, s))
        quantize_int8(odd)
    e, mag = int8_exact(x, w, s)
    assert_within(held[0], e, INT8_SLACK * mag, f"{M} {N} {K}")
    for y in held[1:]:
        assert torch.equal(y, held[0])
    _lib.check_device_status("after the calls")


@pytest.mark.parametrize("M,N,K", [(2, 300, 4096), (13, 129, 512), (16, 5000, 6200), (17, 4100, 8192), (31, 2999, 1700),
                                   (33, 1000, 2048), (48, 11008, 4096), (64, 10120, 3300), (65, 200, 1024),
                                   (200, 2048, 8192)])
def test_parts_of_k_with_uneven_shares_of_the_tokens(M, N, K):
    repeated(M, N, K)


@pytest.mark.parametrize("M,N,K", [(2304, 4096, 16), (2304, 4096, 130), (5001, 1003, 260), (1200, 8000, 900),
                                   (4500, 4500, 64), (2200, 4096, 2048)])
def test_pairs_whose_barriers_are_passed_once_or_often(M, N, K):
    """One block of K, fewer blocks than stages, more than twice as many; one tile to a pair, and several."""
    repeated(M, N, K, calls=30)


@pytest.mark.parametrize("budget", [50, 400, 1500, 6000, 40000])
@pytest.mark.parametrize("M,N,K", [(40, 512, 4096), (200, 2048, 2048), (2304, 4096, 2048), (5001, 1003, 260)])
def test_waits_that_run_out_in_the_middle(M, N, K, budget):
    """Roles give up after some of their blocks or tiles, in one CTA of a pair before the other, while an epilogue is
    between two tiles: the kernel ends, it reports it if it did not finish, and the next call is right."""
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).cuda().bfloat16()
    w, s = quantize_int8(torch.randn(N, K, generator=g).cuda())
    want = int8_linear(x, w, s)
    _lib.check_device_status("before the short waits")
    for _ in range(8):
        _lib.call("ats_set_wait_budget", budget)
        try:
            y = int8_linear(x, w, s)
            torch.cuda.synchronize()
        finally:
            _lib.call("ats_set_wait_budget", 0)
        code = ctypes.c_int(0)
        st = _lib.query("ats_device_status", ctypes.byref(code))
        assert st == (_lib.ATS_OK if code.value == 0 else _lib.ATS_ETIMEOUT)
        assert code.value in (0, 31, 32, 33, 34, 41, 43)  # the shortened waits, none of those that drain
        if code.value == 0:
            assert torch.equal(y, want)
        assert torch.equal(int8_linear(x, w, s), want)
    _lib.check_device_status("after whole calls")
