"""The block operators in CUDA graphs beside other work: as the very first call of a process, behind copies and behind
streams that join, where a dependent launch has no kernel, or several, before it."""

from __future__ import annotations

import subprocess
import sys

import pytest
import torch

from ats_v2_b200.norm_fused import fused_sandwich_norm
from ats_v2_b200.quantization import int8_linear, quantize_int8
from ats_v2_b200.rope import apply_multi_axis_rotary

pytestmark = pytest.mark.gpu

FIRST = """
import torch
from ats_v2_b200.norm_fused import fused_sandwich_norm
from ats_v2_b200.quantization import int8_linear, quantize_int8
from ats_v2_b200.rope import apply_multi_axis_rotary

dev = "cuda"
x = torch.randn({M}, 512, device=dev)
w, s = (t.to(dev) for t in quantize_int8(torch.randn(4096, 512)))
p = torch.ones(512, device=dev, requires_grad=True)
pos = torch.arange({M}, device=dev)[None]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    h, r = fused_sandwich_norm(x, x, p, p)
    (dp,) = torch.autograd.grad((h, r), p, (x, x))
    y = int8_linear(h.detach(), w, s)
    z, _ = apply_multi_axis_rotary(y.view(1, {M}, 64, 64).transpose(1, 2), None, pos, torch.ones(32, device=dev), (32,))
graph.replay()
h, r = fused_sandwich_norm(x, x, p, p)
y2 = int8_linear(h.detach(), w, s)
z2, _ = apply_multi_axis_rotary(y2.view(1, {M}, 64, 64).transpose(1, 2), None, pos, torch.ones(32, device=dev), (32,))
(dp2,) = torch.autograd.grad((h, r), p, (x, x))
assert torch.equal(y, y2) and torch.equal(z, z2) and torch.equal(dp, dp2)
print("as eager")
"""


@pytest.mark.parametrize("M", [1, 40, 2304])
def test_the_first_call_of_a_process_may_be_captured(M):
    run = subprocess.run([sys.executable, "-c", FIRST.replace("{M}", str(M))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "as eager" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("M", [1, 2, 40, 300, 2304])
def test_behind_copies_and_joined_streams(M):
    g = torch.Generator().manual_seed(M)
    src, x = torch.randn(M, 512, generator=g).cuda(), torch.zeros(M, 512, device="cuda")
    w0, s0 = quantize_int8(torch.randn(2048, 512, generator=g).cuda())
    w, s = torch.zeros_like(w0), torch.zeros_like(s0)
    post = torch.rand(512, generator=g).cuda()
    pos = torch.randint(0, 99, (2, 1, M), generator=g).cuda()
    inv = torch.rand(32, generator=g).cuda()
    side = [torch.cuda.Stream() for _ in range(2)]

    def step():
        here = torch.cuda.current_stream()
        x.copy_(src)  # a copy, not a kernel, is the last thing on the stream
        y = int8_linear(x, w0, s0)
        for st in side:
            st.wait_stream(here)
        with torch.cuda.stream(side[0]):
            w.copy_(w0)
            s.copy_(s0)
        with torch.cuda.stream(side[1]):
            h, r = fused_sandwich_norm(x, src, post, post)
        for st in side:
            here.wait_stream(st)
        y2 = int8_linear(h, w, s)  # reads what two streams wrote
        heads = y2.view(1, M, 32, 64).transpose(1, 2)
        z, _ = apply_multi_axis_rotary(heads, None, pos, inv, (20, 12))
        x.zero_()
        return y, h, r, y2, z

    def alone():  # each on one stream, with all done before the next
        torch.cuda.synchronize()
        y = int8_linear(src, w0, s0)
        h, r = fused_sandwich_norm(src, src, post, post)
        torch.cuda.synchronize()
        y2 = int8_linear(h, w0, s0)
        torch.cuda.synchronize()
        return y, h, r, y2, apply_multi_axis_rotary(y2.view(1, M, 32, 64).transpose(1, 2), None, pos, inv, (20, 12))[0]

    want = alone()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    w.zero_()
    s.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        src.copy_(torch.randn(M, 512, generator=g))
        w.zero_()
        s.zero_()
        graph.replay()
        for a, b in zip(held, alone()):
            assert torch.equal(a, b)
