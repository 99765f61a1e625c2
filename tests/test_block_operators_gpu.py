"""The block operators run together as a block runs them: norms at the block's end, the projection of the next block's
input, the rotation of its heads."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from ats_v2_b200.norm_fused import fused_sandwich_norm
from ats_v2_b200.quantization import Int8Linear, int8_linear, quantize_int8
from ats_v2_b200.rope import MultiAxisRotaryEmbedding
from tests.bounds import INT8_SLACK, assert_within, int8_exact, rotate_exact, rotate_slack, sandwich_exact, \
    sandwich_slack, turns_exact

pytestmark = pytest.mark.gpu

HQ, HK, D, SECTIONS = 6, 2, 64, (12, 10, 10)


class Block(nn.Module):
    """The end of one block and the projections of the next, for serving (8-bit weights) or training."""

    def __init__(self, hidden: int) -> None:
        super().__init__()
        self.post, self.pre = (nn.Parameter(1 + 0.1 * torch.randn(hidden)) for _ in range(2))
        self.gate = nn.Parameter(torch.randn(hidden))
        self.qkv = nn.Linear(hidden, (HQ + 2 * HK) * D, bias=False)
        self.rotary = MultiAxisRotaryEmbedding(D, SECTIONS)

    def forward(self, x, residual, positions):
        B, S, _ = x.shape
        h, s = fused_sandwich_norm(x, residual, self.post, self.pre, gate=self.gate, residual_scale=0.9, eps=1e-5)
        qkv = self.qkv(h).view(B, S, HQ + 2 * HK, D).transpose(1, 2)
        q, k = self.rotary(qkv[:, :HQ], qkv[:, HQ:HQ + HK], positions)
        return q, k, qkv[:, HQ + HK:], s


def inputs(B, S, H, dt):
    g = torch.Generator().manual_seed(B * S)
    x, res = (torch.randn(B, S, H, generator=g).to(dt).cuda() for _ in range(2))
    return x, res, torch.randint(0, 3000, (3, B, S), generator=g).cuda()


@pytest.mark.parametrize("B,S", [(1, 1), (32, 1), (2, 75), (1, 1000)])
def test_serving_chain(B, S):
    torch.manual_seed(0)
    block = Block(256).cuda()
    block.qkv = Int8Linear.from_linear(block.qkv)
    x, res, pos = inputs(B, S, 256, torch.bfloat16)
    with torch.no_grad():
        q, k, v, s = block(x, res, pos)
        h, s2 = fused_sandwich_norm(x, res, block.post, block.pre, gate=block.gate, residual_scale=0.9, eps=1e-5)
    e = sandwich_exact(x, res, block.post, block.pre, block.gate, 0.9, 1e-5)
    assert torch.equal(s, s2)
    assert_within(h, e["h"][0], sandwich_slack(256, 0) * e["h"][1])
    y = int8_linear(h, block.qkv.weight, block.qkv.scale)  # each step against its own exact value
    ey, mag = int8_exact(h.view(-1, 256), block.qkv.weight, block.qkv.scale)
    assert_within(y.view(-1, y.shape[-1]), ey, INT8_SLACK * mag)
    heads = y.view(B, S, -1, D).transpose(1, 2)
    turn = turns_exact(pos, block.rotary.inv_freq, bytes([0] * 12 + [1] * 10 + [2] * 10))
    assert_within(q, rotate_exact(heads[:, :HQ], turn), rotate_slack(heads[:, :HQ], 32))
    assert_within(k, rotate_exact(heads[:, HQ:HQ + HK], turn), rotate_slack(heads[:, HQ:HQ + HK], 32))
    assert torch.equal(v, heads[:, HQ + HK:])


def test_serving_chain_as_one_graph():
    torch.manual_seed(0)
    block = Block(256).cuda()
    block.qkv = Int8Linear.from_linear(block.qkv)
    x, res, pos = inputs(8, 1, 256, torch.bfloat16)
    with torch.no_grad():
        block(x, res, pos)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = block(x, res, pos)
        for step in range(3):
            x.copy_(torch.randn_like(x))
            pos.add_(1)
            graph.replay()
            for a, b in zip(held, block(x, res, pos)):
                assert torch.equal(a, b)


def test_training_chain_gradients():
    """float32 training of the chain: autograd through the operators against autograd through the CPU formulas.  Both
    are float32 within 2^-24 * terms of the same values; the longest chain is two norms (256 terms), a projection
    (256) and a sum over 150 rows, so 1e-4 of each gradient's scale is several times the bound."""
    torch.manual_seed(0)
    block = Block(256)
    x, res, pos = inputs(2, 75, 256, torch.float32)
    outs = {}
    for dev in ("cpu", "cuda"):
        b = block.to(dev)
        xs, rs = x.to(dev).requires_grad_(), res.to(dev).requires_grad_()
        out = b(xs, rs, pos.to(dev))
        g = torch.Generator().manual_seed(9)
        seeds = [torch.randn(o.shape, generator=g).to(dev) for o in out]
        outs[dev] = [t.detach().cpu() for t in (*out, *torch.autograd.grad(out, [xs, rs, *b.parameters()], seeds))]
    for a, b in zip(outs["cuda"], outs["cpu"]):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())


def test_a_captured_training_step_follows_an_eager_one():
    """An eager step, its graph dropped, then the same step captured and replayed."""
    torch.manual_seed(0)
    block = Block(128).cuda()
    x, res, pos = inputs(2, 30, 128, torch.bfloat16)
    block.qkv.to(torch.bfloat16)
    params = list(block.parameters())

    def step():
        out = block(x, res, pos)
        return torch.autograd.grad(sum(o.float().square().mean() for o in out), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b in zip(held, want):
        assert float((a.float() - b.float()).abs().max()) <= 1e-2 * float(b.float().abs().max())
