"""Every row counts once in ``fused_sandwich_norm``'s sums over rows.  Each row in turn has one non-zero gradient, in a
column of its own, so the weights' and the gate's gradient holds that row's term alone and is compared with it at the
bound of one row: a row lost, doubled or given to another gate row shows, however many rows there are."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.norm_fused import fused_sandwich_norm
from tests.bounds import assert_within, sandwich_slack

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS, A = 1.0, 0.7  # an eps of the rows' own size: narrow rows do not cancel


def rows_to_try(R, H, g):
    """All rows where a call takes many, else the first, the last and some between."""
    if R <= 8 * H:
        return torch.arange(R)
    some = torch.randint(0, R, (100,), generator=g)
    return torch.cat([torch.arange(50), some, torch.arange(R - 50, R)]).unique()


@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
@pytest.mark.parametrize("B,S,H,xd,wd", [
    (4, 2250, 1, "bf16", "f32"), (4, 2250, 6, "bf16", "f32"), (3, 700, 6, "f32", "f32"), (500, 3, 16, "bf16", "bf16"),
    (4, 625, 363, "bf16", "f32"), (2, 900, 519, "bf16", "bf16"), (6, 250, 1030, "f32", "f32"), (6, 250, 1030, "bf16", "f32"),
    (4, 300, 2509, "bf16", "f32"), (700, 2, 2048, "bf16", "f32"), (3, 341, 2048, "bf16", "f32"),
    (2, 600, 4096, "bf16", "f32"), (4, 225, 4097, "bf16", "f32"), (2, 310, 8192, "f32", "f32"),
    (3, 201, 8200, "bf16", "f32")])
def test_each_row_is_in_the_sums_once(B, S, H, xd, wd, gate):
    g = torch.Generator().manual_seed(B * S + H)

    def randn(*shape):
        return torch.randn(*shape, generator=g)

    shape = {None: None, "channel": (H,), "sequence": (B, 1, H), "token": (B, S, H)}[gate]
    x, res = (randn(B, S, H).to(TD[xd]).cuda() for _ in range(2))
    wp, wn = ((1 + 0.2 * randn(H)).to(TD[wd]).cuda() for _ in range(2))
    gt = None if shape is None else (1 + 0.3 * randn(*shape)).to(TD[xd]).cuda()
    leaves = [t.requires_grad_() for t in (wp, wn, gt) if t is not None]
    out = fused_sandwich_norm(x, res, wp, wn, gate=gt, residual_scale=A, eps=EPS)

    with torch.no_grad():  # the terms of every row and column in 64 bits, and the same on absolute values
        X, W, G = x.double(), wp.double(), 1.0 if gt is None else gt.double()
        rx = (X.square().mean(-1, keepdim=True) + EPS).rsqrt()
        s, sm = A * res.double() + G * W * X * rx, (A * res.double()).abs() + (G * W * X * rx).abs()
        rs = (s.square().mean(-1, keepdim=True) + EPS).rsqrt()
        k = (sm.square().mean(-1, keepdim=True) * rs * rs + 1)
        pre, pre_mag = (s * rs).view(-1, H), (sm * rs * k).view(-1, H)
        post = (G * X * rx).expand(B, S, H).reshape(-1, H)
        gates = (W * X * rx).view(-1, H)
    slack = sandwich_slack(H, 1)
    rows = rows_to_try(B * S, H, g)
    for part in rows.split(H):
        cols = torch.randperm(H, generator=g)[:part.numel()]
        grad = torch.zeros(B * S, H)
        grad[part, cols] = 1 + torch.rand(part.numel(), generator=g)
        grad = grad.to(TD[xd]).cuda().view(B, S, H)
        at = part.cuda(), cols.cuda()
        d, zero = grad.view(-1, H)[at].double(), torch.zeros_like(grad)

        def alone(values):
            return torch.zeros(H, dtype=torch.float64, device="cuda").index_put((at[1],), values)

        dwn = torch.autograd.grad(out, leaves, (grad, zero), retain_graph=True)[1]
        assert_within(dwn, alone(d * pre[at]), slack * alone(d * pre_mag[at]), f"dwn {B} {S} {H} {gate}")
        got = torch.autograd.grad(out, leaves, (zero, grad), retain_graph=True)
        assert_within(got[0], alone(d * post[at]), slack * alone((d * post[at]).abs()), f"dwp {B} {S} {H} {gate}")
        assert not got[1].any()
        if gt is not None:
            want = torch.zeros(B * S, H, dtype=torch.float64, device="cuda").index_put(at, d * gates[at]).view(B, S, H)
            want = {"channel": lambda t: t.sum((0, 1)), "sequence": lambda t: t.sum(1, keepdim=True),
                    "token": lambda t: t}[gate](want)  # one term in each sum: exact
            assert_within(got[2], want, slack * want.abs(), f"dgate {B} {S} {H} {gate}")
