"""The rotary kernels on overlapping and shared views.  The one-axis embedding rounds each operation, so a view gives the
bits of its copy.  The multi-axis one is held to the rotation in 64 bits: a view may be read in narrower pieces than its
copy, by a kernel in which a product of x cos - y sin is rounded before the sum or (in a fused operation) not, half a
step of at most |x| or |y|, which its bound of 10 such units counts."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.rope import apply_multi_axis_rotary, apply_rotary_pos_emb, axis_of_pairs
from tests.bounds import assert_within, rotate_exact, rotate_slack, turns_exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("strides", [(400, 16, 1, 1), (500, 1, 16, 1), (500, 1, 0, 1), (0, 0, 0, 1), (1, 1, 1, 1),
                                     (640, 160, 1, 10), (0, 0, 0, 0)])
def test_views_give_the_results_of_copies(strides, dt):
    g = torch.Generator().manual_seed(3)
    base = torch.randn(3000, generator=g).to(dt).cuda()
    q = torch.as_strided(base, (2, 4, 10, 16), strides)
    k = torch.as_strided(base[7:], (2, 4, 10, 16), strides)
    pos = torch.randint(0, 500, (2, 2, 10), generator=g).cuda()
    inv = torch.rand(8, generator=g).cuda()
    cos, sin = (torch.rand(10, 16, generator=g).to(dt).cuda() for _ in range(2))
    leaves = [torch.randn(2, 4, 10, 16, generator=g).to(dt).cuda().requires_grad_() for _ in range(2)]
    copies = q.contiguous(), k.contiguous()

    turn = turns_exact(pos, inv, axis_of_pairs((5, 3)))
    for got, t in zip(apply_multi_axis_rotary(q, k, pos, inv, (5, 3)), (q, k)):
        assert_within(got, rotate_exact(t, turn), rotate_slack(t, 8), f"{strides}")
    out = apply_multi_axis_rotary(*leaves, pos, inv, (5, 3))
    for got, t in zip(torch.autograd.grad(out, leaves, (q, k)), (q, k)):
        assert_within(got, rotate_exact(t, turn.conj()), rotate_slack(t, 8), f"{strides} backward")

    for a, b in zip(apply_rotary_pos_emb(q, k, cos, sin), apply_rotary_pos_emb(*copies, cos, sin)):
        assert torch.equal(a, b)
    got, want = (torch.autograd.grad(apply_rotary_pos_emb(*leaves, cos, sin), leaves, g) for g in ((q, k), copies))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
