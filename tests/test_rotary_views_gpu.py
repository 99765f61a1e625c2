"""The rotary kernels on overlapping and shared views: the results of a copy."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.rope import apply_multi_axis_rotary, apply_rotary_pos_emb

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
    for call in (lambda *t: apply_multi_axis_rotary(*t, pos, inv, (5, 3)),
                 lambda *t: apply_rotary_pos_emb(*t, cos, sin)):
        for a, b in zip(call(q, k), call(q.contiguous(), k.contiguous())):
            assert torch.equal(a, b)
        leaves = [torch.randn(2, 4, 10, 16, generator=g).to(dt).cuda().requires_grad_() for _ in range(2)]
        got = torch.autograd.grad(call(*leaves), leaves, (q, k))
        want = torch.autograd.grad(call(*leaves), leaves, (q.contiguous(), k.contiguous()))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
