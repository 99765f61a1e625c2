"""What the rotary kernels are given for views of every kind: last axes that are consecutive, in and out."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200 import _lib, rope

VIEWS = {  # strides of [2, 3, 4, 8] (batch, heads, seq, head_dim)
    "dense": (96, 32, 8, 1), "heads inside": (96, 8, 24, 1), "windows over the tokens": (40, 12, 1, 1),
    "windows over the heads": (50, 1, 8, 1), "both, shared": (50, 1, 0, 1), "all shared": (0, 0, 0, 1),
    "transposed": (96, 32, 1, 4), "one number": (0, 0, 0, 0),
}


def view(name):
    return torch.as_strided(torch.arange(400.), (2, 3, 4, 8), VIEWS[name])


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", VIEWS)
@pytest.mark.parametrize("axes", ["one", "several"])
def test_inputs_and_results_have_consecutive_heads(monkeypatch, axes, name, grad):
    seen = []
    monkeypatch.setattr(_lib, "on_cpu", lambda *a: False)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    for fn in ("_launch", "_launch_axes"):  # (q, q_out, k, k_out, ...)
        monkeypatch.setattr(rope, fn, lambda *a: seen.extend(zip(a[0:4:2], a[1:4:2])))
    q, k = view(name), view(name)
    if grad:
        q, k = q.requires_grad_(), k.requires_grad_()
    if axes == "one":
        out = rope.apply_rotary_pos_emb(q, k, torch.ones(4, 8), torch.ones(4, 8))
    else:
        out = rope.apply_multi_axis_rotary(q, k, torch.zeros(2, 4, dtype=torch.int64), torch.ones(4), (2, 2))
    if grad:
        torch.autograd.backward(out, (view(name), view(name)))
    assert len(seen) == (4 if grad else 2)
    for src, dst in seen:
        assert src.shape == dst.shape == (2, 3, 4, 8) and src.stride(-1) == dst.stride(-1) == 1
        places = (torch.tensor(dst.stride()) * torch.cartesian_prod(*map(torch.arange, dst.shape))).sum(1)
        assert places.unique().numel() == dst.numel()  # every value has a place of its own
        if name in ("dense", "heads inside"):
            assert dst.stride() == src.stride()
