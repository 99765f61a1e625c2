"""What the rotary kernels are given for views of every kind: last axes that are consecutive, in and out."""

from __future__ import annotations

import contextlib

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

    def call(name, q, q_out, heads, q_strides, q_out_strides, k, k_out, k_heads, k_strides, k_out_strides, *rest):
        seen.extend([(q_out, tuple(q_strides), tuple(q_out_strides)), (k_out, tuple(k_strides), tuple(k_out_strides))])

    for what, stub in (("on_cpu", lambda *a: False), ("require_cuda", lambda *a: None), ("call", call),
                       ("stream_of", lambda t: 0), ("device_of", lambda t: contextlib.nullcontext())):
        monkeypatch.setattr(_lib, what, stub)
    q, k = view(name), view(name)
    if grad:
        q, k = q.requires_grad_(), k.requires_grad_()
    if axes == "one":
        out = rope.apply_rotary_pos_emb(q, k, torch.ones(4, 8), torch.ones(4, 8))
    else:
        out = rope.apply_multi_axis_rotary(q, k, torch.zeros(2, 4, dtype=torch.int64), torch.ones(4), (2, 2))
    if grad:
        out += torch.autograd.grad(out, (q, k), (view(name), view(name)))
    assert len(out) == len(seen) == (4 if grad else 2)
    for dst, (ptr, src_strides, dst_strides) in zip(out, seen):
        assert dst.data_ptr() == ptr and dst.stride() == (*dst_strides, 1)
        places = (torch.tensor(dst.stride()) * torch.cartesian_prod(*map(torch.arange, dst.shape))).sum(1)
        assert places.unique().numel() == dst.numel()  # every value has a place of its own
        if VIEWS[name][3] == 1:
            assert src_strides == VIEWS[name][:3]  # read where it is
        if name in ("dense", "heads inside"):
            assert dst_strides == src_strides
