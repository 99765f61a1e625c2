"""The block operators (double norm, multi-axis rotary, 8-bit projection) on CPU tensors, and what they refuse.  No
launch happens: arguments are checked before the library is asked."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200 import _lib
from ats_v2_b200.norm_fused import fused_sandwich_norm
from ats_v2_b200.quantization import Int8Linear, int8_linear, quantize_int8
from ats_v2_b200.rope import MultiAxisRotaryEmbedding, apply_multi_axis_rotary, axis_of_pairs
from tests.bounds import (INT8_SLACK, assert_within, int8_exact, rotate_exact, rotate_slack, sandwich_exact,
                          sandwich_slack, turns_exact)


def test_sandwich_norm_formula_and_gradients():
    g = torch.Generator().manual_seed(0)
    x, res, dh, ds = (torch.randn(2, 3, 20, generator=g) for _ in range(4))
    wp, wn = torch.rand(20, generator=g), torch.rand(20, generator=g)
    gate = torch.randn(2, 1, 20, generator=g)
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gate)]
    out = fused_sandwich_norm(x, res, wp, wn, gate=gate, residual_scale=0.9, eps=1e-5)
    grads = torch.autograd.grad(out, leaves, (dh, ds))
    e = sandwich_exact(x, res, wp, wn, gate, 0.9, 1e-5, dh, ds)
    for name, t in zip(("h", "s", "dx", "dres", "dwp", "dwn", "dgate"), (*out, *grads)):
        assert_within(t.detach(), e[name][0], sandwich_slack(20, 6) * e[name][1], name)


def test_sandwich_norm_refusals():
    x, w = torch.randn(2, 3, 8), torch.ones(8)
    for bad in (dict(residual=torch.randn(2, 3, 7)), dict(post_weight=torch.ones(7)), dict(pre_weight=torch.ones(1, 8)),
                dict(gate=torch.ones(3, 8)), dict(gate=torch.ones(1, 3, 8)), dict(gate=torch.ones(2, 3, 1)),
                dict(gate=torch.ones(2, 2, 8)), dict(x=torch.tensor(1.0), residual=torch.tensor(1.0))):
        with pytest.raises(ValueError, match="fused_sandwich_norm"):
            fused_sandwich_norm(**{**dict(x=x, residual=x, post_weight=w, pre_weight=w), **bad})
    with pytest.raises(TypeError, match="residual dtype"):
        fused_sandwich_norm(x, x.bfloat16(), w, w)
    with pytest.raises(TypeError, match="pre_weight dtype"):
        fused_sandwich_norm(x, x, w, w.bfloat16())


def test_axis_of_pairs():
    assert axis_of_pairs((2, 1, 3)) == bytes([0, 0, 1, 2, 2, 2])
    assert axis_of_pairs((2, 1, 3), True) == bytes([0, 1, 2, 0, 2, 2])
    assert axis_of_pairs((24, 20, 20), True) == bytes([0, 1, 2] * 20 + [0] * 4)
    for bad in ((), (0, 0), (-1, 5), (257,), (1.5,)):
        with pytest.raises(ValueError, match="sections"):
            axis_of_pairs(bad)


@pytest.mark.parametrize("interleaved", [False, True])
def test_multi_axis_rotary_formula_and_gradients(interleaved):
    g = torch.Generator().manual_seed(1)
    q, gq = (torch.randn(2, 3, 5, 14, generator=g) for _ in range(2))
    pos = torch.randint(0, 10 ** 6, (2, 2, 5), generator=g)
    inv = torch.rand(6, generator=g)
    q.requires_grad_()
    qo, ko = apply_multi_axis_rotary(q, None, pos, inv, (4, 2), interleaved)
    (dq,) = torch.autograd.grad(qo, q, gq)
    turn = turns_exact(pos, inv, axis_of_pairs((4, 2), interleaved))
    assert ko is None
    assert_within(qo.detach(), rotate_exact(q, turn), rotate_slack(q, 6))
    assert_within(dq, rotate_exact(gq, turn.conj()), rotate_slack(gq, 6))


def test_multi_axis_rotary_refusals():
    q, pos, inv = torch.randn(1, 2, 3, 8), torch.zeros(2, 1, 3, dtype=torch.int64), torch.ones(4)
    ok = dict(q=q, k=None, positions=pos, inv_freq=inv, sections=(2, 2))
    for bad in (dict(q=q[0]), dict(sections=(4, 4)), dict(k=torch.randn(1, 2, 4, 8)), dict(k=torch.randn(2, 2, 3, 8)),
                dict(positions=pos[:1]), dict(positions=pos[..., :2]), dict(inv_freq=torch.ones(5)),
                dict(inv_freq=inv.double()), dict(sections=(4,))):
        with pytest.raises(ValueError):
            apply_multi_axis_rotary(**{**ok, **bad})
    for bad in (dict(positions=pos.double()), dict(k=q.bfloat16())):
        with pytest.raises(TypeError):
            apply_multi_axis_rotary(**{**ok, **bad})
    with pytest.raises(NotImplementedError):
        apply_multi_axis_rotary(**{**ok, "inv_freq": inv.clone().requires_grad_()})
    with pytest.raises(ValueError):
        MultiAxisRotaryEmbedding(8, (2, 3))


def test_int8_linear_formula():
    g = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(3, 2, 50, generator=g), torch.randn(7, 50, generator=g), torch.randn(7, generator=g)
    wq, ws = quantize_int8(w)
    assert wq.shape == (7, 50) and wq.stride(0) == 64
    assert bool(((wq.double() * ws.double()[:, None] - w.double()).abs() <= ws.double()[:, None] * (0.5 + 1e-4)).all())
    y = int8_linear(x, wq, ws, b)
    e, mag = int8_exact(x.view(6, 50), wq, ws, b)
    assert_within(y.view(6, 7), e, INT8_SLACK * mag)


def test_int8_refusals():
    x, (wq, ws) = torch.randn(3, 50), quantize_int8(torch.randn(7, 50))
    with pytest.raises(TypeError, match="int8"):
        int8_linear(x, wq.float(), ws)
    for bad in (dict(x=x[:, :49]), dict(scale=ws[:6]), dict(scale=ws.double()), dict(bias=torch.ones(6)),
                dict(weight=wq[:0], scale=ws[:0])):
        with pytest.raises(ValueError, match="int8_linear"):
            int8_linear(**{**dict(x=x, weight=wq, scale=ws), **bad})
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        int8_linear(x.half(), wq, ws)
    with pytest.raises(NotImplementedError, match="no gradient"):
        int8_linear(x.clone().requires_grad_(), wq, ws)
    with torch.no_grad():
        assert int8_linear(x.clone().requires_grad_(), wq, ws).shape == (3, 7)
    with pytest.raises(ValueError):
        quantize_int8(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        Int8Linear(131073, 4)
    with pytest.raises(TypeError):
        Int8Linear.from_linear(torch.nn.LayerNorm(4))


def test_c_entry_points_check_arguments_on_the_host():
    lib = _lib.load()
    s3 = _lib.strides3(1, 1, 1)
    EB = _lib.ATS_EBADARG

    def axes(pairs=4, D=8, S=1, axis=b"\0\1\0\1", n=2, ptype=1, dt=1, pos=None):
        return lib.ats_rope_axes_apply(None, None, 1, s3, s3, None, None, 0, None, None, pos, ptype, s3, n, None, axis,
                                       pairs, 1, S, D, dt, 0, None)

    assert axes() == EB  # null pointers
    assert axes(S=0) == _lib.ATS_OK  # nothing to do
    for bad in (dict(pairs=5), dict(pairs=0), dict(pairs=257, D=1024), dict(axis=b"\0\1\2\1"), dict(n=0),
                dict(ptype=3), dict(dt=2), dict(axis=None)):
        assert axes(**bad) == EB, bad

    def norm(rows=4, H=8, dt=1, wdt=0, gate=None, span=0):
        return lib.ats_sandwich_norm_fwd(None, None, dt, None, None, wdt, gate, 0, span, 1.0, 1e-6, None, None, None,
                                         None, rows, H, None)

    for bad in (dict(), dict(rows=-1), dict(H=0), dict(dt=3), dict(wdt=9), dict(gate=16, span=3),
                dict(gate=16, span=0)):
        assert norm(**bad) == EB, bad
    assert lib.ats_sandwich_norm_bwd(None, None, None, None, 1, None, None, 0, None, 0, 0, 1.0, None, None, None, None,
                                     None, None, None, None, 0, 4, 8, None) == EB
    assert lib.ats_sandwich_norm_bwd_workspace_bytes(100, 64, 0) > 0
    assert lib.ats_sandwich_norm_bwd_workspace_bytes(100, 64, 7) == 0  # 7 rows do not divide 100

    def int8(M=2, N=4, K=32, ldw=32, dt=1, w=16, ws=None, wsb=0):
        return lib.ats_int8_linear(16, K, dt, w, ldw, 16, None, 0, 16, M, N, K, ws, wsb, None)

    assert int8() == EB and b"workspace" in lib.ats_last_error_message()
    assert int8(M=0) == _lib.ATS_OK
    for bad in (dict(K=131073, ldw=131088), dict(K=0), dict(N=0), dict(ldw=40), dict(ldw=16), dict(w=8), dict(dt=5),
                dict(M=-1)):
        assert int8(**bad) == EB, bad
    assert lib.ats_int8_quantize(16, 8, 0, 16, 4, 16, 2, 8, None) == EB  # rows of q shorter than K
