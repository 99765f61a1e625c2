"""Forward-mode derivatives of the block operators: right where torch operations compute them (CPU tensors), refused
where a kernel would lose the tangent.  The kernels' path is taken on CPU with every launch turned into a failure."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from ats_v2_b200 import _lib
from ats_v2_b200.norm_fused import _SandwichNormFn, fused_sandwich_norm
from ats_v2_b200.quantization import int8_linear, quantize_int8
from ats_v2_b200.rope import _MultiAxisRotaryFn, apply_multi_axis_rotary


@pytest.fixture
def kernels(monkeypatch):
    def launched(*args):
        raise AssertionError("a kernel was launched")

    monkeypatch.setattr(_lib, "on_cpu", lambda *a: False)
    for name in ("call", "query", "stream_of", "device_of"):
        monkeypatch.setattr(_lib, name, launched)


X, W = torch.randn(2, 3, 8), torch.rand(8)
Q, POS, INV = torch.randn(1, 2, 3, 8), torch.zeros(2, 1, 3, dtype=torch.int64), torch.ones(4)
WQ, WS = quantize_int8(torch.randn(5, 8))

CALLS = {
    "norm x": (lambda t: fused_sandwich_norm(t, X, W, W), X),
    "norm residual": (lambda t: fused_sandwich_norm(X, t, W, W), X),
    "norm post": (lambda t: fused_sandwich_norm(X, X, t, W), W),
    "norm pre": (lambda t: fused_sandwich_norm(X, X, W, t), W),
    "norm gate": (lambda t: fused_sandwich_norm(X, X, W, W, gate=t), W),
    "rotary q": (lambda t: apply_multi_axis_rotary(t, None, POS, INV, (2, 2)), Q),
    "rotary k": (lambda t: apply_multi_axis_rotary(Q, t, POS, INV, (2, 2)), Q),
    "rotary frequencies": (lambda t: apply_multi_axis_rotary(Q, None, POS, t, (2, 2)), INV),
    "rotary positions": (lambda t: apply_multi_axis_rotary(Q, None, t, INV, (2, 2)), POS.float()),
    "linear x": (lambda t: int8_linear(t, WQ, WS), X),
    "linear scale": (lambda t: int8_linear(X, WQ, t), WS),
    "linear bias": (lambda t: int8_linear(X, WQ, WS, t), WS),
    "quantise": (quantize_int8, X),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_duals_are_refused_before_a_launch(kernels, name, grad):
    call, t = CALLS[name]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(AssertionError, match="launched"):  # not dual: as ever
            call(t)


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_refused_before_a_launch(kernels, name):
    call, t = CALLS[name]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("fn,n", [(_SandwichNormFn, 2), (_MultiAxisRotaryFn, 2)])
def test_a_backward_of_duals_is_refused(kernels, fn, n):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(X, torch.ones_like(X))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            fn.backward(None, dual, *[None] * (n - 1))


@pytest.mark.parametrize("name", [n for n in CALLS if n[:4] in ("norm", "rota") and "freq" not in n and "pos" not in n]
                         + ["norm post"])
def test_cpu_tensors_have_the_tangent_of_the_differences(name):
    """Central differences in float32: a step of 2^-7 leaves 2^-14 of the third derivative and 2^-24 / 2^-7 of the
    value, each below 1e-3 of the values of order 1 to 10 here."""
    call, t = CALLS[name]
    d = torch.randn(t.shape, generator=torch.Generator().manual_seed(0))
    with forward_ad.dual_level():
        got = [forward_ad.unpack_dual(o).tangent for o in call(forward_ad.make_dual(t, d)) if o is not None]
    up, down = ([o for o in call(t + s * 2.0 ** -7 * d) if o is not None] for s in (1, -1))
    for g, a, b in zip(got, up, down):
        want = (a - b) * 2.0 ** 6
        if g is None:  # q's rotation does not depend on k, nor k's on q
            assert not want.any()
        else:
            assert float((g - want).abs().max()) <= 5e-3 * (1 + float(want.abs().max()))
