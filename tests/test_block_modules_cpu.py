"""The block operators' modules as a model's loading code treats them: made without memory, materialised, cast, loaded."""

from __future__ import annotations

import copy

import pytest
import torch

from ats_v2_b200.quantization import Int8Linear, QuantizedLinear
from ats_v2_b200.rope import MultiAxisRotaryEmbedding


@pytest.mark.parametrize("cast", [None, torch.bfloat16, torch.float64])
def test_rotary_made_on_the_meta_device(cast):
    want = MultiAxisRotaryEmbedding(16, (5, 3), theta=500.0)
    with torch.device("meta"):
        emb = MultiAxisRotaryEmbedding(16, (5, 3), theta=500.0)
    assert emb.inv_freq.is_meta
    if cast is not None:
        emb = emb.to(cast)
        assert emb.inv_freq.is_meta and emb.inv_freq.dtype == torch.float32
    emb = torch.nn.ModuleList([emb]).to_empty(device="cpu")[0]
    assert torch.equal(emb.inv_freq, want.inv_freq)  # in no state dict: it is there without one
    q, pos = torch.randn(2, 3, 4, 16), torch.randint(0, 50, (2, 2, 4))
    assert torch.equal(emb(q, None, pos)[0], want(q, None, pos)[0])


def test_rotary_casts_keep_its_frequencies():
    emb = MultiAxisRotaryEmbedding(16, (5, 3))
    emb.inv_freq *= 0.5  # values of the user's own
    want = emb.inv_freq.clone()
    for m in (emb.half(), copy.deepcopy(emb).bfloat16(), emb.double(), emb.to("cpu"), emb.to_empty(device="cpu")):
        assert m.inv_freq.dtype == torch.float32 and torch.equal(m.inv_freq, want)


@pytest.mark.parametrize("K", [33, 48])
@pytest.mark.parametrize("cast", [None, torch.bfloat16])
def test_int8_linear_made_on_the_meta_device(K, cast):
    want = Int8Linear.from_linear(torch.nn.Linear(K, 5))
    with torch.device("meta"):
        lin = Int8Linear(K, 5, bias=True)
    if cast is not None:
        lin = lin.to(cast)
        assert lin.scale.is_meta and lin.scale.dtype == torch.float32
    lin = torch.nn.ModuleList([lin]).to_empty(device="cpu")[0]
    assert not lin.weight.is_meta and lin.weight.stride() == (48, 1)
    lin.load_state_dict(want.state_dict())
    x = torch.randn(3, K)
    assert lin.scale.dtype == torch.float32
    assert torch.equal(lin(x), want(x)) or cast is not None  # a cast rounds the bias, as it does a Linear's
    assert torch.equal(lin.weight, want.weight) and torch.equal(lin.scale, want.scale)


def test_int8_linear_casts_keep_its_scales():
    lin = Int8Linear.from_linear(torch.nn.Linear(40, 5))
    scale, weight = lin.scale.clone(), lin.weight.clone()
    for m in (lin.half(), copy.deepcopy(lin).bfloat16(), lin.double(), lin.to("cpu")):
        assert m.scale.dtype == torch.float32 and torch.equal(m.scale, scale) and torch.equal(m.weight, weight)
        assert m.weight.stride(0) % 16 == 0


@pytest.mark.parametrize("meta", [False, True])
def test_an_assigned_weight_is_laid_out_once(meta):
    """int8_linear copies a weight whose rows do not start at multiples of 16 bytes: not on every call of a module."""
    want = Int8Linear.from_linear(torch.nn.Linear(33, 7))
    buf = torch.empty(7 * 33 + 1, dtype=torch.int8)[1:].view(7, 33)
    wide = torch.empty(7 * 48 + 1, dtype=torch.int8)[1:].view(7, 48)[:, :33]  # rows of 48 bytes from an odd address
    for weight in (want.weight.contiguous(), want.weight.t().contiguous().t(), buf.copy_(want.weight),
                   wide.copy_(want.weight)):
        with torch.device("meta" if meta else "cpu"):
            lin = Int8Linear(33, 7, bias=True)
        lin.load_state_dict({**want.state_dict(), "weight": weight}, assign=True)
        assert lin.weight.stride() == (48, 1) and lin.weight.data_ptr() % 16 == 0
        assert torch.equal(lin.weight, want.weight)
        x = torch.randn(3, 33)
        assert torch.equal(lin(x), want(x))
        assert set(lin.state_dict()) == {"weight", "scale", "bias"}
    lin = Int8Linear(33, 7, bias=True)
    aligned = want.weight
    lin.load_state_dict({**want.state_dict(), "weight": aligned}, assign=True)
    assert lin.weight.data_ptr() == aligned.data_ptr()  # already so: taken as it is
    for floats in (torch.rand(7, 33), torch.rand(7, 48)[:, :33]):  # not an 8-bit weight: refused, never truncated
        wrong = Int8Linear(33, 7, bias=True)
        wrong.load_state_dict({**want.state_dict(), "weight": floats}, assign=True)
        with pytest.raises(TypeError, match="must be int8"):
            wrong(torch.randn(3, 33))
    with pytest.raises(RuntimeError, match="size mismatch"):
        lin.load_state_dict({**want.state_dict(), "weight": aligned[:, :32]}, assign=True)


def test_a_fake_quantised_layer_is_served_by_its_float_weight():
    """Not by the rounding it trained with: scales per channel and token, the observed ranges unused."""
    qat = QuantizedLinear(40, 6, "int8", bias=True)
    with torch.no_grad():
        qat.weight[0] *= 100  # the one scale of the whole weight, in training
    qat.train()
    for _ in range(3):
        qat(50 * torch.randn(8, 40))  # moves the observed ranges
    plain = torch.nn.Linear(40, 6)
    plain.load_state_dict({"weight": qat.weight, "bias": qat.bias})
    served, want = Int8Linear.from_linear(qat), Int8Linear.from_linear(plain)
    x = torch.randn(3, 40)
    assert torch.equal(served(x), want(x)) and set(served.state_dict()) == {"weight", "scale", "bias"}
    off = (served.weight.double() * served.scale.double()[:, None] - qat.weight.detach().double()).abs()
    assert bool((off <= 0.5001 * served.scale.double()[:, None]).all())  # half a step of each channel's own scale
    assert float(served.scale[1:].max()) < 0.1 * float(served.scale[0])
