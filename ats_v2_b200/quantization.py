"""Linear factory of the expert projections (counterpart of
ats/model/quantization.py:40-193).

``make_linear(in, out, quantization, bias)`` returns a plain ``nn.Linear``
for "none" and a ``QuantizedLinear`` otherwise.  ``QuantizedLinear`` is an
``nn.Linear`` subclass (so state-dict keys stay ``weight``/``bias``) whose
"int8" mode fake-quantises the weight (per tensor, symmetric) and the input
activations (per tensor, affine) to the int8 range on every forward with
torch.ao's FakeQuantize modules and moving-average min/max observers, with
straight-through gradients -- quantization-aware training as the reference
describes it.  "fp8" needs torchao, which this image does not ship: it raises
ImportError, as the reference does without a usable backend.

These modules run their own torch forward; the sm_100a expert kernels take
plain weights and refuse quantized experts (``ffn.require_plain_weights``).

For inference, ``Int8Linear`` holds the weight in 8-bit integers and multiplies
integers: ``quantize_int8`` gives int8 rows with a float32 scale each, and
``int8_linear`` quantises its input per token and runs the integer product on
the sm_100a kernels (not in the reference, whose int8 mode imitates the
rounding in floating point).  Its scales are finer than those that
``QuantizedLinear`` trains with (see ``Int8Linear``): serving a trained layer
this way is a quantisation of its float weights, not the trained rounding.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from ats_v2_b200 import _lib

MODES = ("none", "int8", "fp8")


class QuantizedLinear(nn.Linear):
    def __init__(self, in_features: int, out_features: int, quantization: str = "none", bias: bool = False) -> None:
        if quantization not in MODES:
            raise ValueError(f"Unknown quantization mode '{quantization}'. Fix: use one of 'none', 'int8', 'fp8'.")
        super().__init__(in_features, out_features, bias=bias)
        self.quantization = quantization
        if quantization == "int8":
            from torch.ao.quantization import FakeQuantize, MovingAverageMinMaxObserver

            def fq(scheme):
                return FakeQuantize(observer=MovingAverageMinMaxObserver, quant_min=-128, quant_max=127,
                                    dtype=torch.qint8, qscheme=scheme)

            self._weight_fake_quant = fq(torch.per_tensor_symmetric)
            self._act_fake_quant = fq(torch.per_tensor_affine)
        elif quantization == "fp8":
            try:
                import torchao  # noqa: F401
            except ImportError as exc:
                raise ImportError("FP8 training requires torchao (the supported backend). Install with: "
                                  "pip install torchao") from exc
            raise NotImplementedError("fp8 QuantizedLinear: torchao conversion is not built in ats_v2_b200")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.quantization == "int8":
            return F.linear(self._act_fake_quant(x), self._weight_fake_quant(self.weight), self.bias)
        return F.linear(x, self.weight, self.bias)


def make_linear(in_features: int, out_features: int, quantization: str = "none", bias: bool = False) -> nn.Linear:
    if quantization == "none":
        return nn.Linear(in_features, out_features, bias=bias)
    return QuantizedLinear(in_features, out_features, quantization=quantization, bias=bias)


INT8_MAX_FEATURES = 131072  # the int32 sum of 127 * 128 * in_features stays below 2^31


def _torch_quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_int8`` in torch operations on a [rows, features] tensor: what CPU tensors run."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    finite = amax.isfinite()
    amax = amax.clamp_min(2.0 ** -100)
    full = torch.full_like(amax, 127)  # a quotient of two tensors is rounded once, one with a number may not be
    q = torch.where(finite, torch.round(x * (full / amax)), torch.zeros_like(x)).clamp(-127, 127)
    return q.to(torch.int8), torch.where(finite, amax / full, torch.nan)[:, 0]


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., features] as rows whose elements are consecutive."""
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit quantisation of the rows of x [..., features] (float32 or bfloat16, 1 to
    131072 features): int8 values of x's shape in [-127, 127] and a float32 scale for each row,
    ``q = round(x * (127 / amax))``, ``scale = amax / 127`` in float32 with ties to even, where
    ``amax`` is the row's largest magnitude (at least 2^-100).  A row that holds an infinity or
    NaN gets zeros and a NaN scale.  For a weight [out_features, in_features] the scales are per
    output channel.  Rows of the result start at multiples of 16 bytes, as ``int8_linear`` reads
    them.  Not differentiable: the results have no graph, and forward-mode duals are refused."""
    if x.dim() < 1 or not 1 <= x.shape[-1] <= INT8_MAX_FEATURES:
        raise ValueError(f"quantize_int8: x must be [..., 1 to {INT8_MAX_FEATURES} features], got {tuple(x.shape)}.")
    _lib.refuse_tangents(x)
    lead, K = x.shape[:-1], x.shape[-1]
    x2 = _rows(x.detach())
    Kp = (K + 15) // 16 * 16
    if _lib.on_cpu("quantize_int8", x):
        code = _lib.dtype_code(x.dtype)  # the same types as on CUDA
        q = torch.zeros((x2.shape[0], Kp), dtype=torch.int8)
        q[:, :K], scale = _torch_quantize_int8(x2)
    else:
        code = _lib.dtype_code(x.dtype)
        q = x2.new_empty((x2.shape[0], Kp), dtype=torch.int8)
        scale = x2.new_empty(x2.shape[0], dtype=torch.float32)
        with _lib.device_of(x):
            _lib.call("ats_int8_quantize", x2.data_ptr(), x2.stride(0), code, q.data_ptr(), Kp, scale.data_ptr(),
                      x2.shape[0], K, _lib.stream_of(x))
    return q[:, :K] if len(lead) == 1 else q[:, :K].view(*lead, K), scale.view(lead)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ (weight * scale[:, None]).T + bias`` as an integer product.  x [..., in_features]
    (float32 or bfloat16) is quantised per token as ``quantize_int8`` does; ``weight`` is int8
    [out_features, in_features] with a float32 ``scale`` [out_features], as ``quantize_int8``
    returns them; ``bias`` [out_features] is float32 or bfloat16.  The products are summed
    exactly in int32, then scaled in float32 and rounded once to x's dtype.  A token that holds
    an infinity or NaN gives NaN outputs.  Weight rows should start at multiples of 16 bytes, as
    ``quantize_int8`` lays them out; others are copied on every call.  Inference only: tensors
    that need a gradient and forward-mode duals are refused."""
    if weight.dim() != 2 or weight.dtype != torch.int8:
        raise TypeError(f"int8_linear: weight must be int8 [out_features, in_features], got {weight.dtype} "
                        f"{tuple(weight.shape)}. Fix: pass quantize_int8(weight).")
    N, K = weight.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"int8_linear: x's last dim must be in_features {K}, got {tuple(x.shape)}.")
    if N < 1 or not 1 <= K <= INT8_MAX_FEATURES:
        raise ValueError(f"int8_linear: weight {tuple(weight.shape)} must have at least one output and 1 to "
                         f"{INT8_MAX_FEATURES} input features.")
    if scale.shape != (N,) or scale.dtype != torch.float32:
        raise ValueError(f"int8_linear: scale must be float32 [{N}], got {scale.dtype} {tuple(scale.shape)}.")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"int8_linear: bias shape {tuple(bias.shape)} must be ({N},).")
    if _lib.wants_grad(x, scale, bias):
        raise NotImplementedError("int8_linear has no gradient. Fix: call it under torch.no_grad(), or train with "
                                  "QuantizedLinear.")
    code = _lib.dtype_code(x.dtype)
    bias_code = _lib.dtype_code(bias.dtype) if bias is not None else 0
    x2 = _rows(x)
    M = x2.shape[0]
    if _lib.on_cpu("int8_linear", x, weight, scale, bias):
        q, sx = _torch_quantize_int8(x2)
        y = (q.double() @ weight.double().t()).float() * (sx[:, None] * scale)  # exact: integers below 2^53
        y = (y if bias is None else y + bias.float()).to(x.dtype)
        return y.view(*x.shape[:-1], N)
    ldw = weight.stride(0) if N > 1 else (K + 15) // 16 * 16  # a single row has no next one
    if (weight.stride(1) != 1 and K > 1) or ldw % 16 != 0 or ldw < K or weight.data_ptr() % 16 != 0:
        ldw = (K + 15) // 16 * 16
        weight = torch.empty((N, ldw), dtype=torch.int8, device=weight.device)[:, :K].copy_(weight)
    scale = scale.contiguous()
    bias = bias.contiguous() if bias is not None else None
    y = x.new_empty((*x.shape[:-1], N))
    with _lib.device_of(x):
        wsb = _lib.query("ats_int8_linear_workspace_bytes", M, N, K)
        ws = x.new_empty(wsb, dtype=torch.uint8) if wsb else None
        _lib.call("ats_int8_linear", x2.data_ptr(), x2.stride(0), code, weight.data_ptr(), ldw,
                  scale.data_ptr(), _lib.ptr(bias), bias_code, y.data_ptr(), M, N, K, _lib.ptr(ws), wsb,
                  _lib.stream_of(x))
    return y


class Int8Linear(nn.Module):
    """A Linear for inference with 8-bit weights: buffers ``weight`` (int8), ``scale`` (float32,
    per output channel) and ``bias``; ``forward`` is ``int8_linear``.  ``from_linear`` quantises
    the float weight of an ``nn.Linear``.

    A ``QuantizedLinear`` is an ``nn.Linear`` too, but the result does not round as its training
    did: here each output channel and each token has a symmetric scale of its own, where it
    imitates one symmetric scale for the whole weight and one affine range, observed over many
    batches, for all activations.  Its observers are dropped."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False) -> None:
        super().__init__()
        if in_features < 1 or in_features > INT8_MAX_FEATURES or out_features < 1:
            raise ValueError(f"Int8Linear requires 1 to {INT8_MAX_FEATURES} in_features and positive out_features, "
                             f"got {in_features} and {out_features}.")
        self.in_features = in_features
        self.out_features = out_features
        self.weight: torch.Tensor
        self.scale: torch.Tensor
        self.register_buffer("weight", self._laid_out(torch.zeros((out_features, in_features), dtype=torch.int8)))
        self.register_buffer("scale", torch.ones(out_features))
        self.register_buffer("bias", torch.zeros(out_features) if bias else None)

    @staticmethod
    def _laid_out(weight: torch.Tensor) -> torch.Tensor:
        """weight with rows that start at multiples of 16 bytes."""
        N, K = weight.shape
        if weight.stride(1) == 1 and weight.stride(0) % 16 == 0 and weight.stride(0) >= K and \
                weight.data_ptr() % 16 == 0:
            return weight
        return torch.zeros((N, (K + 15) // 16 * 16), dtype=weight.dtype, device=weight.device)[:, :K].copy_(weight)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        if not isinstance(linear, nn.Linear):
            raise TypeError(f"Int8Linear.from_linear takes an nn.Linear, got {type(linear).__name__}.")
        new = cls(linear.in_features, linear.out_features, bias=linear.bias is not None)
        new.weight, new.scale = quantize_int8(linear.weight.detach())
        new.bias = linear.bias.detach().clone() if linear.bias is not None else None
        return new

    def _apply(self, fn, recurse=True):  # moves keep the scales float32 and the rows aligned
        old = self.scale
        super()._apply(fn, recurse)
        self.scale = self.scale.float() if old.is_meta else old.to(device=self.scale.device)
        self.weight = self._laid_out(self.weight)
        return self

    def _load_from_state_dict(self, *args, **kwargs):  # assign=True takes a weight laid out in any way
        super()._load_from_state_dict(*args, **kwargs)
        self.weight = self._laid_out(self.weight)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int8_linear(x, self.weight, self.scale, self.bias)
