"""Fused RMSNorm + residual on the sm_100a kernels -- mirror of
ats/model/norm_triton.py.

``fused_rmsnorm_residual(x, residual, weight, eps=1e-6)`` validates like the
reference (norm_triton.py:111-120) and computes the reference's PyTorch
formula (norm_triton.py:88-98), ``residual + (x*rsqrt(mean(x^2)+eps)).to(x.dtype)
* weight``, with torch's type promotion at each step, in one CUDA pass.
Unlike the reference's Triton kernel it is differentiable (x, residual and
weight).  ``_cuda_rmsnorm_residual`` is the kernel call without validation.

The reference's tests import three more names from this module
(tests/test_triton.py:19-25,142-149), kept here with the same meaning:
``HAS_TRITON`` says whether the fused GPU kernel is available (here: whether
the CUDA library is built; no Triton is involved), ``_triton_rmsnorm_residual``
is the fused kernel call, and ``_pytorch_rmsnorm_residual`` is the plain torch
formula those tests compare the kernel against.  ``fused_rmsnorm_residual``
runs that formula for CPU tensors, as the reference does
(norm_triton.py:121-123); CUDA tensors always take the kernel.
"""

from __future__ import annotations

import torch

from ats_v2_b200 import _lib

HAS_TRITON = _lib.LIB_PATH.exists()  # the reference's flag name: fused GPU kernel available


def _out_dtype(x: torch.Tensor, w: torch.Tensor) -> torch.dtype:
    return torch.promote_types(x.dtype, w.dtype)


class _RMSNormResidualFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        H = x.shape[-1]
        x2 = x.reshape(-1, H).contiguous()
        r2 = residual.reshape(-1, H).contiguous()
        w = weight.contiguous()
        out = torch.empty(x2.shape, dtype=_out_dtype(x, weight), device=x.device)
        _lib.call("ats_rmsnorm_residual_fwd", x2.data_ptr(), r2.data_ptr(), _lib.dtype_code(x.dtype),
                  w.data_ptr(), _lib.dtype_code(w.dtype), out.data_ptr(), x2.shape[0], H, float(eps),
                  _lib.stream_of(x))
        ctx.save_for_backward(x2, w)
        ctx.eps = eps
        ctx.shape = x.shape
        return out.view(x.shape)

    @staticmethod
    def backward(ctx, dout):
        x2, w = ctx.saved_tensors
        rows, H = x2.shape
        d2 = dout.reshape(rows, H).to(_out_dtype(x2, w)).contiguous()
        dx = torch.empty_like(x2)
        dres = torch.empty_like(x2)
        dw = torch.empty(H, dtype=w.dtype, device=w.device)
        ws_bytes = _lib.query("ats_rmsnorm_bwd_workspace_bytes", rows, H)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x2.device)
        _lib.call("ats_rmsnorm_residual_bwd", d2.data_ptr(), x2.data_ptr(), _lib.dtype_code(x2.dtype),
                  w.data_ptr(), _lib.dtype_code(w.dtype), dx.data_ptr(), dres.data_ptr(), dw.data_ptr(),
                  ws.data_ptr(), ws_bytes, rows, H, float(ctx.eps), _lib.stream_of(x2))
        return dx.view(ctx.shape), dres.view(ctx.shape), dw, None


def _cuda_rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                           eps: float) -> torch.Tensor:
    _lib.require_cuda("fused_rmsnorm_residual", x, residual, weight)
    if residual.dtype != x.dtype:
        raise TypeError(f"fused_rmsnorm_residual: residual dtype {residual.dtype} must equal x dtype {x.dtype}")
    return _RMSNormResidualFn.apply(x, residual, weight, eps)


# fused-kernel name of the reference module (tests/test_triton.py:142-149)
_triton_rmsnorm_residual = _cuda_rmsnorm_residual


def _pytorch_rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                              eps: float) -> torch.Tensor:
    """The torch formula of norm_triton.py:88-98, the comparison of the reference's kernel test."""
    xf = x.to(torch.float32)
    inv = torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)
    return residual + (xf * inv).to(x.dtype) * weight


def fused_rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                           eps: float = 1e-6) -> torch.Tensor:
    """``residual + rms_norm(x) * weight``: one memory pass on CUDA; the torch formula on CPU."""
    if x.shape != residual.shape:
        raise ValueError(
            f"fused_rmsnorm_residual: x shape {tuple(x.shape)} must match "
            f"residual shape {tuple(residual.shape)}."
        )
    if weight.shape[-1] != x.shape[-1]:
        raise ValueError(
            f"fused_rmsnorm_residual: weight last dim {weight.shape[-1]} must match "
            f"x last dim {x.shape[-1]}."
        )
    if _lib.on_cpu("fused_rmsnorm_residual", x, residual, weight):
        return _pytorch_rmsnorm_residual(x, residual, weight, eps)
    return _cuda_rmsnorm_residual(x, residual, weight, eps)


class _AddRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        H = x.shape[-1]
        a = x.reshape(-1, H).contiguous()
        b = residual.reshape(-1, H).contiguous()
        w = weight.contiguous()
        s = torch.empty_like(a)
        y = torch.empty_like(a)
        _lib.call("ats_add_rmsnorm_fwd", a.data_ptr(), b.data_ptr(), _lib.dtype_code(a.dtype), w.data_ptr(),
                  _lib.dtype_code(w.dtype), s.data_ptr(), y.data_ptr(), a.shape[0], H, float(eps),
                  _lib.stream_of(a))
        ctx.save_for_backward(s, w)
        ctx.eps = eps
        ctx.shape = x.shape
        return y.view(x.shape), s.view(x.shape)

    @staticmethod
    def backward(ctx, dy, ds_in):
        s, w = ctx.saved_tensors
        rows, H = s.shape
        dy2 = (dy if dy is not None else torch.zeros_like(s)).reshape(rows, H).to(s.dtype).contiguous()
        di = ds_in.reshape(rows, H).to(s.dtype).contiguous() if ds_in is not None else None
        ds = torch.empty_like(s)
        dw = torch.empty(H, dtype=w.dtype, device=w.device)
        wsb = _lib.query("ats_add_rmsnorm_bwd_workspace_bytes", rows, H)
        ws = torch.empty(wsb, dtype=torch.uint8, device=s.device)
        _lib.call("ats_add_rmsnorm_bwd", dy2.data_ptr(), s.data_ptr(), _lib.ptr(di), _lib.dtype_code(s.dtype),
                  w.data_ptr(), _lib.dtype_code(w.dtype), ds.data_ptr(), dw.data_ptr(), ws.data_ptr(), wsb, rows, H,
                  float(ctx.eps), _lib.stream_of(s))
        ds = ds.view(ctx.shape)
        return ds, ds, dw, None


def add_rmsnorm_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether the fused kernel covers this shape (16-byte rows of at most 512 chunks)."""
    H = x.shape[-1]
    n = 16 // x.element_size()
    return x.dtype in (torch.float32, torch.bfloat16) and weight.dtype in (torch.float32, torch.bfloat16) \
        and H % n == 0 and H // n <= 512


def fused_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``s = residual + x; (rms_norm(s) * weight, s)`` -- the post-attention residual add
    and RMSNorm of TransformerBlock.forward (ats/model/transformer.py:208-212), whose
    ``s`` is the block's next residual.  CUDA tensors: one kernel each way (the
    backward adds the gradient that reaches ``s`` from the next residual add, as
    autograd would).  CPU tensors: the reference's two torch operations."""
    if x.shape != residual.shape:
        raise ValueError(f"fused_add_rmsnorm: x shape {tuple(x.shape)} must match residual shape "
                         f"{tuple(residual.shape)}.")
    if weight.shape != (x.shape[-1],):
        raise ValueError(f"fused_add_rmsnorm: weight shape {tuple(weight.shape)} must be ({x.shape[-1]},).")
    if _lib.on_cpu("fused_add_rmsnorm", x, residual, weight):
        s = residual + x
        return torch.nn.functional.rms_norm(s, (s.shape[-1],), weight, eps), s
    if residual.dtype != x.dtype:
        raise TypeError(f"fused_add_rmsnorm: residual dtype {residual.dtype} must equal x dtype {x.dtype}")
    if not add_rmsnorm_supported(x, weight):
        from ats_v2_b200.norm import rms_norm

        s = residual + x
        return rms_norm(s, weight, eps), s
    return _AddRMSNormFn.apply(x, residual, weight, eps)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous from a multiple of 16 bytes (a view may start anywhere): the kernels read weights and gates so."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _sandwich_forward(x, residual, wp, wn, g, rows_per_gate, residual_scale, eps, train):
    """The forward kernel on contiguous tensors: (h, s, rstd), rstd [2, rows] kept for the backward."""
    H = x.shape[-1]
    rows = x.numel() // H
    s, h = torch.empty_like(x), torch.empty_like(x)
    rstd = x.new_empty((2, rows), dtype=torch.float32) if train else None
    p = rstd.data_ptr() if train else 0
    with _lib.device_of(x):
        _lib.call("ats_sandwich_norm_fwd", x.data_ptr(), residual.data_ptr(), _lib.dtype_code(x.dtype), wp.data_ptr(),
                  wn.data_ptr(), _lib.dtype_code(wp.dtype), g.data_ptr() if g is not None else None,
                  _lib.dtype_code(g.dtype) if g is not None else 0, rows_per_gate, residual_scale, eps, s.data_ptr(),
                  h.data_ptr(), p or None, p + 4 * rows if p else None, rows, H, _lib.stream_of(x))
    return h, s, rstd


class _SandwichNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, post_weight, pre_weight, gate, rows_per_gate, residual_scale, eps):
        ctx.set_materialize_grads(False)  # an unused result's gradient arrives as None and is not read
        x, residual = x.contiguous(), residual.contiguous()
        wp, wn = _aligned(post_weight), _aligned(pre_weight)
        g = _aligned(gate) if gate is not None else None
        h, s, rstd = _sandwich_forward(x, residual, wp, wn, g, rows_per_gate, residual_scale, eps, True)
        ctx.save_for_backward(x, residual, wp, wn, g, rstd)
        ctx.meta = rows_per_gate, residual_scale
        return h, s

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dh, ds):
        if dh is None and ds is None:
            return (None,) * 8
        x, r, wp, wn, g, rstd = ctx.saved_tensors
        rows_per_gate, residual_scale = ctx.meta
        H = x.shape[-1]
        rows = x.numel() // H
        if rows == 0:
            return (torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(wp), torch.zeros_like(wn),
                    torch.zeros_like(g) if g is not None else None, None, None, None)
        dh, ds = (t.to(x.dtype).contiguous() if t is not None else None for t in (dh, ds))
        dx, dr = torch.empty_like(x), torch.empty_like(r)
        dwp, dwn = torch.empty_like(wp), torch.empty_like(wn)
        dg = torch.empty_like(g) if g is not None else None
        with _lib.device_of(x):
            wsb = _lib.query("ats_sandwich_norm_bwd_workspace_bytes", rows, H, rows_per_gate if g is not None else 0)
            ws = x.new_empty(wsb, dtype=torch.uint8)
            _lib.call("ats_sandwich_norm_bwd", _lib.ptr(dh), _lib.ptr(ds), x.data_ptr(), r.data_ptr(),
                      _lib.dtype_code(x.dtype), wp.data_ptr(), wn.data_ptr(), _lib.dtype_code(wp.dtype), _lib.ptr(g),
                      _lib.dtype_code(g.dtype) if g is not None else 0, rows_per_gate, residual_scale,
                      rstd.data_ptr(), rstd.data_ptr() + 4 * rows, dx.data_ptr(), dr.data_ptr(), dwp.data_ptr(),
                      dwn.data_ptr(), _lib.ptr(dg), ws.data_ptr(), wsb, rows, H, _lib.stream_of(x))
        return dx, dr, dwp, dwn, dg, None, None, None


def _rows_per_gate(shape: torch.Size, gate: torch.Tensor) -> int:
    """How many consecutive rows of x share a gate row: gate is [H], or x's shape with
    1 in place of the last axes before H (none of them, some or all)."""
    if gate.dim() == 1 and gate.shape[0] == shape[-1]:
        return max(1, shape[:-1].numel())
    if gate.dim() == len(shape) and gate.shape[-1] == shape[-1]:
        lead = len(shape) - 1
        while lead > 0 and gate.shape[lead - 1] == 1:
            lead -= 1
        if gate.shape[:lead] == shape[:lead]:
            return max(1, shape[lead:-1].numel())
    raise ValueError(f"fused_sandwich_norm: gate shape {tuple(gate.shape)} must be ({shape[-1]},) or x's shape "
                     f"{tuple(shape)} with 1 in place of the last axes before hidden, e.g. [batch, 1, hidden].")


def _torch_sandwich_norm(x, residual, post_weight, pre_weight, gate, residual_scale, eps):
    """The operator in torch operations (float32, rounded once): what CPU tensors run."""
    def norm(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.float()

    p = norm(x.float(), post_weight)
    s = residual_scale * residual.float() + (p if gate is None else gate.float() * p)
    return norm(s, pre_weight).to(x.dtype), s.to(x.dtype)


def fused_sandwich_norm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor,
                        gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                        eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """The end of a transformer block whose output ``x`` is normalised before it joins the
    residual stream, with the next block's norm:

        s = residual_scale * residual + gate * (rms_norm(x) * post_weight)
        h = rms_norm(s) * pre_weight

    Returns (h, s): the next block's input and its residual.  ``x`` and ``residual``
    share shape [..., hidden] and dtype (float32 or bfloat16); the weights [hidden]
    share a dtype (float32 or bfloat16); ``gate`` (optional, float32 or bfloat16) is
    [hidden] (per channel), x's shape (per token) or x's shape with 1 in place of the
    last axes before hidden, e.g. [batch, 1, hidden] (per sequence).  The arithmetic is
    float32 and each result is rounded once.  CUDA tensors run one kernel forward and
    two backward (sums over rows in a fixed order: results repeat bit for bit);
    differentiable once, in every tensor argument, and in reverse mode only (duals are
    refused)."""
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"fused_sandwich_norm expected x of shape [..., hidden], got {tuple(shape)}.")
    if shape != residual.shape:
        raise ValueError(f"fused_sandwich_norm: x shape {tuple(shape)} must match residual shape "
                         f"{tuple(residual.shape)}.")
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w.shape != shape[-1:]:
            raise ValueError(f"fused_sandwich_norm: {name} shape {tuple(w.shape)} must be ({shape[-1]},).")
    if residual.dtype != x.dtype:
        raise TypeError(f"fused_sandwich_norm: residual dtype {residual.dtype} must equal x dtype {x.dtype}")
    if pre_weight.dtype != post_weight.dtype:
        raise TypeError(f"fused_sandwich_norm: pre_weight dtype {pre_weight.dtype} must equal post_weight dtype "
                        f"{post_weight.dtype}")
    rows_per_gate = _rows_per_gate(shape, gate) if gate is not None else 0
    residual_scale, eps = float(residual_scale), float(eps)
    if _lib.on_cpu("fused_sandwich_norm", x, residual, post_weight, pre_weight, gate):
        return _torch_sandwich_norm(x, residual, post_weight, pre_weight, gate, residual_scale, eps)
    if _lib.wants_grad(x, residual, post_weight, pre_weight, gate):
        return _SandwichNormFn.apply(x, residual, post_weight, pre_weight, gate, rows_per_gate, residual_scale, eps)
    return _sandwich_forward(x.contiguous(), residual.contiguous(), _aligned(post_weight), _aligned(pre_weight),
                             _aligned(gate) if gate is not None else None, rows_per_gate, residual_scale, eps, False)[:2]
