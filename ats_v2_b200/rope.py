"""Rotary position embedding on the sm_100a kernels -- mirror of
ats/model/rope.py.

* ``RotaryEmbedding(dim, max_seq_len=4096, theta=10000.)`` builds the same
  float32 ``inv_freq`` and cos/sin cache as rope.py:17-43 (same torch
  expressions, so the tables are identical), grows it by doubling
  (rope.py:50-59), and returns tables cast to the requested device/dtype
  (rope.py:60-61).  The cast tables are cached per (device, dtype) instead of
  being re-cast on every call.
* ``apply_rotary_pos_emb(q, k, cos, sin)`` (rope.py:71-87) rotates q and k
  in ONE kernel launch (``ats_rope_apply``) that reads the strided [B,H,S,D]
  views in place (the attention layout hands in transposed BSHD memory) and
  writes outputs with the inputs' strides; its backward is the adjoint
  rotation, again one launch.
* ``rotate_half`` is kept for API compatibility (rope.py:65-68).

Not in the reference: positions with several axes (time, height and width of
images and video).  ``apply_multi_axis_rotary(q, k, positions, inv_freq,
sections)`` rotates each pair of a head by its own axis's position, and
``MultiAxisRotaryEmbedding`` holds the frequencies.
"""

from __future__ import annotations

import functools
from collections.abc import Sequence

import torch
from torch import nn

from ats_v2_b200 import _lib


class RotaryEmbedding(nn.Module):
    """Drop-in for ats.model.rope.RotaryEmbedding."""

    def __init__(self, dim: int, max_seq_len: int = 4096, theta: float = 10000.0) -> None:
        super().__init__()
        if dim % 2 != 0:
            raise ValueError(
                f"RotaryEmbedding dim must be even, got {dim}. "
                f"Fix: head_dim (hidden_size // num_heads) must be even."
            )
        self.dim = dim
        self.theta = theta
        inv_freq = 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
        self.inv_freq: torch.Tensor
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self._cached_seq_len = 0
        self._cast: dict = {}
        self._build_cache(max_seq_len)

    def _build_cache(self, seq_len: int) -> None:
        t = torch.arange(seq_len, dtype=torch.float32, device=self.inv_freq.device)
        freqs = torch.outer(t, self.inv_freq)
        emb = torch.cat([freqs, freqs], dim=-1)
        self.register_buffer("_cached_cos", emb.cos(), persistent=False)
        self.register_buffer("_cached_sin", emb.sin(), persistent=False)
        self._cached_seq_len = seq_len
        self._cast = {}

    def _apply(self, fn, recurse=True):  # .to()/.cuda() move the buffers: drop cast copies
        self._cast = {}
        return super()._apply(fn, recurse)

    def forward(self, seq_len: int, device: torch.device, dtype: torch.dtype):
        if seq_len <= 0:
            raise ValueError(f"RotaryEmbedding requires seq_len > 0, got {seq_len}.")
        if seq_len > self._cached_seq_len:
            new_len = max(seq_len, self._cached_seq_len * 2 if self._cached_seq_len > 0 else seq_len)
            self._build_cache(new_len)
        key = (torch.device(device), dtype)
        full = self._cast.get(key)
        if full is None:
            full = (self._cached_cos.to(device=device, dtype=dtype),
                    self._cached_sin.to(device=device, dtype=dtype))
            self._cast[key] = full
        return full[0][:seq_len], full[1][:seq_len]


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    """cat(-x2, x1) over the last dim (rope.py:65-68); not used by the kernels."""
    half = x.shape[-1] // 2
    return torch.cat((-x[..., half:], x[..., :half]), dim=-1)


def _last_dim_contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _out_like(t: torch.Tensor) -> torch.Tensor:
    """An empty tensor laid out like t, its last axis consecutive as the kernels write it: empty_like moves another
    axis of an overlapping view (windows of a longer sequence, say) inside of it."""
    out = torch.empty_like(t)
    return out if out.stride()[3] == 1 else t.new_empty(t.shape)


def _table(t: torch.Tensor, D: int, S: int, name: str) -> tuple[torch.Tensor, int]:
    if t.dim() != 2 or t.shape[-1] != D or t.shape[0] not in (S, 1):
        raise ValueError(f"{name}: cos/sin must be [seq_len={S} (or 1), {D}], got {tuple(t.shape)}")
    t = _last_dim_contig(t)
    return t, (0 if t.shape[0] == 1 else t.stride(0))


def _launch(q_in, q_out, k_in, k_out, cos, sin, cs_stride, backward: bool) -> None:
    B, Hq, S, D = q_in.shape
    Hk = k_in.shape[1] if k_in is not None else 0
    qs = _lib.strides3(q_in.stride(0), q_in.stride(1), q_in.stride(2))
    qo = _lib.strides3(q_out.stride(0), q_out.stride(1), q_out.stride(2))
    ks = _lib.strides3(k_in.stride(0), k_in.stride(1), k_in.stride(2)) if k_in is not None else None
    ko = _lib.strides3(k_out.stride(0), k_out.stride(1), k_out.stride(2)) if k_in is not None else None
    _lib.call("ats_rope_apply", q_in.data_ptr(), q_out.data_ptr(), Hq, qs, qo,
              _lib.ptr(k_in), _lib.ptr(k_out), Hk, ks, ko, cos.data_ptr(), sin.data_ptr(), cs_stride,
              B, S, D, _lib.dtype_code(q_in.dtype), 1 if backward else 0, _lib.stream_of(q_in))


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, cs_stride):
        ctx.set_materialize_grads(False)  # an unused output's gradient arrives as None, not zeros
        q_out = _out_like(q)
        k_out = _out_like(k) if k is not None else None
        _launch(q, q_out, k, k_out, cos, sin, cs_stride, False)
        ctx.save_for_backward(cos, sin)
        ctx.cs_stride = cs_stride
        ctx.has_k = k is not None
        return q_out, k_out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        cos, sin = ctx.saved_tensors
        if dq_out is None and (dk_out is None or not ctx.has_k):
            return None, None, None, None, None
        if dq_out is None:  # only k was used downstream: run its adjoint alone
            dk_out = _last_dim_contig(dk_out)
            dk = _out_like(dk_out)
            _launch(dk_out, dk, None, None, cos, sin, ctx.cs_stride, True)
            return None, dk, None, None, None
        dq_out = _last_dim_contig(dq_out)
        dq = _out_like(dq_out)
        dk = None
        if ctx.has_k and dk_out is not None:
            dk_out = _last_dim_contig(dk_out)
            dk = _out_like(dk_out)
        _launch(dq_out, dq, dk_out if dk is not None else None, dk, cos, sin, ctx.cs_stride, True)
        return dq, dk, None, None, None


def _prepare(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, name: str):
    _lib.require_cuda(name, q, k, cos, sin)
    if cos.requires_grad or sin.requires_grad:
        raise NotImplementedError(f"{name}: gradients w.r.t. cos/sin are not supported")
    out_dtype = torch.promote_types(q.dtype, cos.dtype)
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"{name}: q and k must share a dtype ({q.dtype} vs {k.dtype})")
        if k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k.shape[3] != q.shape[3]:
            raise ValueError(f"{name}: k shape {tuple(k.shape)} incompatible with q {tuple(q.shape)}")
    # torch promotes x*cos to the wider dtype; upcasting the narrower operand is exact
    q = _last_dim_contig(q.to(out_dtype))
    k = _last_dim_contig(k.to(out_dtype)) if k is not None else None
    cos, cs_stride = _table(cos.to(out_dtype), q.shape[-1], q.shape[2], name)
    sin, ss_stride = _table(sin.to(out_dtype), q.shape[-1], q.shape[2], name)
    if cs_stride != ss_stride:  # one table broadcast, the other not: materialise both
        S, D = q.shape[2], q.shape[3]
        cos = cos.expand(S, D).contiguous()
        sin = sin.expand(S, D).contiguous()
        cs_stride = D
    return q, k, cos, sin, cs_stride


def apply_rotary_pos_emb(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                         sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """q, k: [batch, heads, seq_len, head_dim] (any b/h/s strides); cos, sin: [seq_len, head_dim].
    One CUDA launch rotates q and k; CPU tensors take the reference's torch formula."""
    if q.shape[-1] != cos.shape[-1]:
        raise ValueError(
            f"apply_rotary_pos_emb: q head_dim ({q.shape[-1]}) does not match "
            f"cos/sin dim ({cos.shape[-1]})."
        )
    if _lib.on_cpu("apply_rotary_pos_emb", q, k, cos, sin):
        # CPU tensors: the reference's torch formula (rope.py:83-86)
        c, s = cos[None, None], sin[None, None]
        return q * c + rotate_half(q) * s, (k * c + rotate_half(k) * s if k is not None else None)
    if q.dim() != 4:
        raise ValueError(f"apply_rotary_pos_emb: q must be [batch, heads, seq_len, head_dim], got {tuple(q.shape)}")
    q, k, cos, sin, cs = _prepare(q, k, cos, sin, "apply_rotary_pos_emb")
    return _RopeFn.apply(q, k, cos, sin, cs)


def axis_of_pairs(sections: tuple[int, ...], interleaved: bool = False) -> bytes:
    """The position axis of each rotated pair.  ``sections[a]`` pairs follow axis a:
    section after section, or (``interleaved``) dealt out one by one to the axes that
    have pairs left."""
    return _axis_of_pairs(bool(interleaved), *sections)


@functools.lru_cache(maxsize=64, typed=True)  # by the counts' types too: 2.0 is refused whether or not 2 was seen
def _axis_of_pairs(interleaved: bool, *sections: int) -> bytes:
    if not sections or any(not isinstance(n, int) or n < 0 for n in sections) or len(sections) > 256 or \
            not 1 <= sum(sections) <= _lib.ATS_ROPE_MAX_PAIRS:
        raise ValueError(f"multi-axis rotary: sections {sections} must be counts of pairs, one per axis, 1 to "
                         f"{_lib.ATS_ROPE_MAX_PAIRS} pairs in all.")
    pairs = [(i, a) for a, n in enumerate(sections) for i in range(n)]
    return bytes(a for _, a in (sorted(pairs) if interleaved else pairs))


def _launch_axes(q, k, positions, inv_freq, axes: bytes, n_axes: int, backward: bool):
    """The rotation of q and k, of which one may be None: (q_out, k_out)."""
    first, second = (q, k) if q is not None else (k, None)
    B, H, S, D = first.shape
    s3 = _lib.strides3
    pos = positions.stride()
    ib, ih, is_, _ = first.stride()
    out = torch.empty_like(first)
    ob, oh, os_, od = out.stride()
    if od != 1:
        out = _out_like(first)
        ob, oh, os_, _ = out.stride()
    out2, kargs = None, (None, None, 0, None, None)
    if second is not None:
        kb, kh, ks, _ = second.stride()
        out2 = torch.empty_like(second)
        cb, ch, cs, cd = out2.stride()
        if cd != 1:
            out2 = _out_like(second)
            cb, ch, cs, _ = out2.stride()
        kargs = (second.data_ptr(), out2.data_ptr(), second.shape[1], s3(kb, kh, ks), s3(cb, ch, cs))
    with _lib.device_of(first):
        _lib.call("ats_rope_axes_apply", first.data_ptr(), out.data_ptr(), H, s3(ib, ih, is_), s3(ob, oh, os_), *kargs,
                  positions.data_ptr(), _lib.ATS_POS_TYPES[positions.dtype],
                  s3(pos[0], pos[1] if len(pos) == 3 else 0, pos[-1]), n_axes, inv_freq.data_ptr(), axes, len(axes),
                  B, S, D, _lib.dtype_code(first.dtype), 1 if backward else 0, _lib.stream_of(first))
    return (out, out2) if q is not None else (None, out)


class _MultiAxisRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axes, n_axes):
        ctx.set_materialize_grads(False)  # an unused output's gradient arrives as None, not zeros
        q_out, k_out = _launch_axes(q, k, positions, inv_freq, axes, n_axes, False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.axes = axes, n_axes
        return q_out, k_out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dq_out, dk_out):
        positions, inv_freq = ctx.saved_tensors
        dq_out, dk_out = (_last_dim_contig(t) if t is not None else None for t in (dq_out, dk_out))
        if dq_out is None and dk_out is None:
            return (None,) * 6
        return *_launch_axes(dq_out, dk_out, positions, inv_freq, *ctx.axes, True), None, None, None, None


def _torch_multi_axis(x: torch.Tensor, positions, inv_freq, axes: bytes) -> torch.Tensor:
    """The rotation in torch operations (angles in 64 bits, float32 arithmetic): what CPU tensors run."""
    n = len(axes)
    pos = positions if positions.dim() == 3 else positions[:, None]
    angle = pos.double()[list(axes)].permute(1, 2, 0) * inv_freq.double()  # [B, S, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    f = x.float()
    a, b = f[..., :n], f[..., n:2 * n]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, f[..., 2 * n:]], -1).to(x.dtype)


def apply_multi_axis_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                            sections: Sequence[int], interleaved: bool = False
                            ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary embedding of q and k (optional) [batch, heads, seq_len, head_dim] whose positions
    have several axes.  ``positions`` is [axes, batch, seq_len] or [axes, seq_len] (int32, int64
    or float32); ``sections[a]`` pairs of each head follow axis a, consecutive or
    (``interleaved``) dealt out in turn to the axes with pairs left; pair j joins columns j and
    j + sum(sections) and turns by ``positions[axis] * inv_freq[j]`` radians (``inv_freq``
    float32 [sum(sections)]).  Columns from 2*sum(sections) on pass unchanged.  The angles are
    reduced in 64 bits, so far positions keep their accuracy; the rest is float32, rounded once.
    Any batch, head and sequence strides; the results of dense inputs are laid out like them.
    One launch each way on CUDA tensors; differentiable once, in q and k, and in reverse mode only
    (duals are refused)."""
    axes = _axis_of_pairs(bool(interleaved), *sections)
    n_axes = len(sections)
    if q.dim() != 4 or q.shape[-1] < 2 * len(axes):
        raise ValueError(f"apply_multi_axis_rotary: q must be [batch, heads, seq_len, head_dim >= {2 * len(axes)}], "
                         f"got {tuple(q.shape)}.")
    B, _, S, D = q.shape
    if k is not None:
        if k.dim() != 4 or (k.shape[0], k.shape[2], k.shape[3]) != (B, S, D):
            raise ValueError(f"apply_multi_axis_rotary: k shape {tuple(k.shape)} incompatible with q {tuple(q.shape)}.")
        if k.dtype != q.dtype:
            raise TypeError(f"apply_multi_axis_rotary: q and k must share a dtype ({q.dtype} vs {k.dtype})")
    if tuple(positions.shape) not in ((n_axes, B, S), (n_axes, S)):
        raise ValueError(f"apply_multi_axis_rotary: positions must be [{n_axes}, {B}, {S}] or [{n_axes}, {S}], got "
                         f"{tuple(positions.shape)}.")
    if positions.dtype not in _lib.ATS_POS_TYPES:
        raise TypeError(f"apply_multi_axis_rotary: positions must be int32, int64 or float32, got {positions.dtype}")
    if inv_freq.shape != (len(axes),) or inv_freq.dtype != torch.float32:
        raise ValueError(f"apply_multi_axis_rotary: inv_freq must be float32 [{len(axes)}], got {inv_freq.dtype} "
                         f"{tuple(inv_freq.shape)}.")
    if positions.requires_grad or inv_freq.requires_grad:
        raise NotImplementedError("apply_multi_axis_rotary: gradients w.r.t. positions and inv_freq are not supported")
    if _lib.on_cpu("apply_multi_axis_rotary", q, k, positions, inv_freq):
        return (_torch_multi_axis(q, positions, inv_freq, axes),
                _torch_multi_axis(k, positions, inv_freq, axes) if k is not None else None)
    q = _last_dim_contig(q)
    k = _last_dim_contig(k) if k is not None else None
    inv_freq = inv_freq.contiguous()
    if _lib.wants_grad(q, k, positions, inv_freq):  # the last two need none: they may be duals
        return _MultiAxisRotaryFn.apply(q, k, positions, inv_freq, axes, n_axes)
    return _launch_axes(q, k, positions, inv_freq, axes, n_axes, False)


class MultiAxisRotaryEmbedding(nn.Module):
    """Rotary embedding over several position axes, as ``RotaryEmbedding`` is over one: pair j of
    the ``dim`` rotated columns has frequency theta^(-2j/dim) and follows the axis that
    ``sections`` (pairs per axis, summing to dim/2) gives it.  With the same position on every
    axis it is the rotation of ``RotaryEmbedding``."""

    def __init__(self, dim: int, sections: Sequence[int], theta: float = 10000.0, interleaved: bool = False) -> None:
        super().__init__()
        if dim % 2 != 0 or 2 * len(axis_of_pairs(tuple(sections), bool(interleaved))) != dim:
            raise ValueError(f"MultiAxisRotaryEmbedding: sections {tuple(sections)} must sum to dim / 2, got dim {dim}.")
        self.dim = dim
        self.sections = tuple(sections)
        self.theta = theta
        self.interleaved = bool(interleaved)
        self.inv_freq: torch.Tensor
        self.register_buffer("inv_freq", self._frequencies(), persistent=False)

    def _frequencies(self, device: torch.device | None = None) -> torch.Tensor:
        return 1.0 / (self.theta ** (torch.arange(0, self.dim, 2, dtype=torch.float32, device=device) / self.dim))

    def _apply(self, fn, recurse=True):
        old = self.inv_freq
        super()._apply(fn, recurse)
        new = self.inv_freq
        if old.is_meta and not new.is_meta:  # no state dict holds what belongs there
            self.inv_freq = self._frequencies(new.device)
        else:  # .to(dtype) must not round the frequencies, nor to_empty lose them
            self.inv_freq = old.to(device=new.device)
        return self

    def forward(self, q: torch.Tensor, k: torch.Tensor | None,
                positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor | None]:
        return apply_multi_axis_rotary(q, k, positions, self.inv_freq, self.sections, self.interleaved)
