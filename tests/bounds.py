"""Error bounds of the block operators' tests, from the arithmetic.

A result is compared with its formula in 64 bits.  A float32 computation of a
few stages, each a sum of at most n terms in any order, is off by at most
``stages * n * 2^-24`` of the same formula on absolute values (first order);
rounding the result once to type t adds ``eps(t) / 2`` of the value.
"""

from __future__ import annotations

from fractions import Fraction

import torch

U32 = 2.0 ** -24


def assert_within(got: torch.Tensor, exact: torch.Tensor, slack, what: str = "") -> None:
    """|got - exact| <= half a step of got's type at the value, plus slack."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    e = exact.double().cpu()
    half = torch.finfo(got.dtype).eps / 2
    slack = slack.double().cpu() if isinstance(slack, torch.Tensor) else slack
    bound = half * (e.abs() + slack) + slack
    off = (got.double().cpu() - e).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst by " \
                                f"{float((off / bound.clamp_min(1e-300)).max()):.3g} times the bound"


def sandwich_exact(x, res, wp, wn, gate, a, eps, dh=None, ds=None):
    """fused_sandwich_norm in 64 bits.  Returns {name: (value, magnitude)}: the same formulas on absolute
    values give the magnitudes.  dh or ds None: zero."""
    H = x.shape[-1]
    x, res, wp, wn = (t.detach().double().cpu() for t in (x, res, wp, wn))
    g = torch.ones(()).double() if gate is None else gate.detach().double().cpu()

    def mean(t):
        return t.sum(-1, keepdim=True) / H

    rx = (mean(x * x) + eps).rsqrt()
    p, pm = x * rx * wp, (x * rx * wp).abs()
    s, sm = a * res + g * p, (a * res).abs() + g.abs() * pm
    rs = (mean(s * s) + eps).rsqrt()
    # the error of mean(s^2), relative to it, is up to mean(sm^2) / mean(s^2) steps
    k = mean(sm * sm) * rs * rs + 1
    out = {"s": (s, sm), "h": (s * rs * wn, sm * rs * wn.abs() * k)}
    if dh is None and ds is None:
        return out
    dh = torch.zeros_like(x) if dh is None else dh.double().cpu()
    ds = torch.zeros_like(x) if ds is None else ds.double().cpu()
    u = dh * wn
    S = ds + rs * u - s * rs ** 3 * mean(u * s)
    Sm = ds.abs() + k * (rs * u.abs() + 3 * sm * rs ** 3 * mean(u.abs() * sm))
    v, vm = S * g * wp, Sm * (g * wp).abs()
    dx = rx * v - x * rx ** 3 * mean(v * x)
    dxm = rx * vm + 3 * x.abs() * rx ** 3 * mean(vm * x.abs())

    def total(t):  # over the rows
        return t.reshape(-1, H).sum(0)

    A, Am = S * x * rx, Sm * (x * rx).abs()
    out |= {"dx": (dx, dxm), "dres": (a * S, abs(a) * Sm), "dwp": (total(g * A), total(g.abs() * Am)),
            "dwn": (total(dh * s * rs), total(dh.abs() * sm * rs * k))}
    if gate is not None:
        def fold(t):  # over the axes the gate was broadcast along
            t = total(t) if gate.dim() == 1 else t
            axes = [i for i in range(t.dim()) if gate.dim() > 1 and gate.shape[i] == 1 and t.shape[i] != 1]
            return (t.sum(axes, keepdim=True) if axes else t).reshape(gate.shape)

        out["dgate"] = (fold(wp * A), fold(wp.abs() * Am))
    return out


def sandwich_slack(H: int, rows: int) -> float:
    """Five stages (two norms forward, two means and a sum over rows backward), each of up to H or rows terms;
    a thread sums at most H/32 + 8 terms of a row before the log-depth rest."""
    return 5 * (H / 32 + 16 + rows) * U32


PI = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


def turns_exact(positions, inv_freq, axes):
    """exp(i angle) [B, S, pairs] of the rotation, in 64 bits.  The angle of a far position has more digits than a
    double: it is reduced by whole turns as a fraction first."""
    pos = (positions if positions.dim() == 3 else positions[:, None]).cpu()
    n, B, S = pos.shape
    inv = [Fraction(v) for v in inv_freq.double().tolist()]
    if float(pos.abs().max()) * max(map(float, inv)) < 2 ** 16 if pos.numel() else True:
        angle = pos.double()[list(axes)].permute(1, 2, 0) * inv_freq.double().cpu()  # off by at most 2^-37
    else:
        v = pos.tolist()
        angle = torch.tensor([[[float((Fraction(v[a][b][s]) * inv[j] + PI) % (2 * PI) - PI)
                                for j, a in enumerate(axes)] for s in range(S)] for b in range(B)],
                             dtype=torch.float64)
    return torch.polar(torch.ones((), dtype=torch.float64), angle)


def rotate_exact(t, turn):
    """t [B, heads, S, D] rotated by turn, in 64 bits."""
    n = turn.shape[-1]
    t = t.detach().double().cpu()
    z = torch.complex(t[..., :n], t[..., n:2 * n]) * turn.unsqueeze(1)
    return torch.cat([z.real, z.imag, t[..., 2 * n:]], -1)


def rotate_slack(t, n):
    """The remainder of the angle rounds to float32 (half a step of at most 1/2 turn: pi 2^-24 radians), the
    cosine and sine are good to 2 steps (4 units), the products and the sum round: 10 units of |a| + |b|."""
    m = t.detach().double().cpu().abs()
    pair = m[..., :n] + m[..., n:2 * n]
    return 10 * U32 * torch.cat([pair, pair, torch.zeros_like(m[..., 2 * n:])], -1)


def int8_exact(x, w, scale, bias=None):
    """int8_linear: the quantised activations are float32 by definition, the rest in 64 bits.
    Returns (value, magnitude of the terms that are added)."""
    x = x.detach().float().cpu()
    amax = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    full = torch.full_like(amax, 127)
    q = torch.round(x * (full / amax)).double()
    y = (q @ w.double().cpu().t()) * ((amax / full).double() * scale.double().cpu())
    if bias is None:
        return y, y.abs()
    b = bias.double().cpu()
    return y + b, y.abs() + b.abs()


INT8_SLACK = 4 * U32  # the sum's conversion, the product of the scales, its application, the bias
