"""``fused_sandwich_norm`` on CUDA against its formula in 64 bits: results and every gradient, for each gate form,
type and width the kernels treat apart."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.norm_fused import fused_sandwich_norm
from tests.bounds import assert_within, sandwich_exact, sandwich_slack

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(shape, xd, wd="f32", gate=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    H = shape[-1]

    def randn(*s):
        return torch.randn(s, generator=g)

    gshape = {None: None, "channel": (H,), "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (H,), "token": shape,
              "one": (1,) * (len(shape) - 1) + (H,)}[gate]
    x = (randn(*shape) * (1 + 5 * (randn(H) > 2))).to(TD[xd]).cuda()
    res = (2 * randn(*shape)).to(TD[xd]).cuda()
    wp, wn = ((1 + 0.2 * randn(H)).to(TD[wd]).cuda() for _ in range(2))
    gt = None if gshape is None else (0.5 * randn(*gshape)).to(TD[xd]).cuda()
    dh, ds = (randn(*shape).to(TD[xd]).cuda() for _ in range(2))
    return x, res, wp, wn, gt, dh, ds


def check(shape, xd, wd, gate, a=0.7, eps=1e-5, seed=0, only=None):
    x, res, wp, wn, gt, dh, ds = make(shape, xd, wd, gate, seed)
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt) if t is not None]
    h, s = fused_sandwich_norm(x, res, wp, wn, gate=gt, residual_scale=a, eps=eps)
    assert h.dtype == s.dtype == x.dtype and h.shape == s.shape == x.shape
    outs, grads = {None: ((h, s), (dh, ds)), "h": ((h,), (dh,)), "s": ((s,), (ds,))}[only]
    got = torch.autograd.grad(outs, leaves, grads, allow_unused=True)
    e = sandwich_exact(x, res, wp, wn, gt, a, eps, None if only == "s" else dh, None if only == "h" else ds)
    rows = x.numel() // shape[-1]
    row_slack, sum_slack = sandwich_slack(shape[-1], 0), sandwich_slack(shape[-1], rows)
    named = [("h", h, row_slack), ("s", s, row_slack)]
    named += list(zip(("dx", "dres", "dwp", "dwn", "dgate"), got, (row_slack, row_slack) + (sum_slack,) * 3))
    for name, t, slack in named:
        assert_within(t.detach(), e[name][0], slack * e[name][1], f"{name} {shape} {xd} {wd} {gate}")


@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token", "one"])
@pytest.mark.parametrize("xd,wd", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
def test_gate_forms_and_types(gate, xd, wd):
    check((3, 37, 512), xd, wd, gate)


@pytest.mark.parametrize("H", [1, 2, 7, 31, 64, 96, 250, 513, 1030, 2048, 4096, 4104, 8192, 8200, 12001, 16392, 20000,
                               33000])
@pytest.mark.parametrize("xd", ["bf16", "f32"])
def test_widths(H, xd):
    check((2, 5, H), xd, "f32", "sequence" if H % 2 else "channel", seed=H)


@pytest.mark.parametrize("rows", [1, 2, 147, 300, 1500])
@pytest.mark.parametrize("gate", ["channel", "token"])
def test_row_counts(rows, gate):
    check((rows, 256), "bf16", "f32", gate, seed=rows)


@pytest.mark.parametrize("B,S", [(700, 2), (400, 3), (2, 400), (1, 9)])
def test_many_and_few_sequences(B, S):
    check((B, S, 128), "bf16", "f32", "sequence", seed=B)


@pytest.mark.parametrize("only", ["h", "s"])
@pytest.mark.parametrize("gate", [None, "sequence"])
def test_one_result_unused(only, gate):
    x, res, wp, wn, gt, dh, ds = make((2, 9, 264), "bf16", "f32", gate)
    check((2, 9, 264), "bf16", "f32", gate, only=only)


def test_four_axes_and_a_plain_row():
    check((2, 3, 4, 72), "bf16", "f32", "sequence")
    check((40,), "f32", "f32", "channel")


def test_misaligned_and_strided_inputs():
    """Rows of a wider buffer, and a gradient that is a broadcast: laid out anew, not misread."""
    base = torch.randn(6, 11, 520, generator=torch.Generator().manual_seed(3)).cuda().bfloat16()
    x = base[..., 1:513].detach().requires_grad_()
    flat = base.reshape(-1)[1:1 + 6 * 11 * 512].view(6, 11, 512).detach().requires_grad_()  # 2-byte aligned storage
    wp, wn = (1 + torch.rand(512, device="cuda") for _ in range(2))
    h, s = fused_sandwich_norm(x, flat, wp, wn, eps=1e-5)
    dh = torch.randn(512, device="cuda").bfloat16().expand(6, 11, 512)
    dx, dr = torch.autograd.grad(h, (x, flat), dh)
    e = sandwich_exact(x, flat, wp, wn, None, 1.0, 1e-5, dh, None)
    k = sandwich_slack(512, 0)
    for t, n in ((h, "h"), (s, "s"), (dx, "dx"), (dr, "dres")):
        assert_within(t.detach(), e[n][0], k * e[n][1], n)


def test_empty_input():
    x = torch.empty(0, 5, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    g = torch.ones(64, device="cuda", requires_grad=True)
    h, s = fused_sandwich_norm(x, x, w, w, gate=g)
    assert h.shape == s.shape == (0, 5, 64)
    dx, dw, dg = torch.autograd.grad((h.sum() + s.sum()), (x, w, g))
    assert dx.shape == x.shape and float(dw.abs().sum()) == 0 and float(dg.abs().sum()) == 0


def test_zero_rows_and_non_finite_values():
    """A row of zeros stays finite; an infinity or NaN stays in its own row."""
    x, res, wp, wn, _, _, _ = make((4, 256), "f32")
    x[0] = 0
    res[0] = 0
    x[1, 3] = float("inf")
    res[2, 5] = float("nan")
    h, s = fused_sandwich_norm(x, res, wp, wn, eps=1e-6)
    assert torch.equal(h[0], torch.zeros_like(h[0])) and torch.equal(s[0], torch.zeros_like(s[0]))
    assert h[1].isnan().any() and h[2].isnan().all()
    assert h[3].isfinite().all() and s[3].isfinite().all()


def test_gradients_against_differences():
    """Central differences of the operator itself in float32: the step's error h^2/6 f''' and the rounding
    2^-24 |f| / h are both under 1e-3 of the slope's scale at h = 1e-2."""
    x, res, wp, wn, gt, dh, ds = make((2, 3, 16), "f32", "f32", "sequence", seed=5)
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt)]

    def f():
        h, s = fused_sandwich_norm(x, res, wp, wn, gate=gt, residual_scale=1.3, eps=1e-3)
        return (h.double() * dh + s.double() * ds).sum()

    grads = torch.autograd.grad(f(), leaves)
    step = 1e-2
    with torch.no_grad():
        for t, g in zip(leaves, grads):
            flat = t.view(-1)
            for i in range(0, flat.numel(), max(1, flat.numel() // 12)):
                keep = flat[i].item()
                flat[i] = keep + step
                up = f().item()
                flat[i] = keep - step
                down = f().item()
                flat[i] = keep
                assert abs((up - down) / (2 * step) - g.view(-1)[i].item()) < 5e-3 * (1 + float(g.abs().max()))


def test_results_repeat_bit_for_bit():
    x, res, wp, wn, gt, dh, ds = make((3, 333, 1024), "bf16", "f32", "sequence")
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt)]

    def once():
        out = fused_sandwich_norm(x, res, wp, wn, gate=gt)
        return [*out, *torch.autograd.grad(out, leaves, (dh, ds))]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_other_stream_and_graph_replay():
    """Forward and backward on a side stream and captured into a graph, replayed on new inputs."""
    x, res, wp, wn, gt, dh, ds = make((2, 200, 512), "bf16", "f32", "channel")
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt)]

    def once():
        out = fused_sandwich_norm(x, res, wp, wn, gate=gt)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (dh, ds)))

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        ds.copy_(torch.randn_like(ds))
    graph.replay()
    held = [t.clone() for t in held]
    for a, b in zip(held, once()):
        assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    x, res, wp, wn, _, _, _ = make((2, 3, 64), "f32")
    x.requires_grad_()
    h, s = fused_sandwich_norm(x, res, wp, wn)
    (dx,) = torch.autograd.grad(h.sum() + s.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.parametrize("gate", ["channel", "sequence", "token"])
@pytest.mark.parametrize("xd,gd", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("H", [192, 1030, 1033, 4096, 6144])
def test_gates_of_another_type(H, xd, gd, gate):
    """A gate in another type than the rows is read in other pieces than they are."""
    x, res, wp, wn, gt, dh, ds = make((2, 9, H), xd, "f32", gate, seed=H)
    gt = gt.to(TD[gd])
    leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt)]
    out = fused_sandwich_norm(x, res, wp, wn, gate=gt, residual_scale=1.2, eps=1e-5)
    got = torch.autograd.grad(out, leaves, (dh, ds))
    assert got[4].dtype == gt.dtype
    e = sandwich_exact(x, res, wp, wn, gt, 1.2, 1e-5, dh, ds)
    for name, t in zip(("h", "s", "dx", "dres", "dwp", "dwn", "dgate"), (*out, *got)):
        slack = sandwich_slack(H, 18 if name[:2] in ("dw", "dg") else 0)
        assert_within(t.detach(), e[name][0], slack * e[name][1], f"{name} {H} {xd} {gd} {gate}")


def test_views_that_start_anywhere():
    """Weights and a gate cut from larger buffers at odd elements."""
    H = 264
    x, res, wp, wn, gt, dh, ds = make((3, 8, H), "bf16", "f32", "token")
    buf = torch.empty(2 * H + 3, device="cuda")
    buf[1:H + 1], buf[H + 2:2 * H + 2] = wp, wn
    gbuf = torch.empty(gt.numel() + 1, dtype=gt.dtype, device="cuda")
    gbuf[1:] = gt.reshape(-1)
    ins = [t.requires_grad_() for t in (x, res, buf[1:H + 1], buf[H + 2:2 * H + 2], gbuf[1:].view_as(gt))]
    out = fused_sandwich_norm(*ins[:4], gate=ins[4])
    got = torch.autograd.grad(out, ins, (dh, ds))
    same = [t.detach().requires_grad_() for t in (x, res, wp, wn, gt)]
    want_out = fused_sandwich_norm(*same[:4], gate=same[4])
    want = torch.autograd.grad(want_out, same, (dh, ds))
    for a, b in zip((*out, *got), (*want_out, *want)):
        assert torch.equal(a, b)


def test_one_tensor_in_several_places():
    """x as its own residual and one weight for both norms: the gradients add up."""
    x, _, w, _, _, dh, ds = make((2, 5, 128), "f32")
    x.requires_grad_()
    w.requires_grad_()
    out = fused_sandwich_norm(x, x, w, w, residual_scale=0.5)
    dx, dw = torch.autograd.grad(out, (x, w), (dh, ds))
    e = sandwich_exact(x, x, w, w, None, 0.5, 1e-6, dh, ds)
    k = sandwich_slack(128, 10)
    assert_within(dx, e["dx"][0] + e["dres"][0], 2 * k * (e["dx"][1] + e["dres"][1]))
    assert_within(dw, e["dwp"][0] + e["dwn"][0], 2 * k * (e["dwp"][1] + e["dwn"][1]))


def test_two_streams_at_once():
    ins = [make((2, 700, 1024), "bf16", "f32", "sequence", seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ins]

    def once(i):
        x, res, wp, wn, gt, dh, ds = ins[i]
        leaves = [t.requires_grad_() for t in (x, res, wp, wn, gt)]
        out = fused_sandwich_norm(x, res, wp, wn, gate=gt)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (dh, ds)))

    want = [once(i) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(once(i))
        torch.cuda.synchronize()
        for a, b in zip(want[0] + want[1], got[0] + got[1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H,rows", [(1, 9000), (363, 2500), (2509, 1200), (4097, 900), (6, 9000), (1030, 1500)])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
def test_odd_widths_over_many_rows(H, rows, gate):
    """Several rows to a block in the narrow vectors: a row ahead in registers, or in the ring."""
    check((4, rows // 4, H), "bf16", "f32", gate, seed=H)


@pytest.mark.parametrize("only", ["h", "s"])
def test_odd_width_with_one_result_unused(only):
    check((2, 600, 519), "bf16", "bf16", "token", only=only)
