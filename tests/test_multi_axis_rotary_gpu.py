"""``apply_multi_axis_rotary`` on CUDA against the rotation in 64 bits: axes, head sizes, layouts, far positions."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.rope import (MultiAxisRotaryEmbedding, RotaryEmbedding, apply_multi_axis_rotary, apply_rotary_pos_emb,
                              axis_of_pairs)
from tests.bounds import assert_within, rotate_exact, rotate_slack, turns_exact

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(B, S, Hq, Hk, D, sections, dt, reach=5000, layout="bshd", seed=0, ptype=torch.int64):
    g = torch.Generator().manual_seed(seed)

    def heads(n):
        if layout == "bshd":
            return torch.randn(B, S, n, D, generator=g).to(TD[dt]).cuda().transpose(1, 2)
        return torch.randn(B, n, S, D, generator=g).to(TD[dt]).cuda()

    q, k = heads(Hq), heads(Hk)
    pos = torch.randint(0, reach, (len(sections), B, S), generator=g)
    pos = (pos + 0.37 if ptype == torch.float32 else pos).to(ptype).cuda()
    n = sum(sections)
    inv = (1.0 / 10000.0 ** (torch.arange(n).float() / n)).cuda()
    return q, k, pos, inv, heads(Hq), heads(Hk)


def check(B, S, Hq, Hk, D, sections, dt, interleaved=False, **kw):
    q, k, pos, inv, gq, gk = make(B, S, Hq, Hk, D, sections, dt, **kw)
    q.requires_grad_()
    k.requires_grad_()
    qo, ko = apply_multi_axis_rotary(q, k, pos, inv, sections, interleaved=interleaved)
    assert qo.stride() == q.stride() and ko.stride() == k.stride() and qo.dtype == q.dtype
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    turn = turns_exact(pos, inv, axis_of_pairs(tuple(sections), interleaved))
    n = sum(sections)
    for got, src, by in ((qo, q, turn), (ko, k, turn), (dq, gq, turn.conj()), (dk, gk, turn.conj())):
        assert_within(got.detach(), rotate_exact(src, by), rotate_slack(src, n), f"{D} {sections} {dt}")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [(128, (24, 20, 20)), (72, (18, 18)), (96, (12, 10, 10)), (64, (32,)),
                                        (2, (1,)), (6, (1, 0, 2)), (256, (64, 30, 34)), (512, (256,)),
                                        (130, (3, 5, 7, 11)), (66, (16, 16)), (98, (48,))])
def test_head_sizes_and_sections(D, sections, interleaved, dt):
    check(2, 19, 6, 3, D, sections, dt, interleaved)


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (1, 1, 64, 8), (32, 1, 32, 8), (3, 777, 5, 1), (1, 5000, 2, 2),
                                       (7, 33, 40, 40), (2, 1200, 1, 1)])
@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
def test_shapes_and_layouts(B, S, Hq, Hk, layout):
    check(B, S, Hq, Hk, 64, (10, 12, 10), "bf16", layout=layout)


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32])
def test_position_types(ptype):
    check(2, 50, 4, 2, 64, (16, 16), "f32", ptype=ptype)


@pytest.mark.parametrize("reach", [2 ** 20, 2 ** 31, 2 ** 40])
def test_far_positions(reach):
    check(1, 64, 2, 1, 128, (24, 20, 20), "f32", reach=reach)


def test_negative_positions_and_shared_over_the_batch():
    q, k, pos, inv, _, _ = make(3, 40, 4, 2, 64, (16, 16), "f32")
    one = pos[:, 0] - 2500
    qo, ko = apply_multi_axis_rotary(q, k, one, inv, (16, 16))
    turn = turns_exact(one, inv, axis_of_pairs((16, 16)))
    assert_within(qo, rotate_exact(q, turn.expand(3, -1, -1)), rotate_slack(q, 32))
    assert_within(ko, rotate_exact(k, turn.expand(3, -1, -1)), rotate_slack(k, 32))


def test_strided_positions_and_inputs():
    """Positions taken from a [batch, seq, axes] tensor, heads cut from a fused qkv buffer, an odd offset."""
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2, 30, 12 * 64 + 1, generator=g).cuda().bfloat16()
    pos = torch.randint(0, 900, (2, 30, 3), generator=g).cuda().permute(2, 0, 1)
    inv = (1.0 / 10000.0 ** (torch.arange(32).float() / 32)).cuda()
    for off in (0, 1):
        q = qkv[..., off:off + 8 * 64].unflatten(-1, (8, 64)).transpose(1, 2)
        k = qkv[..., off + 512:off + 768].unflatten(-1, (4, 64)).transpose(1, 2)
        qo, ko = apply_multi_axis_rotary(q, k, pos, inv, (12, 10, 10))
        turn = turns_exact(pos, inv, axis_of_pairs((12, 10, 10)))
        assert_within(qo, rotate_exact(q, turn), rotate_slack(q, 32))
        assert_within(ko, rotate_exact(k, turn), rotate_slack(k, 32))


def test_broadcast_inputs_and_transposed_last_axis():
    g = torch.Generator().manual_seed(2)
    inv = torch.ones(4, device="cuda")
    pos = torch.arange(5, device="cuda")[None].expand(2, 5)
    q = torch.randn(1, 1, 5, 8, generator=g).cuda().expand(3, 6, 5, 8).requires_grad_()  # shared heads
    k = torch.randn(3, 2, 8, 5, generator=g).cuda().transpose(2, 3).requires_grad_()
    qo, ko = apply_multi_axis_rotary(q, k, pos, inv, (2, 2))
    turn = turns_exact(pos, inv, axis_of_pairs((2, 2))).expand(3, -1, -1)
    assert_within(qo.detach(), rotate_exact(q, turn), rotate_slack(q, 4))
    assert_within(ko.detach(), rotate_exact(k, turn), rotate_slack(k, 4))
    gq = torch.randn(6, 5, 8, generator=g).cuda().expand(3, 6, 5, 8)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, torch.ones_like(ko)))
    assert_within(dq, rotate_exact(gq, turn.conj()), rotate_slack(gq, 4))
    assert_within(dk, rotate_exact(torch.ones_like(ko), turn.conj()), rotate_slack(torch.ones_like(ko), 4))


def test_gradient_of_a_shared_leaf():
    """One key head used for every query group: its gradient is the sum over the uses."""
    q, k, pos, inv, gq, _ = make(2, 21, 6, 1, 32, (8, 8), "f32")
    k.requires_grad_()
    out, _ = apply_multi_axis_rotary(k.expand(2, 6, 21, 32), None, pos, inv, (8, 8))
    (dk,) = torch.autograd.grad(out, k, gq)
    turn = turns_exact(pos, inv, axis_of_pairs((8, 8))).conj()
    slack = rotate_slack(gq, 16).sum(1, keepdim=True) + 6 * 2.0 ** -24 * gq.abs().double().cpu().sum(1, keepdim=True)
    assert_within(dk, rotate_exact(gq, turn).sum(1, keepdim=True), slack)


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_result_unused(which):
    q, k, pos, inv, gq, gk = make(1, 17, 4, 2, 64, (16, 16), "bf16")
    q.requires_grad_()
    k.requires_grad_()
    qo, ko = apply_multi_axis_rotary(q, k, pos, inv, (16, 16))
    out, g = (qo, gq) if which == "q" else (ko, gk)
    dq, dk = torch.autograd.grad(out, (q, k), g, allow_unused=True)
    turn = turns_exact(pos, inv, axis_of_pairs((16, 16))).conj()
    got, none = (dq, dk) if which == "q" else (dk, dq)
    assert none is None
    assert_within(got, rotate_exact(g, turn), rotate_slack(g, 32))


def test_empty_and_without_k():
    inv = torch.ones(4, device="cuda")
    pos = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    q = torch.empty(2, 3, 0, 8, device="cuda", requires_grad=True)
    qo, ko = apply_multi_axis_rotary(q, None, pos, inv, (4,))
    assert qo.shape == q.shape and ko is None
    assert torch.autograd.grad(qo.sum(), q)[0].shape == q.shape


def test_same_position_on_every_axis_is_the_one_axis_embedding():
    """bf16 operations of the one-axis embedding round its tables, products and sum: half a step each of values up to
    |a| + |b|, against one rounding here."""
    B, S, D = 2, 130, 128
    emb = MultiAxisRotaryEmbedding(D, (24, 20, 20)).cuda().bfloat16()
    assert emb.inv_freq.dtype == torch.float32
    q = torch.randn(B, 4, S, D, generator=torch.Generator().manual_seed(4)).cuda().bfloat16()
    pos = torch.arange(S, device="cuda").expand(3, S)
    got, _ = emb(q, None, pos)
    cos, sin = RotaryEmbedding(D, S).cuda()(S, q.device, q.dtype)
    want, _ = apply_rotary_pos_emb(q, q, cos, sin)
    m = q.double().abs()
    pair = (m[..., :64] + m[..., 64:]).repeat(1, 1, 1, 2)
    # the float32 tables' angles are off by up to 2^-24 of a position up to 129
    assert bool(((got.double() - want.double()).abs() <= (5 * 2.0 ** -8 + 129 * 2.0 ** -23) * pair).all())


def test_other_stream_and_graph_replay():
    q, k, pos, inv, gq, gk = make(2, 64, 8, 4, 128, (24, 20, 20), "bf16")
    q.requires_grad_()
    k.requires_grad_()

    def once():
        out = apply_multi_axis_rotary(q, k, pos, inv, (24, 20, 20))
        return [o.detach() for o in out] + list(torch.autograd.grad(out, (q, k), (gq, gk)))

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
        q.mul_(-2)
        pos.add_(11)
    graph.replay()
    held = [t.clone() for t in held]
    for a, b in zip(held, once()):
        assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    q, _, pos, inv, _, _ = make(1, 4, 2, 1, 32, (16,), "f32")
    q.requires_grad_()
    out, _ = apply_multi_axis_rotary(q, None, pos, inv, (16,))
    (dq,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.sum().backward()


def test_no_query_heads_and_many_heads():
    g = torch.Generator().manual_seed(6)
    inv = (1.0 / 100.0 ** (torch.arange(8).float() / 8)).cuda()
    pos = torch.randint(0, 99, (2, 2, 3), generator=g).cuda()
    turn = turns_exact(pos, inv, axis_of_pairs((4, 4)))
    for Hq, Hk in ((0, 3), (3, 0), (0, 0), (700, 1), (1, 300)):
        q, k = (torch.randn(2, n, 3, 20, generator=g).cuda() for n in (Hq, Hk))
        qo, ko = apply_multi_axis_rotary(q, k, pos, inv, (4, 4))
        assert_within(qo, rotate_exact(q, turn), rotate_slack(q, 8))
        assert_within(ko, rotate_exact(k, turn), rotate_slack(k, 8))


def test_many_axes():
    g = torch.Generator().manual_seed(7)
    n = 64
    inv = (1.0 / 100.0 ** (torch.arange(n).float() / n)).cuda()
    pos = torch.randint(0, 99, (n, 3, 50), generator=g).cuda()
    q = torch.randn(3, 2, 50, 2 * n, generator=g).cuda()
    for interleaved in (False, True):
        qo, _ = apply_multi_axis_rotary(q, None, pos, inv, (1,) * n, interleaved)
        turn = turns_exact(pos, inv, axis_of_pairs((1,) * n, interleaved))
        assert_within(qo, rotate_exact(q, turn), rotate_slack(q, n))


def test_every_head_and_token_count_has_its_heads_once():
    """The launch splits heads and tokens by rules on their numbers: small grids of both."""
    for Hq, Hk, D, secs in ((1, 1, 64, (32,)), (5, 2, 96, (16, 16)), (33, 8, 128, (64,)), (7, 0, 12, (3, 1))):
        for S in (1, 2, 15, 148, 400, 1500):
            check(1, S, Hq, Hk, D, secs, "bf16", seed=S) if Hk else None
            q, _, pos, inv, _, _ = make(1, S, Hq, 1, D, secs, "f32", seed=S + 1)
            qo, _ = apply_multi_axis_rotary(q, None, pos, inv, secs)
            assert_within(qo, rotate_exact(q, turns_exact(pos, inv, axis_of_pairs(secs))), rotate_slack(q, sum(secs)))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,pairs", [(96, 7), (80, 29), (190, 93), (100, 2), (67, 33), (130, 65), (77, 20), (48, 16)])
def test_pairs_and_copied_columns_of_every_alignment(D, pairs, dt):
    check(2, 37, 5, 3, D, (pairs,), dt, seed=D)


@pytest.mark.parametrize("B,S,Hq,Hk,D,sections,dt", [
    (2, 4096, 13, 3, 64, (32,), "bf16"), (1, 6001, 20, 5, 96, (12, 10, 10), "bf16"), (1, 9000, 24, 6, 34, (5, 12), "bf16"),
    (3, 3000, 1, 17, 20, (1, 3), "bf16"), (1, 5000, 18, 1, 38, (19,), "f32"), (2, 2500, 7, 9, 128, (40, 24), "f32"),
    (1, 700, 70, 70, 32, (7, 9), "bf16")])
@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
def test_threads_that_walk_many_heads(B, S, Hq, Hk, D, sections, dt, layout):
    """Enough tokens that a thread takes up to 16 heads one after the other, from q over to k."""
    check(B, S, Hq, Hk, D, sections, dt, layout=layout, seed=Hq)


@pytest.mark.parametrize("D,sections,dt", [(96, (0, 2, 1, 2), "bf16"), (128, (32,), "bf16"), (80, (5,), "f32"),
                                           (96, (0, 7), "f32"), (68, (2, 13), "bf16"), (20, (1, 3), "bf16"),
                                           (190, (81, 12), "bf16"), (128, (6,), "bf16"), (128, (8,), "bf16"), (40, (1,), "f32")])
def test_copied_columns_of_many_heads(D, sections, dt):
    """Heads with more copied columns than a thread each, and with fewer."""
    check(2, 1500, 17, 4, D, sections, dt, seed=D)
    check(1, 40, 3, 8, D, sections, dt, layout="bhsd", seed=D)
