"""``quantize_int8`` and ``int8_linear`` on CUDA: the integers equal the definition's, the products their 64-bit value."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200.quantization import Int8Linear, QuantizedLinear, int8_linear, quantize_int8
from tests.bounds import INT8_SLACK, assert_within, int8_exact

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(M, N, K, dt="bf16", bias=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * (1 + 7 * (torch.randn(K, generator=g) > 2))).to(TD[dt])
    w = torch.randn(N, K, generator=g) * (0.1 + torch.rand(N, 1, generator=g))
    b = torch.randn(N, generator=g) if bias else None
    wq, ws = quantize_int8(w.cuda())
    return x.cuda(), wq, ws, None if b is None else b.cuda()


def check(M, N, K, dt="bf16", bias=False, seed=0):
    x, wq, ws, b = make(M, N, K, dt, bias, seed)
    y = int8_linear(x, wq, ws, b)
    assert y.dtype == x.dtype and y.shape == (M, N)
    e, mag = int8_exact(x, wq, ws, b)
    assert_within(y, e, INT8_SLACK * mag, f"{M} {N} {K} {dt}")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 17), (5, 255), (64, 256), (7, 1000), (33, 4096), (2, 8200), (3, 30001),
                                    (1, 131072)])
def test_quantised_integers_equal_the_definition(rows, K, dt):
    g = torch.Generator().manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g).to(TD[dt])
    x[0] *= 1e-20
    q, s = quantize_int8(x.cuda())
    qc, sc = quantize_int8(x)  # the CPU runs the definition in torch operations
    assert q.dtype == torch.int8 and torch.equal(q.cpu(), qc) and torch.equal(s.cpu(), sc)
    assert q.stride(0) % 16 == 0


def test_ties_zeros_and_tiny_rows():
    """Halves of the largest value land on 63.5 steps, rounded as float32 rounds x * (127 / amax)."""
    x = torch.zeros(6, 64)
    x[0, 0], x[0, 1], x[0, 2] = 2.0, 1.0, -1.0
    x[2] = 1e-38
    x[3] = torch.arange(64).float() * 2.0 ** -30
    x[4] = -127.0
    x[5] = torch.linspace(-127, 127, 64)
    for dt in (torch.float32, torch.bfloat16):
        t = x.to(dt)
        q, s = quantize_int8(t.cuda())
        qc, sc = quantize_int8(t)
        assert torch.equal(q.cpu(), qc) and torch.equal(s.cpu(), sc)
        assert int(q[1].abs().max()) == 0 and bool(s.isfinite().all())


def test_non_finite_rows_are_nan_and_stay_apart():
    x, wq, ws, b = make(6, 40, 96, "f32", True)
    x[1, 5], x[3, 0], x[4, 95] = float("inf"), float("nan"), float("-inf")
    y = int8_linear(x, wq, ws, b)
    q, s = quantize_int8(x)
    for r in range(6):
        if r in (1, 3, 4):
            assert y[r].isnan().all() and s[r].isnan() and int(q[r].abs().max()) == 0
        else:
            e, mag = int8_exact(x[r:r + 1], wq, ws, b)
            assert_within(y[r:r + 1], e, INT8_SLACK * mag)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127, 128, 129, 200, 256, 257,
                               300, 512, 777])
def test_token_counts(M):
    check(M, 384, 512, seed=M)


@pytest.mark.parametrize("N,K", [(1, 1), (1, 64), (2, 16), (15, 15), (16, 31), (127, 128), (128, 129), (129, 250),
                                 (130, 4096), (1003, 1001), (2048, 48), (4096, 4096), (256, 11008), (600, 640)])
@pytest.mark.parametrize("M", [1, 6, 40, 150])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_feature_counts(M, N, K, dt):
    check(M, N, K, dt, bias=True, seed=N + K)


@pytest.mark.parametrize("M,N,K", [(2048, 1024, 2048), (1111, 2056, 1000), (4100, 520, 272), (700, 11264, 512), (5001, 1003, 260),
                                   (2000, 3001, 500), (4500, 4500, 64), (2304, 4096, 16), (1400, 2500, 130)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_larger_products(M, N, K, dt):
    check(M, N, K, dt, bias=True)


def test_the_longest_sum_does_not_overflow():
    """131072 products of 127 * 127 (and -128 in a weight given by hand) in int32."""
    K = 131072
    for M in (1, 20, 140):
        x = torch.ones(M, K, device="cuda")
        w = torch.full((3, K), 127, dtype=torch.int8, device="cuda")
        w[1] = -128
        w[2, ::2] = -127
        s = torch.ones(3, device="cuda")
        y = int8_linear(x, w, s)
        e, mag = int8_exact(x, w, s)
        assert_within(y, e, INT8_SLACK * mag)


def test_strides_views_and_leading_axes():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4, 6, 200, generator=g).cuda()
    w = torch.randn(64, 100, generator=g).cuda()
    wq, ws = quantize_int8(w)
    part = x[:, 1:5, 7:107]  # strided rows at an odd offset
    y = int8_linear(part, wq, ws)
    e, mag = int8_exact(part.reshape(-1, 100), wq, ws)
    assert_within(y.view(-1, 64), e, INT8_SLACK * mag)
    assert torch.equal(int8_linear(part, wq.contiguous(), ws), y)  # rows of 100 bytes: copied
    assert torch.equal(int8_linear(part, wq.t().contiguous().t(), ws), y)
    rows = x[0, :, :100]
    assert torch.equal(int8_linear(rows.t().contiguous().t(), wq, ws), int8_linear(rows.contiguous(), wq, ws))
    one = x[0, 0, :100]
    assert torch.equal(int8_linear(one, wq, ws), int8_linear(one[None], wq, ws)[0])
    assert int8_linear(x[:0, 0, :100], wq, ws).shape == (0, 64)
    q3, s3 = quantize_int8(part)
    q2, s2 = quantize_int8(part.reshape(-1, 100))
    assert torch.equal(q3.reshape(-1, 100), q2) and torch.equal(s3.reshape(-1), s2)
    q1, s1 = quantize_int8(one)
    assert q1.shape == (100,) and s1.shape == () and torch.equal(q1, quantize_int8(one[None])[0][0])


def test_bytes_past_the_features_are_not_used():
    """A weight that is a view of wider rows whose other bytes hold anything."""
    for M in (1, 7, 40, 150, 600):
        x, wq, ws, _ = make(M, 200, 90, "f32")
        wide = torch.randint(-128, 128, (200, 112), dtype=torch.int8, device="cuda")
        wide[:, :90] = wq
        assert torch.equal(int8_linear(x, wide[:, :90], ws), int8_linear(x, wq, ws))


def test_a_token_does_not_depend_on_its_batch():
    """Integer sums are exact, so every batch size gives a token the same result."""
    x, wq, ws, b = make(1100, 640, 1024, "bf16", True)
    whole = int8_linear(x, wq, ws, b)
    for n in (1, 3, 8, 30, 100, 128, 400):
        assert torch.equal(int8_linear(x[:n], wq, ws, b), whole[:n])


@pytest.mark.parametrize("M", [2, 50, 900])
def test_other_stream_and_graph_replay(M):
    x, wq, ws, b = make(M, 512, 768, "bf16", True)
    want = int8_linear(x, wq, ws, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8_linear(x, wq, ws, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    graphs, held = [], []
    for _ in range(2):  # two graphs of one pool, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            held.append(int8_linear(x, wq, ws, b))
        graphs.append(g)
    x.copy_(torch.randn_like(x))
    want = int8_linear(x, wq, ws, b)
    for g, h in zip(graphs, held):
        g.replay()
        assert torch.equal(h, want)


def test_modules():
    lin = torch.nn.Linear(300, 120).cuda()
    q = Int8Linear.from_linear(lin)
    x = torch.randn(5, 300, device="cuda")
    e, mag = int8_exact(x, q.weight, q.scale, q.bias)
    assert_within(q(x), e, INT8_SLACK * mag)
    # against the float layer: half a step of weight and activation each
    step = (x.abs().amax(-1, keepdim=True) / 127).double() / 2 * lin.weight.double().abs().sum(1) \
        + q.scale.double() / 2 * (x.double().abs().sum(-1, keepdim=True) * 1.01)
    assert bool(((q(x).double() - lin(x).double()).abs() <= 1.01 * step + 1e-4).all())
    back = Int8Linear(300, 120, bias=True)
    back.load_state_dict(q.state_dict())
    back = back.cuda()
    assert back.weight.stride(0) % 16 == 0 and torch.equal(back(x), q(x))
    half = Int8Linear.from_linear(lin).to(torch.bfloat16)
    assert half.scale.dtype == torch.float32 and half.weight.dtype == torch.int8
    assert half(x.bfloat16()).dtype == torch.bfloat16
    qat = QuantizedLinear(64, 32, "int8")
    served = Int8Linear.from_linear(qat).cuda()
    assert served(torch.randn(2, 64, device="cuda")).shape == (2, 32)


def test_two_streams_at_once_and_fresh_weights():
    """Calls on two streams, each right after its weights were written on that stream."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    for M in (1, 24, 300, 2100):
        data = [make(M, 1536, 1024, "bf16", True, seed=M + i) for i in range(2)]
        want = [int8_linear(*d) for d in data]
        torch.cuda.synchronize()
        for _ in range(4):
            got = []
            for st, (x, w, s, b) in zip(streams, data):
                with torch.cuda.stream(st):
                    w2, s2, x2 = torch.empty_like(w), torch.empty_like(s), torch.empty_like(x)
                    x2.copy_(x)
                    s2.copy_(s)
                    w2.copy_(w)  # the last thing before the product reads it
                    got.append(int8_linear(x2, w2, s2, b))
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_in_a_row_do_not_meet():
    """Each call's product starts before its quantisation has ended: a chain of calls on new inputs in reused memory."""
    for M in (1, 12, 64, 500, 2200):
        x, w, s, _ = make(M, 1024, 1024, "bf16")
        w = torch.where(torch.rand(w.shape, device="cuda") < 0.1, w, torch.zeros_like(w))
        chain = [x]
        for _ in range(6):
            chain.append(int8_linear(chain[-1], w, s))
        for a, b in zip(chain, chain[1:]):
            e, mag = int8_exact(a, w, s)
            assert_within(b, e, INT8_SLACK * mag)


@pytest.mark.parametrize("K", [1, 2, 15, 17, 18, 511, 512, 514, 2047, 2049, 2050, 8191, 8194, 33001, 33002, 33024])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rows_of_every_alignment(K, dt):
    """Rows that start at any element, read 16, 4 or 2 bytes at a time, from one warp to a row to longer ones than its
    threads hold; the largest value, or what is not finite, at the end of a row, and values past it that do not count."""
    rows = 5
    g = torch.Generator().manual_seed(K)
    for start, behind in ((0, 0), (1, 0), (2, 2), (0, 1), (8, 8), (3, 5)):
        whole = torch.randn(rows, start + K + behind, generator=g).to(TD[dt])
        whole[:, :start] = float("nan")
        whole[:, start + K:] = float("inf")
        whole[0, start + K - 1] = 50.0
        whole[1, start + K - 1] = float("nan")
        whole[2, start] = -50.0
        q, s = quantize_int8(whole.cuda()[:, start:start + K])
        qc, sc = quantize_int8(whole[:, start:start + K])
        assert torch.equal(q.cpu(), qc) and torch.equal(s.cpu().nan_to_num(-1), sc.nan_to_num(-1))


@pytest.mark.parametrize("M,N,K", [(5, 10000, 3200), (30, 10000, 3201), (48, 11008, 4096), (64, 10120, 3300), (20, 2900, 1600),
                                   (10, 5000, 6200), (31, 2999, 1700), (40, 4096, 8192), (2, 2900, 1600)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_clusters_of_every_size(M, N, K, dt):
    """K in 3, 4, 6 and 8 parts on 148 SMs, tokens that the parts share unevenly."""
    check(M, N, K, dt, bias=True, seed=M)
