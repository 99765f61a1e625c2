"""Operators around a transformer block's matrix products, measured: the gated double norm at a block's end, the
rotary embedding with several position axes, and the 8-bit integer projection.

``listed()`` names fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass, ``work(case)`` its unavoidable bytes and operations, and
``exact(case, seed)`` the result in 64 bits.  With ``own`` false ``run`` computes each operator's plain form with
elementary torch operations in 32 bits; with ``own`` true it calls ``ats_v2_b200``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # -- the end of a block: post-norm, gate, scaled residual, the next block's pre-norm
        # one decoding step of 8 sequences
        _norm("norm_decode_8x4096", 8, 1, 4096, "bf16", "channel", 1.0, False),
        # a training step of a 7B-sized block (hidden 4096, 4 sequences of 4096 tokens), per-channel gate
        _norm("norm_train_16384x4096", 4, 4096, 4096, "bf16", "channel", 0.5, True),
        # a conditioned block (one gate row per sequence) of hidden 2048 with sequences of odd length
        _norm("norm_train_sequence_gate", 6, 1023, 2048, "bf16", "sequence", 1.0, True),
        # float32 training of a small odd width, a gate for every token
        _norm("norm_train_f32_token_gate", 5, 333, 1030, "f32", "token", 0.8, True),
        # -- rotary embedding over time, height and width
        # one decoding step of 32 sequences, positions far into long contexts
        _rope("rope_decode_32", 32, 1, 32, 8, 128, "24,20,20", False, "bf16", False, 200000),
        # a training step of the 7B-sized attention (32 query and 8 key heads of 128)
        _rope("rope_train_4x4096", 4, 4096, 32, 8, 128, "24,20,20", False, "bf16", True, 4096),
        # the patches of one image: two axes, heads of 72, float32
        _rope("rope_image_f32", 1, 5041, 16, 16, 72, "18,18", False, "f32", False, 71),
        # a training step with odd length and dealt-out pairs, 64 of the 96 dimensions rotated
        _rope("rope_train_partial", 3, 777, 20, 5, 96, "12,10,10", True, "bf16", True, 60000),
        # -- projections with 8-bit weights and per-token activations
        # one token through an attention projection
        _int8("int8_token_4096x4096", 1, 4096, 4096, "bf16", False),
        # a decoding batch through the up projection of a 7B-sized FFN
        _int8("int8_batch48_11008x4096", 48, 11008, 4096, "bf16", False),
        # a ragged float32 batch with bias and sizes that are no multiple of anything
        _int8("int8_ragged_777x1003x1001", 777, 1003, 1001, "f32", True),
        # prefill through the gate and up projections of the 8192-token MoE configuration's expert width
        _int8("int8_prefill_8192x11264x2048", 8192, 11264, 2048, "bf16", False),
    ]


def _norm(name, batch, seq, hidden, dtype, gate, scale, train):
    return {"name": name, "op": "norm", "batch": batch, "seq": seq, "hidden": hidden, "dtype": dtype, "gate": gate,
            "residual_scale": scale, "train": train}


def _rope(name, batch, seq, q_heads, k_heads, dim, sections, interleaved, dtype, train, reach):
    return {"name": name, "op": "rope", "batch": batch, "seq": seq, "q_heads": q_heads, "k_heads": k_heads,
            "dim": dim, "sections": sections, "interleaved": interleaved, "dtype": dtype, "train": train,
            "reach": reach}


def _int8(name, tokens, out_features, in_features, dtype, bias):
    return {"name": name, "op": "int8", "tokens": tokens, "out_features": out_features, "in_features": in_features,
            "dtype": dtype, "bias": bias}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "int8"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        hidden = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            hidden = max(64, hidden // 64 * 64)
        batch = rng.randint(1, 8)
        seq = _log(rng, 1, max(1, min(8192, 4 * 4096 * 4096 // (hidden * batch))))
        case = _norm("", batch, seq, hidden, dtype, rng.choice(["none", "channel", "sequence", "token"]),
                     rng.choice([1.0, 0.5, 1.4]), rng.random() < 0.6)
    elif op == "rope":
        dim = 2 * rng.randint(8, 128) if rng.random() < 0.4 else rng.choice([64, 80, 96, 128, 256])
        pairs = dim // 2 if rng.random() < 0.6 else rng.randint(4, dim // 2)
        axes = rng.randint(1, 4)
        cuts = sorted(rng.randint(0, pairs) for _ in range(axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
        k_heads = rng.choice([1, 2, 4, 5, 8, 16])
        q_heads = min(64, k_heads * rng.choice([1, 1, 2, 4, 5, 8]))
        batch = rng.randint(1, 8)
        seq = _log(rng, 1, max(1, min(8192, 4 * 4096 * 40 * 128 // (batch * (q_heads + k_heads) * dim))))
        case = _rope("", batch, seq, q_heads, k_heads, dim, sections, rng.random() < 0.5, dtype, rng.random() < 0.5,
                     _log(rng, 16, 1000000))
    else:
        tokens, inf = _log(rng, 1, 8192), _log(rng, 16, 11264)
        outf = _log(rng, 16, 11264)
        if rng.random() < 0.5:
            outf, inf = max(16, outf // 16 * 16), max(16, inf // 16 * 16)
        while tokens * inf * outf > 8192 * 2048 * 11264:
            tokens = max(1, tokens // 2)
        case = _int8("", tokens, outf, inf, dtype, rng.random() < 0.4)
    del case["name"]
    return case


def _sections(case):
    return tuple(int(v) for v in case["sections"].split(","))


def _inv_freq(pairs, theta=500000.0):
    return 1.0 / (theta ** (torch.arange(pairs, dtype=torch.float32, device="cuda") / pairs))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    st = {"case": dict(case)}
    if case["op"] == "norm":
        B, S, H = case["batch"], case["seq"], case["hidden"]
        # a block's output has some channels far larger than the rest; the residual stream is wider still
        x = (randn(B, S, H) * (1 + 6 * (randn(H) > 2.2))).to(dt)
        res = (randn(B, S, H) * (1 + 20 * (randn(H) > 2.5))).to(dt)
        shape = {"none": None, "channel": (H,), "sequence": (B, 1, H), "token": (B, S, H)}[case["gate"]]
        gate = None if shape is None else 0.3 * randn(*shape)
        if gate is not None and case["gate"] != "channel":  # computed by a projection, in the activations' type
            gate = gate.to(dt)
        st |= {"x": x, "residual": res, "gate": gate, "post": 1 + 0.1 * randn(H), "pre": 1 + 0.1 * randn(H)}
        st["leaves"] = [st[n] for n in ("x", "residual", "post", "pre", "gate") if st[n] is not None]
        if case["train"]:
            st["grads"] = [randn(B, S, H).to(dt), randn(B, S, H).to(dt)]
    elif case["op"] == "rope":
        B, S, D = case["batch"], case["seq"], case["dim"]
        secs = _sections(case)

        def heads(n):  # the projection's [batch, seq, heads, dim] memory seen as [batch, heads, seq, dim]
            return randn(B, S, n, D).to(dt).transpose(1, 2)

        st |= {"q": heads(case["q_heads"]), "k": heads(case["k_heads"]), "sections": secs,
               "inv_freq": _inv_freq(sum(secs)),
               "positions": torch.randint(0, case["reach"], (len(secs), B, S), generator=g, device="cuda")}
        st["leaves"] = [st["q"], st["k"]]
        if case["train"]:
            st["grads"] = [heads(case["q_heads"]), heads(case["k_heads"])]
    else:
        M, N, K = case["tokens"], case["out_features"], case["in_features"]
        x = (randn(M, K) * (1 + 8 * (randn(K) > 2.4))).to(dt)
        w = randn(N, K) * (0.02 + 0.01 * randn(N, 1).abs())
        scale = w.abs().amax(-1) / 127
        data = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :K]  # rows start every 16 bytes
        data.copy_(torch.round(w / scale[:, None]))
        st |= {"x": x, "weight": data, "scale": scale, "bias": randn(N).to(dt) if case["bias"] else None}
        st["leaves"] = []
    if case.get("train"):
        for t in st["leaves"]:
            t.requires_grad_(True)
    return st


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        out = _run_norm(state, case)
    elif case["op"] == "rope":
        out = _run_rope(state, case)
    else:
        return [_run_int8(state)]
    if not case["train"]:
        return list(out)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, state["leaves"], state["grads"]))


def _run_norm(state, case):
    if own:
        from ats_v2_b200.norm_fused import fused_sandwich_norm

        return fused_sandwich_norm(state["x"], state["residual"], state["post"], state["pre"], gate=state["gate"],
                                   residual_scale=case["residual_scale"], eps=1e-5)
    x, dt = state["x"].float(), state["x"].dtype
    p = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * state["post"].float()
    if state["gate"] is not None:
        p = p * state["gate"].float()
    s = state["residual"].float() * case["residual_scale"] + p
    h = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-5) * state["pre"].float()
    return h.to(dt), s.to(dt)


def _axis_of_pair(sections, interleaved):
    """The position axis of each rotated pair: section by section, or dealt out in turn to the axes with pairs left."""
    pairs = [(i, a) for a, n in enumerate(sections) for i in range(n)]
    return [a for _, a in (sorted(pairs) if interleaved else pairs)]


def _run_rope(state, case):
    if own:
        from ats_v2_b200.rope import apply_multi_axis_rotary

        return apply_multi_axis_rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                                       state["sections"], interleaved=case["interleaved"])
    axes = _axis_of_pair(state["sections"], case["interleaved"])
    # far positions: the angle in 64 bits, its cosine and sine in 32
    angle = state["positions"].double()[axes].permute(1, 2, 0) * state["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = len(axes)

    def rotate(t):
        f = t.float()
        a, b, rest = f[..., :half], f[..., half:2 * half], f[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(t.dtype)

    return rotate(state["q"]), rotate(state["k"])


def _run_int8(state):
    if own:
        from ats_v2_b200.quantization import int8_linear

        return int8_linear(state["x"], state["weight"], state["scale"], bias=state["bias"])
    x = state["x"].float()
    amax = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    full = torch.full_like(amax, 127)  # tensor by tensor, so that both quotients are correctly rounded
    q = torch.round(x * (full / amax))
    acc = (q.double() @ state["weight"].double().t()).float()  # integers past 2^24: summed in 64 bits
    y = acc * ((amax / full) * state["scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        rows, H = case["batch"] * case["seq"], case["hidden"]
        gate = {"none": 0, "channel": 4 * H, "sequence": case["batch"] * H * es, "token": rows * H * es}[case["gate"]]
        fixed = 8 * H + gate
        if not case["train"]:
            return {"bytes": 4 * rows * H * es + fixed, "flops": 12 * rows * H}
        # forward: x and the residual in, both results out; backward: those and two gradients in, two gradients out
        return {"bytes": 10 * rows * H * es + 3 * fixed, "flops": 40 * rows * H}
    if case["op"] == "rope":
        n = case["batch"] * case["seq"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        passes = 2 if case["train"] else 1
        fixed = case["batch"] * case["seq"] * len(_sections(case)) * 8
        return {"bytes": passes * (2 * n * es + fixed), "flops": passes * 3 * n}
    M, N, K = case["tokens"], case["out_features"], case["in_features"]
    return {"bytes": M * K * es + N * K + 4 * N + M * N * es + (N * es if case["bias"] else 0), "flops": 2 * M * N * K}


def exact(case, seed):
    """The operators' definitions in 64 bits: closed-form gradients, rotation as complex multiplication, and the
    product of the dequantised numbers."""
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(st, case)
        if case["op"] == "rope":
            return _exact_rope(st, case)
        # the quantised values are float32 by definition; what is made of them is in 64 bits
        x = st["x"].float()
        top = torch.maximum(x.max(-1).values, -x.min(-1).values).clamp(min=2.0 ** -100)
        top = top.unsqueeze(1)
        steps = torch.full_like(top, 127)
        left = (x * (steps / top)).round().double() * (top / steps).double()
        y = torch.einsum("mk,nk->mn", left, st["weight"].double() * st["scale"].double().unsqueeze(1))
        return [y if st["bias"] is None else y + st["bias"].double()]


def _exact_norm(st, case):
    H, eps, a = case["hidden"], 1e-5, case["residual_scale"]
    x, r = st["x"].double(), st["residual"].double()
    wp, wn = st["post"].double(), st["pre"].double()
    g = 1.0 if st["gate"] is None else st["gate"].double()
    rx = (x.square().sum(-1, keepdim=True) / H + eps).pow(-0.5)
    xn = x * rx
    s = a * r + g * wp * xn
    rs = (s.square().sum(-1, keepdim=True) / H + eps).pow(-0.5)
    out = [s * rs * wn, s]
    if not case["train"]:
        return out
    dh, ds = (t.double() for t in st["grads"])
    u = dh * wn
    ds = ds + rs * u - s * rs.pow(3) * ((u * s).sum(-1, keepdim=True) / H)
    dpre = (dh * s * rs).sum((0, 1))
    v = ds * g * wp
    dx = rx * v - x * rx.pow(3) * ((v * x).sum(-1, keepdim=True) / H)
    out += [dx, a * ds, (ds * g * xn).sum((0, 1)), dpre]
    if st["gate"] is not None:
        dg = ds * wp * xn
        out.append({"channel": lambda: dg.sum((0, 1)), "sequence": lambda: dg.sum(1, keepdim=True),
                    "token": lambda: dg}[case["gate"]]())
    return out


def _exact_rope(st, case):
    secs = torch.tensor(st["sections"], device="cuda")
    axis = torch.repeat_interleave(torch.arange(secs.numel(), device="cuda"), secs)
    if case["interleaved"]:  # the first pair of every axis, then the second of every axis, ...
        nth = torch.arange(axis.numel(), device="cuda") - (secs.cumsum(0) - secs)[axis]
        axis = axis[torch.argsort(nth, stable=True)]
    n = axis.numel()
    pos = torch.stack([st["positions"][int(i)] for i in axis], -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double() * st["inv_freq"].double())

    def turned(t, by):
        z = torch.complex(t[..., :n].double(), t[..., n:2 * n].double()) * by.unsqueeze(1)
        return torch.cat([z.real, z.imag, t[..., 2 * n:].double()], -1)

    out = [turned(st["q"], turn), turned(st["k"], turn)]
    if case["train"]:
        out += [turned(t, turn.conj()) for t in st["grads"]]
    return out
