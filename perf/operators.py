"""Operators next to the KDA path, as their users call them: the gated delta rule with one decay per head (training, prompts,
decoding) and group normalisation with an activation over channels-last activations.

  train     ``chunk_gated_delta_rule`` forward and backward, dense batches or packed documents
  prefill   ``chunk_gated_delta_rule`` under ``no_grad``: a prompt in, outputs and the state for decoding out
  burst     ``fused_recurrent_gated_delta_rule``: a few tokens per sequence
  step      ``recurrent_gated_delta_rule_step``: one token per sequence, the state updated in place
  norm      ``group_norm``, forward, or forward and backward

Values: q, k, v, do ~ N(0,1); with ``gate`` the decay is -exp(A_log) softplus(a + dt_bias) of a gate input a ~ N(0,1) with
A ~ U(1,16) and a step softplus(dt_bias) ~ logU(0.001, 0.1), so that slow heads remember thousands of tokens and fast ones a
few; beta is the sigmoid of N(0,1); without ``gate`` the log decay itself and beta are given in FP32.  Initial states ~ N(0, 0.3).
Activations of the norm ~ N(m, s) with an offset m ~ N(0,1) per channel.
"""

from __future__ import annotations

import math

import torch
from torch.utils.checkpoint import checkpoint

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
CHUNK = 64
NORM_EPS = 1e-5


def listed():
    return [
        # one layer's training step on the primary batch of the benchmark
        dict(name="train_primary", kind="train", batch=16, time=2048, heads=6, vheads=6, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=False),
        # documents of uneven length packed into one row, two value heads per key head, a state carried in and out
        dict(name="train_packed", kind="train", batch=1, time=24571, heads=4, vheads=8, kdim=128, vdim=128, dtype="bf16", docs=12, gate=True, state=True),
        # the FP32 mode that other runs are validated against: given log decays, narrow keys, wide values
        dict(name="train_fp32", kind="train", batch=2, time=509, heads=2, vheads=4, kdim=64, vdim=128, dtype="fp32", docs=0, gate=False, state=True),
        # a chat prompt of an odd length
        dict(name="prefill_chat", kind="prefill", batch=1, time=509, heads=6, vheads=6, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=False),
        # one long document continued from a state: a single chain of chunks per head
        dict(name="prefill_long", kind="prefill", batch=1, time=32749, heads=4, vheads=8, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=True),
        # one user's chat: a token at a time, the latency of a single call
        dict(name="step_one", kind="step", batch=1, time=1, heads=6, vheads=6, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=True),
        # a serving batch: every state is read and written once per token
        dict(name="step_batch", kind="step", batch=256, time=1, heads=6, vheads=12, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=True),
        # drafts of seven tokens checked for five sequences
        dict(name="burst_draft", kind="burst", batch=5, time=7, heads=4, vheads=8, kdim=128, vdim=128, dtype="bf16", docs=0, gate=True, state=True),
        # the output norm of a layer: every token normalised over the channels of each head, training
        dict(name="norm_heads", kind="norm", batch=32768, space=1, channels=768, groups=6, dtype="bf16", act="silu", train=True),
        # the same for the few tokens of a decoding step
        dict(name="norm_step", kind="norm", batch=7, space=1, channels=768, groups=6, dtype="bf16", act="silu", train=False),
        # statistics over whole sequences of an odd length, training
        dict(name="norm_sequence", kind="norm", batch=4, space=8191, channels=768, groups=32, dtype="bf16", act="silu", train=True),
        # FP32 without an activation, groups of an odd number of channels
        dict(name="norm_fp32", kind="norm", batch=3, space=1009, channels=510, groups=6, dtype="fp32", act="none", train=True),
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm; most of what comes out is odd or ragged
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("train", "train", "packed", "fp32", "prefill", "prefill", "step", "burst", "norm", "norm"))
    if kind == "norm":
        channels = rng.choice((8, 24, 96, 256, 510, 512, 768, 1000, 1024, 2048))
        groups = rng.choice([n for n in (1, 2, 4, 5, 6, 8, 12, 16, 32) if channels % n == 0])
        total = size(1, 24_000_000 // channels)
        space = 1 if rng.random() < 0.4 else max(1, total // size(1, min(64, total)))
        return dict(kind="norm", batch=max(1, total // space), space=space, channels=channels, groups=groups,
                    dtype=rng.choice(("bf16", "bf16", "fp32")), act=rng.choice(("silu", "silu", "none")), train=rng.random() < 0.7)
    heads = rng.choice((1, 2, 3, 4, 6))
    c = dict(kind=kind, batch=1, time=1, heads=heads, vheads=heads * rng.choice((1, 1, 2, 4)), kdim=rng.choice((64, 128, 128)),
             vdim=rng.choice((64, 128, 128)), dtype="bf16", docs=0, gate=rng.random() < 0.7, state=rng.random() < 0.6)
    rows = 160_000 // c["vheads"]
    if kind == "step":
        c.update(batch=size(1, 3000 // c["vheads"]), dtype=rng.choice(("bf16", "bf16", "fp32")), state=True)
    elif kind == "burst":
        c.update(batch=size(1, 500 // c["vheads"]), time=rng.randint(2, 24), dtype=rng.choice(("bf16", "bf16", "fp32")))
    elif kind == "packed":
        c.update(kind="train", time=size(64, min(rows, 30000)))
        c.update(docs=rng.randint(2, max(2, min(24, c["time"] // 16))))
    elif kind == "fp32":
        c.update(kind="train", dtype="fp32", batch=rng.randint(1, 3), time=size(3, 1500), state=True)
    else:
        c.update(time=size(1, min(rows, 32768)) if kind == "prefill" else size(2, 4096))
        c.update(batch=max(1, min(size(1, 16), rows // c["time"])))
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Document lengths of a packed case, of the sizes alone (seeded by them), some short, all together ``time`` tokens."""
    gen = torch.Generator().manual_seed(case["time"] * 31 + case["docs"])
    share = -torch.log(torch.rand(case["docs"], generator=gen, dtype=torch.float64).clamp_min(1e-9))
    cuts = (share.cumsum(0) / share.sum() * case["time"]).round().to(torch.int64)
    cuts[-1] = case["time"]
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts])


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        N, S, C = case["batch"], case["space"], case["channels"]
        shape = (N, C) if S == 1 else (N, S, C)
        offset = _randn(gen, C)
        s = dict(case=case, x=(_randn(gen, *shape) * 1.5 + offset).to(dt),
                 weight=1 + 0.2 * _randn(gen, C), bias=0.2 * _randn(gen, C), dy=_randn(gen, *shape, dtype=dt))
        s["leaves"] = ["x", "weight", "bias"] if case["train"] else []
    else:
        B, T, H, HV, K, V = (case[n] for n in ("batch", "time", "heads", "vheads", "kdim", "vdim"))
        N = case["docs"] or B
        s = dict(case=case, q=_randn(gen, B, T, H, K, dtype=dt), k=_randn(gen, B, T, H, K, dtype=dt), v=_randn(gen, B, T, HV, V, dtype=dt),
                 do=_randn(gen, B, T, HV, V, dtype=dt), A_log=None, dt_bias=None, cu=None, cu_cpu=None, h0=None, dht=None)
        A = torch.rand(HV, generator=gen, device="cuda") * 15 + 1
        step = torch.exp(torch.rand(HV, generator=gen, device="cuda") * math.log(100.0) + math.log(0.001))
        dt_bias = torch.log(torch.expm1(step))
        a, b = _randn(gen, B, T, HV), _randn(gen, B, T, HV)
        if case["gate"]:
            s.update(g=a.to(dt), beta=b.to(dt), A_log=A.log(), dt_bias=dt_bias)
        else:
            s.update(g=-A * torch.nn.functional.softplus(a + dt_bias), beta=b.sigmoid())
        if case["state"]:
            s["h0"] = _randn(gen, N, HV, K, V) * 0.3
            s["dht"] = _randn(gen, N, HV, K, V)
        if case["docs"]:
            s["cu_cpu"] = _lengths(case)
            s["cu"] = s["cu_cpu"].cuda()
        s["leaves"] = [n for n in ("q", "k", "v", "g", "beta", "A_log", "dt_bias", "h0") if s[n] is not None] if case["kind"] == "train" else []
        if case["kind"] == "step":
            s.update({n: s[n][:, 0].contiguous() for n in ("q", "k", "v", "g", "beta")})
    for n in s["leaves"]:
        s[n].requires_grad_()
    return s


# ---- the plain forms: FP32 in elementary operations, rounded once at the end ------------------------------------------

def _unit(x):
    return x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6)


def _prologue(s, wide):
    """q, k, v with one key head per value head, log decay and beta, in the type ``wide``."""
    rep = s["v"].shape[-2] // s["q"].shape[-2]
    q, k = (_unit(s[n].to(wide)).repeat_interleave(rep, -2) for n in ("q", "k"))
    g, beta = s["g"].to(wide), s["beta"].to(wide)
    if s["A_log"] is not None:
        x = g + s["dt_bias"].to(wide)
        g = -s["A_log"].to(wide).exp() * (x.clamp_min(0) + torch.log1p(torch.exp(-x.abs())))
        beta = 1 / (1 + torch.exp(-beta))
    return q, k, s["v"].to(wide), g, beta


def _spread(s, tensors):
    """Packed documents laid out as a batch [N, longest, ...] with rows of zeros behind each, and the places of their tokens."""
    cu = s["cu_cpu"]
    lens = cu[1:] - cu[:-1]
    doc = torch.repeat_interleave(torch.arange(len(lens)), lens)
    at = (doc.cuda(), (torch.arange(int(cu[-1])) - cu[:-1][doc]).cuda())
    return [x.new_zeros(len(lens), max(1, int(lens.max())), *x.shape[2:]).index_put(at, x[0]) for x in tensors], at


def _unit_lower_inverse(L):
    """(I + L)^-1 of strictly lower triangular L [.., C, C], by blocks of doubling size: the inverse of two neighbouring blocks
    is theirs, less their product around what joins them."""
    C = L.shape[-1]
    i = torch.arange(C, device=L.device)
    X = torch.eye(C, dtype=L.dtype, device=L.device).expand_as(L)
    for s in (1, 2, 4, 8, 16, 32):
        joins = (i[:, None] // (2 * s) == i[None] // (2 * s)) & (i[:, None] // s > i[None] // s)
        X = X - X @ torch.where(joins, L, 0.0) @ X
    return X


def _chunked(q, k, v, g, beta, scale, S):
    """The gated delta rule over chunks of 64 tokens, [B, T, H, .] and a state [B, H, K, V]."""
    B, T, H, V = v.shape
    n = -(-T // CHUNK)

    def cut(x):  # [B, H, n, 64, ...], rows of zeros behind the last token
        x = torch.cat([x, x.new_zeros(B, n * CHUNK - T, *x.shape[2:])], 1)
        return x.reshape(B, n, CHUNK, *x.shape[2:]).movedim(3, 1)

    q, k, v, g, beta = cut(q), cut(k), cut(v), cut(g), cut(beta)[..., None]
    G = g.double().cumsum(-1)
    i = torch.arange(CHUNK, device=q.device)
    lower = i[:, None] >= i[None]
    D = torch.where(lower, torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], 0.0)), 0.0).float()
    rise, fall, last = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None], G[..., -1].exp().float()
    A = scale * (q @ k.mT) * D
    Tm = _unit_lower_inverse(torch.where(i[:, None] > i[None], beta * (k @ k.mT) * D, 0.0)) * beta.mT
    U, W = Tm @ v, Tm @ (k * rise)
    o = []
    for c in range(n):
        Vn = U[:, :, c] - W[:, :, c] @ S
        o.append(scale * (q[:, :, c] * rise[:, :, c]) @ S + A[:, :, c] @ Vn)
        S = S * last[:, :, c, None, None] + (k[:, :, c] * fall[:, :, c]).mT @ Vn
    return torch.stack(o, 2).movedim(1, 3).reshape(B, n * CHUNK, H, V)[:, :T], S


def _recurrent(q, k, v, g, beta, scale, S, block=64):
    """The gated delta rule token by token, [B, T, H, .] and a state [B, H, K, V], as its definition says; a block's steps are
    taken again in the backward instead of kept."""
    def steps(S, q, k, v, g, beta):
        o = []
        for t in range(v.shape[1]):
            S = S * torch.exp(g[:, t])[..., None, None]
            e = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None] @ S).squeeze(-2))
            S = S + k[:, t, ..., None] * e[..., None, :]
            o.append(scale * (q[:, t, :, None] @ S).squeeze(-2))
        return torch.stack(o, 1), S

    out = []
    for t in range(0, v.shape[1], block):
        part = [x[:, t:t + block] for x in (q, k, v, g, beta)]
        o, S = checkpoint(steps, S, *part, use_reentrant=False) if torch.is_grad_enabled() else steps(S, *part)
        out.append(o)
    return torch.cat(out, 1), S


def _delta_rule(s, wide, rule):
    """Outputs [B, T, HV, V] and final states of a case, in the type ``wide``, by ``rule``."""
    xs = _prologue(s, wide)
    at = None
    if s["case"]["kind"] == "step":
        xs = [x[:, None] for x in xs]
    if s["cu"] is not None:
        xs, at = _spread(s, xs)
    q, k, v = xs[:3]
    S = q.new_zeros(v.shape[0], v.shape[2], q.shape[-1], v.shape[-1]) if s["h0"] is None else s["h0"].to(wide)
    o, S = rule(*xs, q.shape[-1] ** -0.5, S)
    if at is not None:
        o = o[at][None]
    return (o[:, 0] if s["case"]["kind"] == "step" else o), S


def _group_norm(s, wide):
    c = s["case"]
    x = s["x"].to(wide).reshape(c["batch"], c["space"], c["groups"], -1)
    mean = x.mean((1, 3), keepdim=True)
    var = (x - mean).square().mean((1, 3), keepdim=True)
    y = ((x - mean) / (var + NORM_EPS).sqrt()).reshape(s["x"].shape) * s["weight"].to(wide) + s["bias"].to(wide)
    return y / (1 + torch.exp(-y)) if c["act"] == "silu" else y


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _own(s):
    import openkimi_b200 as kimi

    c = s["case"]
    if c["kind"] == "norm":
        return kimi.group_norm(s["x"], c["groups"], s["weight"], s["bias"], eps=NORM_EPS, activation=None if c["act"] == "none" else c["act"]), None
    how = dict(A_log=s["A_log"], dt_bias=s["dt_bias"], use_qk_l2norm_in_kernel=True, use_gate_in_kernel=c["gate"], use_beta_sigmoid_in_kernel=c["gate"])
    args = [s[n] for n in ("q", "k", "v", "g", "beta")]
    if c["kind"] == "step":
        return kimi.recurrent_gated_delta_rule_step(*args, s["h0"], inplace=True, **how)
    if c["kind"] == "burst":
        return kimi.fused_recurrent_gated_delta_rule(*args, initial_state=s["h0"], output_final_state=True, **how)
    return kimi.chunk_gated_delta_rule(*args, initial_state=s["h0"], output_final_state=c["kind"] == "prefill" or c["state"],
                                       cu_seqlens=s["cu"], cu_seqlens_cpu=s["cu_cpu"], **how)


def _plain(s):
    c = s["case"]
    if c["kind"] == "norm":
        return _group_norm(s, torch.float32).to(s["x"].dtype), None
    o, S = _delta_rule(s, torch.float32, _recurrent if c["kind"] in ("step", "burst") else _chunked)
    if c["kind"] == "step":
        S = s["h0"].copy_(S)
    return o.to(s["v"].dtype), S if c["kind"] != "train" or c["state"] else None


def _pass(s, forward):
    """One pass: the outputs and, where the case trains, the gradients of everything that has one."""
    c = s["case"]
    with torch.set_grad_enabled(bool(s["leaves"])):
        o, S = forward(s)
    out = dict(o=o.detach())
    if S is not None:
        out["state"] = S.detach()
    if s["leaves"]:
        ends = [o] if c["kind"] == "norm" or not c["state"] else [o, S]
        given = [s["dy"]] if c["kind"] == "norm" else [s["do"], s["dht"]][:len(ends)]
        grads = torch.autograd.grad(ends, [s[n] for n in s["leaves"]], [d.to(e.dtype) for d, e in zip(given, ends)])
        out.update({"d" + n: d for n, d in zip(s["leaves"], grads)})
    return out


def run(state):
    return _pass(state, _own if own else _plain)


def exact(case, seed):
    """The same from the definitions in 64 bits: the recurrence a token at a time, the norm as it is written."""
    if case["kind"] == "norm":
        if case["batch"] * case["space"] * case["channels"] > 60_000_000:
            return None
        return _pass(_doubled(prepare(case, seed)), lambda s: (_group_norm(s, torch.float64), None))

    def forward(s):
        o, S = _delta_rule(s, torch.float64, _recurrent)
        return o, S if case["kind"] != "train" or case["state"] else None

    return _pass(_doubled(prepare(case, seed)), forward)


def _doubled(s):
    for n, x in s.items():
        if isinstance(x, torch.Tensor) and x.is_floating_point():
            s[n] = x.detach().double().requires_grad_(x.requires_grad)
    return s


def work(case):
    """Bytes: every input read and every output written once.  Operations: of the recurrence, a product with the state three times
    a token (prediction, update, output), and twice that for its gradients; of the norm, a few per value."""
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        n = case["batch"] * case["space"] * case["channels"]
        return {"bytes": (5 if case["train"] else 2) * n * es, "flops": (30 if case["train"] else 12) * n}
    B, T, H, HV, K, V = (case[n] for n in ("batch", "time", "heads", "vheads", "kdim", "vdim"))
    tokens, N = B * T, case["docs"] or B
    ge = es if case["gate"] else 4
    inputs = tokens * (2 * H * K * es + HV * V * es + 2 * HV * ge)
    states = N * HV * K * V * 4
    total, flops = inputs + tokens * HV * V * es, 6.0 * K * V * tokens * HV
    if case["kind"] == "train":
        total += 2 * inputs + tokens * HV * V * es + (4 * states if case["state"] else 0)
        flops *= 3
    else:
        total += states * (2 if case["state"] else 1)
    return {"bytes": total, "flops": flops}
