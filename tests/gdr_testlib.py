"""Shared helpers of the gated delta rule's tests: inputs, the recurrence in 64 bits with autograd, and error bounds.

Bounds.  A computed operand is held to 2^-24 and a product sums at most K + 64 <= 192 terms in FP32, so a product is off by at most
192 2^-24 = 1.15e-5 of the sum of its terms' magnitudes; typical errors are the square root of that count smaller, so relative to the
2-norm of the result that figure bounds the few products that follow one another.  Single elements are held to four times that of
the largest one.  A BF16 result is rounded once more, by at most 2^-8 of itself.
"""
import torch

UNIT = 192 * 2.0 ** -24
FLOOR = 2.0 ** -126  # a decay below 2^-149 is 0 in FP32, and what it multiplies is a sum below 192 max^3 < 2^23 here
NAMES = ("q", "k", "v", "g", "beta", "A_log", "dt_bias", "h0")


def make(B, T, H, HV, K, V, dtype, *, gate=True, h0=True, docs=None, seed=0, slow=(0.001, 0.1), keys_alike=0.0, device="cuda"):
    """docs: document offsets (batch 1)."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    N = len(docs) - 1 if docs is not None else B
    x = dict(q=r(B, T, H, K).to(dtype), k=(r(B, T, H, K) + keys_alike * r(1, 1, H, K)).to(dtype), v=r(B, T, HV, V).to(dtype),
             do=r(B, T, HV, V).to(dtype), dht=r(N, HV, K, V))
    A = torch.rand(HV, generator=gen) * 15 + 1
    lo, hi = (torch.tensor(s).log() for s in slow)
    bias = torch.log(torch.expm1(torch.exp(torch.rand(HV, generator=gen) * (hi - lo) + lo)))
    a, b = r(B, T, HV), r(B, T, HV)
    if gate:
        x.update(g=a.to(dtype), beta=b.to(dtype), A_log=A.log(), dt_bias=bias)
    else:
        x.update(g=-A * torch.nn.functional.softplus(a + bias), beta=b.sigmoid())
    if h0:
        x["h0"] = 0.3 * r(N, HV, K, V)
    x = {n: t.to(device) for n, t in x.items()}
    x["docs"] = docs
    x["gate"] = gate
    return x


def reference(x, *, l2=True, final=True, scale=None, grads=True):
    """The recurrence a token at a time in 64 bits; outputs and gradients by name."""
    leaf = {n: x[n].detach().double().requires_grad_(grads) for n in NAMES if n in x}
    q, k, v, g, beta = (leaf[n] for n in ("q", "k", "v", "g", "beta"))
    B, T, HV, V = v.shape
    K = q.shape[-1]
    rep = HV // q.shape[2]
    unit = lambda t: t / t.norm(dim=-1, keepdim=True).clamp_min(1e-6) if l2 else t  # noqa: E731
    qs, ks = (unit(t).repeat_interleave(rep, 2) for t in (q, k))
    if x["gate"]:
        g = -leaf["A_log"].exp() * torch.nn.functional.softplus(g + leaf["dt_bias"])
        beta = beta.sigmoid()
    scale = K ** -0.5 if scale is None else scale
    o = torch.zeros_like(v)
    ends = []
    docs = x["docs"]
    spans = [(0, docs[i], docs[i + 1]) for i in range(len(docs) - 1)] if docs is not None else [(b, 0, T) for b in range(B)]
    outs = {}
    for n, (b, s, e) in enumerate(spans):
        S = leaf["h0"][n] if "h0" in leaf else torch.zeros(HV, K, V, dtype=torch.float64, device=v.device)
        rows = []
        for t in range(s, e):
            S = S * torch.exp(g[b, t])[:, None, None]
            err = beta[b, t][:, None] * (v[b, t] - torch.einsum("hk,hkv->hv", ks[b, t], S))
            S = S + ks[b, t][:, :, None] * err[:, None]
            rows.append(scale * torch.einsum("hk,hkv->hv", qs[b, t], S))
        ends.append(S)
        if rows:
            outs[n] = (b, s, e, torch.stack(rows))
    for b, s, e, rows in outs.values():
        idx = torch.arange(s, e, device=v.device)
        o = o.index_put((torch.full_like(idx, b), idx), rows)
    ht = torch.stack(ends)
    res = dict(o=o.detach(), ht=ht.detach())
    if grads:
        loss = (o * x["do"].double()).sum() + ((ht * x["dht"].double()).sum() if final else 0.0)
        names = list(leaf)
        d = torch.autograd.grad(loss, [leaf[n] for n in names], allow_unused=True)
        res.update({"d" + n: torch.zeros_like(leaf[n]) if t is None else t for n, t in zip(names, d)})
        res["g_terms"] = (res["dg"], x["g"])
    return res


def device_run(x, *, l2=True, final=True, scale=None, v_first=False, grads=True, **over):
    from openkimi_b200 import chunk_gated_delta_rule

    tr = (lambda t: t.transpose(-1, -2).contiguous()) if v_first else (lambda t: t)
    leaf = {n: (tr(x[n]) if n == "h0" else x[n]).detach().clone().requires_grad_(grads) for n in NAMES if n in x}
    docs = x["docs"]
    cu = None if docs is None else torch.tensor(docs)
    kw = dict(A_log=leaf.get("A_log"), dt_bias=leaf.get("dt_bias"), scale=scale, initial_state=leaf.get("h0"), output_final_state=final,
              use_qk_l2norm_in_kernel=l2, use_gate_in_kernel=x["gate"], use_beta_sigmoid_in_kernel=x["gate"], state_v_first=v_first,
              cu_seqlens=None if cu is None else cu.cuda(), cu_seqlens_cpu=cu)
    kw.update(over)
    o, ht = chunk_gated_delta_rule(*(leaf[n] for n in ("q", "k", "v", "g", "beta")), **kw)
    res = dict(o=o.detach())
    if final:
        res["ht"] = tr(ht.detach())
    if grads:
        ends, given = ([o, ht], [x["do"], tr(x["dht"])]) if final else ([o], [x["do"]])
        d = torch.autograd.grad(ends, list(leaf.values()), given)
        res.update({"d" + n: (tr(t) if n == "h0" else t) for n, t in zip(leaf, d)})
    return res


def check(got, ref, names=None):
    bad = []
    for n, y in got.items():
        if names is not None and n not in names:
            continue
        r = ref[n].double()
        y64 = y.double()
        if not torch.isfinite(y64).all():
            bad.append(f"{n}: not finite")
            continue
        if not r.numel():
            continue
        err, big, norm = (y64 - r).abs(), r.abs().max(), r.norm()
        if n in ("dA_log", "ddt_bias"):
            # sums over all tokens with cancellation: relative to the sum of their terms' magnitudes
            lim = UNIT * ref[n + "_terms"] + 1e-30
            if not (err <= lim).all():
                bad.append(f"{n}: {float((err / lim).max()):.2f} of its bound")
            continue
        round_to = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24
        lim = round_to * r.abs() + 4 * UNIT * big + FLOOR
        l2 = max(0.0, float(err.norm()) - FLOOR * r.numel() ** 0.5) / max(float(norm), 1e-300)
        if not (err <= lim).all() or l2 > round_to + UNIT:
            bad.append(f"{n}: rel l2 {l2:.2e}, worst element {float((err / lim.clamp_min(1e-300)).max()):.2f} of its bound")
    assert not bad, "; ".join(bad)


def add_terms(ref, x):
    """Sums of the magnitudes that dA_log and ddt_bias are made of."""
    if x["gate"]:
        a = x["g"].double() + x["dt_bias"].double()
        A = x["A_log"].double().exp()
        dlog = ref["dg"] / (-A * a.sigmoid()).clamp(max=-1e-300)
        ref["dA_log_terms"] = (dlog * A * torch.nn.functional.softplus(a)).abs().sum((0, 1))
        ref["ddt_bias_terms"] = ref["dg"].abs().sum((0, 1))
    return ref
