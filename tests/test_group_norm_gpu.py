"""Group normalisation with an activation against its definition in 64 bits.

Bounds: an output is rounded once (2^-8 of itself in BF16, 2^-24 in FP32) and computed in FP32 from statistics in 64 bits or from sums
of at most 1024 values: 1024 2^-24 of the largest magnitudes covers every sum here, 16 2^-24 the elementwise arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def reference(x, G, w, b, eps, act, dy):
    leaf = [t.detach().double().requires_grad_() if t is not None else None for t in (x, w, b)]
    xd, wd, bd = leaf
    N, Ch = x.shape[0], x.shape[-1]
    v = xd.reshape(N, -1, G, Ch // G)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    z = ((v - mean) / (var + eps).sqrt()).reshape(x.shape)
    if wd is not None:
        z = z * wd
    if bd is not None:
        z = z + bd
    y = z * z.sigmoid() if act else z
    have = [t for t in leaf if t is not None]
    return [y.detach(), *torch.autograd.grad(y, have, dy.double())]


def run(x, G, w, b, eps, act, dy):
    from openkimi_b200 import group_norm

    leaf = [t.detach().clone().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaf)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = group_norm(args[0], G, args[1], args[2], eps=eps, activation="silu" if act else None)
    return [y.detach(), *torch.autograd.grad(y, leaf, dy)]


def check(got, ref, terms=None):
    for i, (a, r) in enumerate(zip(got, ref)):
        assert a.shape == r.shape and torch.isfinite(a).all()
        step = 2.0 ** -8 if a.dtype == BF else 2.0 ** -24
        big = r.abs().max() if i < 2 else terms
        lim = step * r.abs() + 1024 * 2.0 ** -24 * big
        err = (a.double() - r).abs()
        assert (err <= lim).all(), (i, float((err / lim.clamp_min(1e-300)).max()))


SHAPES = [((1, 8), 8), ((1, 12), 1), ((7, 768), 6), ((333, 768), 6), ((5, 510), 6), ((40, 2048), 1), ((9, 1024), 1), ((3, 1000), 8), ((1000, 24), 2),
          ((2, 1, 64), 4), ((2, 33, 768), 32), ((3, 101, 510), 6), ((1, 5, 7, 96), 3), ((2, 700, 8), 8), ((600, 3, 32), 1), ((1, 4097, 256), 2),
          ((2, 3, 4100), 4)]


@pytest.mark.parametrize("shape,G", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", [True, False])
def test_against_the_definition(shape, G, dtype, act):
    gen = torch.Generator().manual_seed(sum(shape) + G)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    Ch = shape[-1]
    x, dy = (r(*shape) * 1.5 + r(Ch)).to(dtype).cuda(), r(*shape).to(dtype).cuda()
    w, b = (1 + 0.2 * r(Ch)).cuda(), (0.2 * r(Ch)).cuda()
    ref = reference(x, G, w, b, 1e-5, act, dy)
    check(run(x, G, w, b, 1e-5, act, dy), ref, terms=4 * dy.double().abs().reshape(-1, Ch).sum(0).max())


@pytest.mark.parametrize("shape", [(30, 96), (2, 50, 96)])
def test_without_weight_or_bias_and_no_grad(shape):
    from openkimi_b200 import group_norm

    gen = torch.Generator().manual_seed(1)
    x, dy = torch.randn(*shape, generator=gen).cuda(), torch.randn(*shape, generator=gen).cuda()
    w = torch.rand(96, generator=gen).cuda()
    top = 4 * dy.double().abs().reshape(-1, 96).sum(0).max()
    for ww, bb in ((None, None), (w, None), (None, w)):
        got = run(x, 4, ww, bb, 1e-3, True, dy)
        check(got, reference(x, 4, ww, bb, 1e-3, True, dy), terms=top)
        assert torch.equal(got[0], group_norm(x, 4, ww, bb, eps=1e-3, activation="silu"))


@pytest.mark.parametrize("shape", [(16, 256), (2, 300, 256)])
def test_offsets_far_above_the_spread(shape):
    """A mean of 1000 times the spread: the variance comes from deviations, not from a difference of squares.  FP32 holds x to 2^-24
    of 1000, which is the input; the bound is that of the statistics."""
    gen = torch.Generator().manual_seed(2)
    x, dy = (1000 + torch.randn(*shape, generator=gen)).cuda(), torch.randn(*shape, generator=gen).cuda()
    got, ref = run(x, 8, None, None, 1e-5, False, dy), reference(x, 8, None, None, 1e-5, False, dy)
    # mean and x - mean are rounded to 2^-24 of 1000, against a spread of 1
    for a, r in zip(got, ref):
        assert float((a.double() - r).abs().max()) <= 4 * 1000 * 2.0 ** -24 * float(r.abs().max())


@pytest.mark.parametrize("shape,G", [((7, 768), 6), ((333, 96), 3), ((2, 33, 96), 3)])
def test_without_an_epsilon(shape, G):
    """Lanes that have no row in a turn add nothing to the parameters' gradients, where 1 / sqrt(0) would be infinite."""
    gen = torch.Generator().manual_seed(6)
    x, dy = torch.randn(*shape, generator=gen).cuda(), torch.randn(*shape, generator=gen).cuda()
    w, b = torch.rand(shape[-1], generator=gen).cuda(), torch.randn(shape[-1], generator=gen).cuda()
    check(run(x, G, w, b, 0.0, True, dy), reference(x, G, w, b, 0.0, True, dy), terms=4 * dy.double().abs().reshape(-1, shape[-1]).sum(0).max())


def test_constant_input_and_large_values():
    from openkimi_b200 import group_norm

    for shape in ((4, 32), (2, 20, 32)):
        x = torch.full(shape, 3.0, device="cuda")
        b = torch.randn(32, device="cuda")
        assert torch.equal(group_norm(x, 4, None, b), b.expand(shape))
        y = group_norm(torch.randn(*shape, device="cuda") * 1e18, 4, None, torch.full((32,), -200.0, device="cuda"), activation="silu")
        assert torch.isfinite(y).all() and float(y.abs().max()) < 1e-30


def test_nan_stays_in_its_group():
    from openkimi_b200 import group_norm

    for shape in ((6, 32), (6, 40, 32)):
        x = torch.randn(*shape, device="cuda")
        want = group_norm(x, 4)
        x.view(6, -1, 32)[2, 0, 9] = float("nan")
        y = group_norm(x, 4)
        hit = torch.zeros_like(y, dtype=torch.bool).view(6, -1, 32)
        hit[2, :, 8:16] = True
        assert torch.isnan(y[hit.view(shape)]).all() and torch.equal(y[~hit.view(shape)], want[~hit.view(shape)])


def test_strides_alignment_types_and_repeatability():
    from openkimi_b200 import group_norm

    gen = torch.Generator().manual_seed(3)
    x = torch.randn(3, 40, 64, generator=gen).to(BF).cuda()
    want = group_norm(x, 4, activation="silu")
    assert torch.equal(group_norm(x.transpose(1, 2).contiguous().transpose(1, 2), 4, activation="silu"), want)
    buf = torch.empty(x.numel() + 1, dtype=BF, device="cuda")
    assert torch.equal(group_norm(buf[1:].view_as(x).copy_(x), 4, activation="silu"), want)
    w = torch.ones(64, dtype=BF, device="cuda", requires_grad=True)
    a = torch.autograd.grad(group_norm(x, 4, w).float().square().sum(), w)[0]
    b = torch.autograd.grad(group_norm(x, 4, w).float().square().sum(), w)[0]
    assert a.dtype == BF and torch.equal(a, b)
    assert group_norm(torch.empty(0, 64, device="cuda"), 4).shape == (0, 64)
    assert group_norm(torch.empty(3, 0, 64, device="cuda"), 4).shape == (3, 0, 64)


def test_refusals():
    from openkimi_b200 import group_norm

    x = torch.zeros(4, 12, device="cuda")
    with pytest.raises(ValueError):
        group_norm(x, 5)
    with pytest.raises(ValueError):
        group_norm(x, 3, torch.ones(11, device="cuda"))
    with pytest.raises(ValueError):
        group_norm(x[0], 3)
    with pytest.raises(ValueError):
        group_norm(x, 3, eps=-1.0)
    with pytest.raises(TypeError):
        group_norm(x.half(), 3)
    with pytest.raises(RuntimeError):
        group_norm(x, 3, torch.ones(12))


def test_layer_of_gated_delta_rule_and_norm():
    """The operators as a layer runs them: rule, norm over each head's channels with its activation, gradients through both."""
    from openkimi_b200 import FusedGroupNorm, chunk_gated_delta_rule
    from tests.gdr_testlib import make, reference as rule

    x = make(2, 100, 2, 4, 64, 64, F32, seed=4)
    norm = FusedGroupNorm(4, 256, activation="silu").cuda()
    leaf = {n: x[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "beta", "A_log", "dt_bias")}
    o, _ = chunk_gated_delta_rule(leaf["q"], leaf["k"], leaf["v"], leaf["g"], leaf["beta"], A_log=leaf["A_log"], dt_bias=leaf["dt_bias"],
                                  initial_state=x["h0"], use_qk_l2norm_in_kernel=True, use_gate_in_kernel=True, use_beta_sigmoid_in_kernel=True)
    y = norm(o.reshape(200, 256))
    dy = torch.randn(200, 256, generator=torch.Generator().manual_seed(5)).cuda()
    got = torch.autograd.grad(y, [*leaf.values(), norm.weight, norm.bias], dy)
    ref_o = rule(x, grads=False)["o"].reshape(200, 256)
    ref = reference(ref_o, 4, norm.weight, norm.bias, 1e-5, True, dy)
    assert float((y.double() - ref[0]).norm() / ref[0].norm()) < 5e-5
    want = rule(dict(x, do=ref[1].reshape(x["do"].shape)), final=False)
    for n, g in zip(leaf, got):
        r = want["d" + n]
        assert float((g.double() - r).norm()) <= 2e-4 * float(r.norm()), n  # (the norm divides by a spread well below 1)
    assert float((got[-2].double() - ref[2]).norm()) <= 2e-4 * float(ref[2].norm())
    assert float((got[-1].double() - ref[3]).norm()) <= 2e-4 * float(ref[3].norm())
