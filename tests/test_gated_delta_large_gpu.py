"""Offsets past 32 bits: states, records and activations of more than 2^31 elements, compared with calls on their last part; and values at
the ends of their range in the tensor-core kernels."""
import pytest
import torch

from tests import gdr_testlib as lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def free_memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("v_first", [False, True])
def test_more_states_than_32_bits_count(v_first):
    from openkimi_b200 import recurrent_gated_delta_rule_step

    N, HV = 17000, 8  # 2.2e9 state elements
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    q, k, v, g, beta = r(N, 4, 128), r(N, 4, 128), r(N, HV, 128), -r(N, HV).abs(), r(N, HV).sigmoid()
    state = r(N, HV, 128, 128)
    tail = slice(N - 40, N)
    want = recurrent_gated_delta_rule_step(*(t[tail].contiguous() for t in (q, k, v, g, beta, state)), use_qk_l2norm_in_kernel=True, state_v_first=v_first)
    o, s = recurrent_gated_delta_rule_step(q, k, v, g, beta, state, use_qk_l2norm_in_kernel=True, state_v_first=v_first, inplace=True)
    assert s.data_ptr() == state.data_ptr()
    # (the columns a warp holds depend on the number of states, and with them the order of a sum over 128 channels)
    for a, b in ((o[tail], want[0]), (s[tail], want[1])):
        assert float((a - b).abs().max()) <= 4 * lib.UNIT * float(b.abs().max())


def test_more_records_than_32_bits_count():
    """137 500 units of 64 tokens: 2.25e9 elements of kept states.  The last tokens, from the state that the others leave."""
    from openkimi_b200 import chunk_gated_delta_rule

    T, HV, cut = 1_100_000, 8, 1_099_008
    gen = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=BF)  # noqa: E731
    args = [r(1, T, 1, 128), r(1, T, 1, 128), r(1, T, HV, 128), -r(1, T, HV).float().abs() * 0.02, r(1, T, HV).float().sigmoid()]
    do = r(1, T, HV, 128)
    leaf = [t.requires_grad_() for t in args]
    o, ht = chunk_gated_delta_rule(*leaf, use_qk_l2norm_in_kernel=True, output_final_state=True)
    d = torch.autograd.grad([o, ht], leaf, [do, torch.ones_like(ht)])
    with torch.no_grad():
        _, mid = chunk_gated_delta_rule(*(t[:, :cut] for t in args), use_qk_l2norm_in_kernel=True, output_final_state=True)
    tail = [t.detach()[:, cut:].contiguous().requires_grad_() for t in args]
    o2, ht2 = chunk_gated_delta_rule(*tail, use_qk_l2norm_in_kernel=True, initial_state=mid, output_final_state=True)
    d2 = torch.autograd.grad([o2, ht2], tail, [do[:, cut:].contiguous(), torch.ones_like(ht2)])
    for a, b in zip((o[:, cut:], ht, *(t[:, cut:] for t in d)), (o2, ht2, *d2)):
        a, b = a.detach().double(), b.detach().double()
        step = 2.0 ** -7 if o.dtype == BF else 0.0  # both sides are rounded to BF16
        assert torch.isfinite(a).all() and ((a - b).abs() <= step * b.abs() + 8 * lib.UNIT * b.abs().max()).all()


def test_more_activations_than_32_bits_count():
    from openkimi_b200 import group_norm

    gen = torch.Generator(device="cuda").manual_seed(3)
    w, b = torch.rand(768, generator=gen, device="cuda"), torch.randn(768, generator=gen, device="cuda")
    x = torch.empty(2_900_000, 768, dtype=BF, device="cuda").normal_(generator=gen)  # 2.2e9 elements
    x.requires_grad_()
    y = group_norm(x, 6, w, b, activation="silu")
    (dx,) = torch.autograd.grad(y, x, y.detach())
    end = x.detach()[-50:].clone().requires_grad_()
    y2 = group_norm(end, 6, w, b, activation="silu")
    (dx2,) = torch.autograd.grad(y2, end, y2.detach())
    assert torch.equal(y[-50:], y2) and torch.equal(dx[-50:], dx2)
    x = x.detach().view(4, 725_000, 768)
    y = group_norm(x, 32, w, b, activation="silu")
    y2 = group_norm(x[3:].contiguous(), 32, w, b, activation="silu")
    # statistics from other slices: FP32 sums of 725 000 x 24 values, then two roundings to BF16
    a, c = y[3].float(), y2[0].float()
    assert ((a - c).abs() <= 2.0 ** -7 * c.abs() + 1e-4).all()


@pytest.mark.parametrize("T", [130, 900])
def test_resets_in_the_tensor_core_kernels(T):
    """Log decays of -inf (which count as -1000) and of -200 inside chunks, at their ends and in long, segmented sequences."""
    x = lib.make(1, T, 1, 2, 128, 128, BF, gate=False, seed=21)
    y = dict(x, g=x["g"].clone())
    for t in (0, 40, 41, 63, 64, 100, 128, T - 1):
        y["g"][:, t] = -float("inf")
        x["g"][:, t] = -1000.0
    for z in (x, y):
        z["g"][:, 70:75] = -200.0
    lib.check(lib.device_run(y), lib.reference(x))


@pytest.mark.parametrize("size", [1e-18, 1e15])
def test_sizes_of_rows_under_the_norm(size):
    """Rows far from length 1: squares of 1e15 are within FP32, and a row of 1e-18 is divided by 1e-6, whatever its length."""
    x = lib.make(1, 100, 1, 2, 128, 128, BF, gate=False, seed=22)
    x["q"], x["k"] = x["q"] * size, x["k"] * size
    ref = lib.reference(x)
    lib.check(lib.device_run(x), ref, names=("o", "ht", "dv", "dg", "dbeta", "dh0", "dq", "dk"))


def test_state_in_place_of_any_alignment():
    from openkimi_b200 import recurrent_gated_delta_rule_step

    gen = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    q, k, v, g, beta, state = r(3, 2, 64), r(3, 2, 64), r(3, 4, 128), -r(3, 4).abs(), r(3, 4).sigmoid(), r(3, 4, 64, 128)
    want = recurrent_gated_delta_rule_step(q, k, v, g, beta, state)
    for place in (torch.empty(state.numel() + 1, device="cuda")[1:].view_as(state), torch.empty(3, 4, 128, 64, device="cuda").transpose(2, 3),
                  torch.empty(5, 4, 64, 128, device="cuda")[::2]):
        place.copy_(state)
        o, s = recurrent_gated_delta_rule_step(q, k, v, g, beta, place, inplace=True)
        assert torch.equal(o, want[0]) and torch.equal(place, want[1]) and s.data_ptr() == place.data_ptr()
