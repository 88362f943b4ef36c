"""The gated delta rule with one decay per head against its recurrence in 64 bits (bounds: gdr_testlib)."""
import pytest
import torch

from tests.gdr_testlib import add_terms, check, device_run, make, reference

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("K,V", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gate", [True, False])
def test_forward_and_backward(K, V, dtype, gate):
    x = make(2, 150, 2, 4, K, V, dtype, gate=gate, seed=K + V)
    check(device_run(x), add_terms(reference(x), x))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_lengths(T, dtype):
    x = make(1, T, 1, 1, 128, 128, dtype, seed=T)
    check(device_run(x), add_terms(reference(x), x))


@pytest.mark.parametrize("H,HV", [(1, 1), (1, 4), (3, 3), (2, 6), (1, 7)])
def test_head_layouts(H, HV):
    for dtype in (F32, BF):
        x = make(2, 70, H, HV, 64, 64, dtype, seed=HV)
        check(device_run(x), add_terms(reference(x), x))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_without_norm_state_or_final_gradient(dtype):
    x = make(1, 100, 2, 2, 64, 128, dtype, gate=False, h0=False, seed=5)
    x["k"] = (x["k"] / 8).to(dtype)
    ref = reference(x, l2=False, final=False, scale=0.3)
    check(device_run(x, l2=False, final=False, scale=0.3), ref)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_value_first_states(dtype):
    x = make(2, 90, 1, 2, 64, 128, dtype, seed=6)
    check(device_run(x, v_first=True), add_terms(reference(x), x))


@pytest.mark.parametrize("docs", [[0, 1, 1, 64, 130, 131, 260], [0, 200], [0, 63, 128]])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_packed_documents(docs, dtype):
    x = make(1, docs[-1], 2, 4, 128, 64, dtype, docs=docs, seed=7)
    check(device_run(x), add_terms(reference(x), x))


def test_rows_outside_the_documents_are_zero():
    x = make(1, 200, 1, 2, 64, 64, BF, docs=[3, 70, 150], seed=8)
    ref = add_terms(reference(x), x)
    got = device_run(x)
    check(got, ref)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert not got[n][:, :3].any() and not got[n][:, 150:].any(), n


@pytest.mark.parametrize("slow", [(1e-6, 1e-4), (0.5, 2.0), (20.0, 60.0)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_decays_from_none_to_complete(slow, dtype):
    x = make(1, 192, 1, 2, 128, 128, dtype, slow=slow, seed=9)
    check(device_run(x), add_terms(reference(x), x))


def test_decay_of_minus_infinity_clears_the_state():
    """-inf counts as -1000, whose exponential is 0 in FP32: the state restarts there, and nothing becomes a NaN."""
    x = make(1, 130, 1, 2, 64, 64, F32, gate=False, seed=10)
    y = dict(x, g=x["g"].clone())
    for t in (0, 40, 41, 64, 129):
        y["g"][:, t] = -float("inf")
        x["g"][:, t] = -1000.0
    ref = reference(x)
    check(device_run(y), ref)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_equal_keys(dtype):
    """All rows of k nearly parallel: the triangular system is as full as it gets."""
    x = make(1, 192, 1, 1, 128, 128, dtype, slow=(1e-5, 1e-4), keys_alike=20.0, seed=11)
    check(device_run(x), add_terms(reference(x), x))


def test_rows_of_zeros_and_beta_zero():
    x = make(1, 100, 1, 2, 64, 64, F32, gate=False, seed=12)
    x["k"][:, 10:20] = 0
    x["q"][:, 15:70] = 0
    x["beta"][:, 30:50] = 0
    ref = reference(x)
    got = device_run(x)
    # a row of zeros is divided by 1e-6: its gradient is 1e6 times the others' and is compared by itself
    for n, rows in (("dk", slice(10, 20)), ("dq", slice(15, 70))):
        a, b = got[n][:, rows].double(), ref[n][:, rows]
        assert float((a - b).norm()) <= 1.2e-5 * float(b.norm())
        got[n][:, rows] = 0
        ref[n][:, rows] = 0
    check(got, ref)


def test_gradients_against_differences():
    """Central differences of the 64-bit recurrence confirm its autograd on a small case, and the kernels agree with it."""
    x = make(1, 5, 1, 2, 64, 64, F32, gate=True, seed=13)
    ref = reference(x)
    loss = lambda y: float((lambda r: (r["o"] * x["do"].double()).sum() + (r["ht"] * x["dht"].double()).sum())(reference(y, grads=False)))  # noqa: E731
    gen = torch.Generator().manual_seed(1)
    for n in ("q", "k", "v", "g", "beta", "A_log", "dt_bias", "h0"):
        d = torch.randn(x[n].shape, generator=gen).double().cuda()
        h = 1e-5
        num = (loss(dict(x, **{n: x[n].double() + h * d})) - loss(dict(x, **{n: x[n].double() - h * d}))) / (2 * h)
        assert abs(num - float((ref["d" + n] * d).sum())) <= 1e-6 * (1 + abs(num)), n
    check(device_run(x), add_terms(ref, x))


def test_non_contiguous_inputs_and_other_types():
    x = make(2, 66, 2, 2, 64, 64, BF, gate=False, seed=14)
    ref = reference(x)
    y = dict(x)
    for n in ("q", "k", "v"):
        y[n] = x[n].transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.empty(x["g"].numel() + 1, device="cuda")
    y["g"] = buf[1:].view_as(x["g"]).copy_(x["g"])  # not on a 16-byte boundary
    check(device_run(y), ref)


def test_calls_are_repeatable_and_without_grad_the_same():
    x = make(2, 300, 2, 4, 128, 128, BF, seed=15)
    a, b = device_run(x), device_run(x)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    c = device_run(x, grads=False)
    assert torch.equal(a["o"], c["o"]) and torch.equal(a["ht"], c["ht"])


def test_state_carried_over_a_cut_of_the_sequence():
    from openkimi_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule, recurrent_gated_delta_rule_step

    x = make(2, 200, 2, 4, 128, 128, F32, seed=16)
    ref = reference(x, grads=False)
    how = dict(A_log=x["A_log"], dt_bias=x["dt_bias"], use_qk_l2norm_in_kernel=True, use_gate_in_kernel=True, use_beta_sigmoid_in_kernel=True)
    part = lambda a, b: [x[n][:, a:b] for n in ("q", "k", "v", "g", "beta")]  # noqa: E731
    o0, s = chunk_gated_delta_rule(*part(0, 130), initial_state=x["h0"], output_final_state=True, **how)
    o1, s = fused_recurrent_gated_delta_rule(*part(130, 170), initial_state=s, output_final_state=True, **how)
    o2, s = chunk_gated_delta_rule(*part(170, 190), initial_state=s, output_final_state=True, **how)
    outs = [o0, o1, o2]
    for t in range(190, 200):
        o, s2 = recurrent_gated_delta_rule_step(*(y[:, 0] for y in part(t, t + 1)), s, inplace=True, **how)
        assert s2.data_ptr() == s.data_ptr()
        outs.append(o[:, None])
    check(dict(o=torch.cat(outs, 1), ht=s), ref)


@pytest.mark.parametrize("K,V", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v_first", [False, True])
def test_recurrent_forms(K, V, dtype, v_first):
    from openkimi_b200 import fused_recurrent_gated_delta_rule

    for B, T, H, HV, gate in ((1, 1, 1, 1, True), (3, 19, 2, 4, True), (200, 2, 2, 6, False)):
        x = make(B, T, H, HV, K, V, dtype, gate=gate, seed=B + K + V)
        ref = reference(x, grads=False)
        h0 = x["h0"].transpose(-1, -2).contiguous() if v_first else x["h0"]
        o, s = fused_recurrent_gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=h0, output_final_state=True,
                                                A_log=x.get("A_log"), dt_bias=x.get("dt_bias"), use_qk_l2norm_in_kernel=True,
                                                use_gate_in_kernel=gate, use_beta_sigmoid_in_kernel=gate, state_v_first=v_first)
        check(dict(o=o, ht=s.transpose(-1, -2) if v_first else s), ref)


def test_empty_calls():
    from openkimi_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule

    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    h0 = torch.randn(2, 2, 64, 64, device="cuda", requires_grad=True)
    for fn in (chunk_gated_delta_rule, fused_recurrent_gated_delta_rule):
        o, s = fn(z(2, 0, 1, 64), z(2, 0, 1, 64), z(2, 0, 2, 64), z(2, 0, 2), z(2, 0, 2), initial_state=h0, output_final_state=True)
        assert o.shape == (2, 0, 2, 64) and torch.equal(s, h0)
    o, s = chunk_gated_delta_rule(z(2, 0, 1, 64), z(2, 0, 1, 64), z(2, 0, 2, 64), z(2, 0, 2), z(2, 0, 2), initial_state=h0, output_final_state=True)
    d, = torch.autograd.grad(s.sum() * 2, h0)
    assert torch.equal(d, torch.full_like(d, 2.0))
    cu = torch.tensor([0, 0, 0])
    o, s = chunk_gated_delta_rule(z(1, 5, 1, 64), z(1, 5, 1, 64), z(1, 5, 2, 64), z(1, 5, 2), z(1, 5, 2), initial_state=h0,
                                  output_final_state=True, cu_seqlens=cu.cuda(), cu_seqlens_cpu=cu)
    assert not o.any() and torch.equal(s, h0)


def test_other_streams_and_graphs():
    x = make(2, 140, 2, 4, 128, 128, BF, seed=17)
    want = device_run(x, grads=False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = device_run(x, grads=False)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got["o"], want["o"]) and torch.equal(got["ht"], want["ht"])
    from openkimi_b200 import chunk_gated_delta_rule

    args = [x[n].clone() for n in ("q", "k", "v", "g", "beta")]
    how = dict(A_log=x["A_log"], dt_bias=x["dt_bias"], use_qk_l2norm_in_kernel=True, use_gate_in_kernel=True,
               use_beta_sigmoid_in_kernel=True, initial_state=x["h0"], output_final_state=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, ht = chunk_gated_delta_rule(*args, **how)
    other = make(2, 140, 2, 4, 128, 128, BF, seed=18)
    for a, n in zip(args, ("q", "k", "v", "g", "beta")):
        a.copy_(other[n])
    graph.replay()
    again = chunk_gated_delta_rule(*args, **how)
    assert torch.equal(o, again[0]) and torch.equal(ht, again[1])
