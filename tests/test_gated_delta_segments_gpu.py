"""Long sequences on few heads: the walks cut into segments, against the recurrence in 64 bits and against themselves."""
import pytest
import torch

from tests.gdr_testlib import add_terms, check, device_run, make, reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("T,H,HV", [(256, 1, 1), (641, 1, 2), (1500, 2, 2), (4099, 1, 1)])
def test_long_sequences(T, H, HV):
    x = make(1, T, H, HV, 128, 128, BF, seed=T, slow=(1e-4, 0.05))
    check(device_run(x), add_terms(reference(x), x))


@pytest.mark.parametrize("docs", [[0, 700, 701, 701, 1400], [0, 64, 1300], [5, 1000, 1300]])
def test_uneven_documents(docs):
    """Segments of the longest document: shorter ones end in the middle of theirs, and the last segments are empty."""
    x = make(1, docs[-1], 1, 2, 128, 128, BF, docs=docs, seed=docs[-1], slow=(1e-4, 0.05))
    check(device_run(x), add_terms(reference(x), x))


def test_value_first_states_and_no_initial_state():
    x = make(1, 900, 1, 1, 128, 128, BF, seed=3, slow=(1e-5, 1e-3))
    check(device_run(x, v_first=True), add_terms(reference(x), x))
    x = make(1, 900, 1, 1, 128, 128, BF, seed=4, h0=False, gate=False)
    check(device_run(x, final=False), reference(x, final=False))


def test_prompt_of_a_long_document_continues():
    """The whole document at once, and cut in two calls with the state handed over: FP32 states, so close but not the same bits."""
    from openkimi_b200 import chunk_gated_delta_rule

    x = make(1, 2048, 1, 1, 128, 128, BF, seed=5, slow=(1e-4, 1e-2))
    how = dict(A_log=x["A_log"], dt_bias=x["dt_bias"], use_qk_l2norm_in_kernel=True, use_gate_in_kernel=True, use_beta_sigmoid_in_kernel=True,
               output_final_state=True)
    part = lambda a, b: [x[n][:, a:b] for n in ("q", "k", "v", "g", "beta")]  # noqa: E731
    o, s = chunk_gated_delta_rule(*part(0, 2048), initial_state=x["h0"], **how)
    o1, s1 = chunk_gated_delta_rule(*part(0, 1000), initial_state=x["h0"], **how)
    o2, s2 = chunk_gated_delta_rule(*part(1000, 2048), initial_state=s1, **how)
    assert float((s2 - s).norm() / s.norm()) < 2e-5
    assert float((torch.cat([o1, o2], 1).float() - o.float()).abs().max()) <= 2.0 ** -7 * float(o.float().abs().max())


def test_batches_around_the_line():
    """Numbers of walks on both sides of where segments stop paying give the same outputs to rounding."""
    a = make(2, 1024, 1, 1, 128, 128, BF, seed=6)
    one = {n: (t[:1] if isinstance(t, torch.Tensor) and t.dim() > 2 else t) for n, t in a.items()}
    many = {n: (t[:1].expand(80, *t.shape[1:]).contiguous() if isinstance(t, torch.Tensor) and t.dim() > 2 else t) for n, t in a.items()}
    r1, r2 = device_run(one), device_run(many)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        p, q = r1[n].float(), r2[n][:1].float()
        assert float((p - q).abs().max()) <= 2.0 ** -7 * float(p.abs().max()), n
    for n in ("ht", "dh0"):
        assert float((r1[n] - r2[n][:1]).norm() / r1[n].norm()) < 2e-5, n
