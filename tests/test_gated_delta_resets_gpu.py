"""Tokens whose decay is 0 in FP32 (a log decay below -104) cut a document off from what came before: nothing passes through them, so the
gradients of their gates are 0, not the rounding errors of sums that cancel, times A or the log decay."""
import pytest
import torch

from tests import gdr_testlib as lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
AT = [0, 17, 40, 41, 63, 64, 100, 149]


@pytest.mark.parametrize("K,V,dtype", [(128, 128, BF), (64, 128, BF), (64, 64, F32)])
@pytest.mark.parametrize("A_log,gate_input", [(2.0, 3000.0), (2.0, 60.0), (8.0, 4.0), (12.0, 4.0), (95.0, 4.0)])
def test_gates_that_cut(K, V, dtype, A_log, gate_input):
    """Two heads: one whose gate is wide open at some tokens, one that is slow all the time."""
    x = lib.make(2, 150, 1, 2, K, V, dtype, seed=31)
    x["A_log"] = torch.tensor([A_log, 0.5], device="cuda")
    if A_log > 2:
        x["dt_bias"][0] = 0.0
        x["g"][..., 0] = -60.0  # (softplus 1e-26: no decay, at the first three sizes of A)
    x["g"][:, AT, 0] = gate_input
    ref = lib.add_terms(lib.reference(x), x)
    got = lib.device_run(x)
    assert not got["dg"][:, AT, 0].any()
    lib.check(got, ref)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_log_decays_that_cut(dtype):
    x = lib.make(1, 150, 1, 2, 128, 128, dtype, gate=False, seed=32)
    for i, t in enumerate(AT):
        x["g"][:, t] = (-104.5, -200.0, -1000.0, -5000.0)[i % 4]
    ref = lib.reference(dict(x, g=x["g"].clamp_min(-1000)))
    got = lib.device_run(x)
    assert not got["dg"][:, AT].any()
    lib.check(got, ref)


def test_not_a_number_passes_a_cut():
    """A NaN in the token's own row is still one in its gradients."""
    x = lib.make(1, 150, 1, 1, 128, 128, BF, gate=False, seed=33)
    x["g"][:, 40] = -200.0
    x["do"][:, 100] = float("nan")
    assert torch.isnan(lib.device_run(x)["dg"][0, :64]).all()
