"""Shared key heads: the value heads' shares of dq and dk are left before the gradient of the L2 norm, which is taken once, of their sum."""
import pytest
import torch

from tests.gdr_testlib import UNIT, make
from tests.test_gated_delta_transitions_gpu import Call

pytestmark = pytest.mark.gpu


def test_shares_are_summed_before_the_norm():
    docs, HV, K = [0, 64, 128, 192], 3, 128
    x = make(1, 192, 1, HV, K, 128, torch.bfloat16, docs=docs, gate=False, seed=1)
    call = Call(x, docs, False)
    got = call.run()
    n = 3 * HV  # units: (chunk, value head)
    at = n * (K * 128 + 64 * 128) * 4 + -(-n * 8 // 256) * 256  # behind dS, Y and the gate's shares
    shares = call.scratch[at:at + n * 2 * 64 * K * 4].view(torch.float32).view(3, HV, 2, 64, K).double()
    for i, name in enumerate(("q", "k")):
        rows = x[name].double().view(3, 64, K)
        along = (shares[:, :, i] * rows[:, None]).sum(-1) / (shares[:, :, i].norm(dim=-1) * rows.norm(dim=-1)[:, None])
        assert float(along.abs().mean()) > 0.02, name
        total = shares[:, :, i].sum(1)
        want = total - rows * (rows * total).sum(-1, keepdim=True) / rows.square().sum(-1, keepdim=True)
        d = got["grad_" + name].double().view(3, 64, K)
        assert ((d - want).abs() <= 2.0 ** -8 * want.abs() + 4 * UNIT * want.abs().max()).all(), name
