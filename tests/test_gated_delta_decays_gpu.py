"""Gradients of the gate where tokens reach back little: dA_log and ddt_bias of every head by itself, against the recurrence in 64 bits and
relative to the sum of their terms' magnitudes (gdr_testlib).  The gradient of a log decay is a running sum in which a chunk's pairs of
tokens cancel; what is left of it must not be the rounding of larger pairs."""
import pytest
import torch

from tests import gdr_testlib as lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
KINDS = [(128, 128, BF), (128, 64, BF), (64, 64, F32), (128, 128, F32)]


@pytest.mark.parametrize("K,V,dtype", KINDS)
@pytest.mark.parametrize("T,docs,h0", [(200, None, True), (465, [25, 275, 379, 416], False), (159, [0, 126, 149, 159], True)])
def test_decays_of_a_few_tokens(K, V, dtype, T, docs, h0):
    """Log decays of -0.3 to -32."""
    x = lib.make(1, T, 3, 15, K, V, dtype, docs=docs, h0=h0, slow=(0.3, 2.0), keys_alike=5.0, seed=158715)
    lib.check(lib.device_run(x), lib.add_terms(lib.reference(x), x))


@pytest.mark.parametrize("K,V,dtype", KINDS)
@pytest.mark.parametrize("T,docs", [(1, None), (8, None), (50, [0, 34, 47, 50]), (130, None)])
def test_decays_of_one_token(K, V, dtype, T, docs):
    """Log decays of -1 to -128: gradients down to e^-100 of the others' in the chunk."""
    x = lib.make(1 if docs else 2, T, 1, 3, K, V, dtype, docs=docs, slow=(1.0, 8.0), seed=T)
    lib.check(lib.device_run(x), lib.add_terms(lib.reference(x), x))
