"""More of the sizes and values at which the gated delta rule and group norm go other ways through their kernels."""
import pytest
import torch

from tests import gdr_testlib as lib
from tests import test_group_norm_gpu as norm

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


# one and two elements an access with many of them a lane; groups of more than 1024 channels row by row, few and many; more groups than
# 48 KB of shared memory hold
@pytest.mark.parametrize("shape,G", [((7, 510), 1), ((7, 510), 2), ((5, 1022), 1), ((5, 1023), 1), ((300, 510), 2), ((5, 2048), 1), ((5000, 2048), 1),
                                     ((9, 4100), 2), ((1, 5001), 1), ((2, 3, 8192), 8192), ((2, 3, 8192), 4096), ((2, 3, 2, 510), 2)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", [True, False])
def test_norm_against_the_definition(shape, G, dtype, act):
    norm.test_against_the_definition(shape, G, dtype, act)


@pytest.mark.parametrize("K,V", [(64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("T,docs", [(1500, None), (1900, [0, 700, 701, 1900])])
def test_long_sequences_of_narrow_heads(K, V, T, docs):
    x = lib.make(1, T, 1, 2, K, V, BF, docs=docs, seed=K + V, slow=(1e-4, 0.05))
    lib.check(lib.device_run(x), lib.add_terms(lib.reference(x), x))


@pytest.mark.parametrize("K,V,dtype", [(128, 128, BF), (64, 64, F32)])
@pytest.mark.parametrize("name", ["g", "beta"])
@pytest.mark.parametrize("gate", [True, False])
def test_not_a_number_in_a_gate(K, V, dtype, name, gate):
    """It stays in its document and value head, and for dq, dk in the heads' key head; what follows it in the document is one too."""
    docs = [0, 90, 220, 400]
    x = lib.make(1, 420, 2, 4, K, V, dtype, docs=docs, gate=gate, seed=3)
    want = lib.device_run(x)
    x[name] = x[name].clone()
    x[name][0, 100, 2] = float("nan")
    x[name][0, 405:] = float("nan")  # rows of no document
    got = lib.device_run(x)
    assert torch.isnan(got["o"][0, 100:220, 2]).all() and torch.isnan(got["ht"][1, 2]).all()
    for n in ("o", "dv", "dg", "dbeta"):
        a, b = got[n], want[n]
        assert torch.equal(a[:, :90], b[:, :90]) and torch.equal(a[:, 220:], b[:, 220:]) and torch.equal(a[:, :, [0, 1, 3]], b[:, :, [0, 1, 3]]), n
    for n in ("ht", "dh0"):
        a, b = got[n], want[n]
        assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, [0, 1, 3]], b[1, [0, 1, 3]]), n
    for n in ("dq", "dk"):
        a, b = got[n], want[n]
        assert torch.equal(a[:, :90], b[:, :90]) and torch.equal(a[:, 220:], b[:, 220:]) and torch.equal(a[:, :, 0], b[:, :, 0]), n


@pytest.mark.parametrize("kind", [dict(H=2, HV=4, K=128, V=128, dtype=BF), dict(H=2, HV=4, K=64, V=128, dtype=F32)])
def test_passes_repeat_whatever_lies_in_memory(kind):
    """Workspaces come from memory that held other things: the bits are the same over zeros, NaN and large numbers."""
    x = lib.make(1, 900, docs=[0, 130, 131, 900], seed=4, **kind)
    want = lib.device_run(x)
    for byte in (0x00, 0xFF, 0x7F):
        junk = [torch.full((n,), byte, dtype=torch.uint8, device="cuda") for n in (1 << 28, 1 << 26, 1 << 24, 1 << 20, 1 << 16) for _ in range(3)]
        del junk
        got = lib.device_run(x)
        assert all(torch.equal(got[n], want[n]) for n in want), byte
