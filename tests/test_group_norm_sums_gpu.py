"""Group normalisation where sums are long: many rows per thread, first rows far from the others, constant gradients, whose sums have
rounding errors of one sign.

Bounds: an FP32 sum adds at most 1024 rows, so its relative error is at most 1024 2^-24 = 6.1e-5 whatever the signs; what joins sums is in 64
bits.  Statistics are sums of squares about the middle of the rows, so the same holds for the variance, and half of it for 1 / sqrt.
`check` (of the tests of the definition) has that figure."""
import pytest
import torch

from tests.test_group_norm_gpu import check, reference, run

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def free_memory():
    yield
    torch.cuda.empty_cache()


def compare(x, G, dy, samples):
    got = run(x, G, None, None, 1e-8, False, dy)
    at = torch.tensor(samples, device="cuda")
    check([t[at] for t in got], reference(x[at], G, None, None, 1e-8, False, dy[at]))


# one slice a sample and a row as wide as the CTA; the same with narrow rows; more slices in the first pass than in the second; few samples
SHAPES = [((223, 9001, 386), 1), ((300, 20001, 8), 2), ((1, 400_000, 386), 2), ((3, 150_000, 8), 2), ((2, 9, 64), 4), ((1, 3000, 24), 3)]


@pytest.mark.parametrize("shape,G", SHAPES)
def test_first_rows_far_from_the_others(shape, G):
    """All but the first row of a sample lie within 0.001 of 1; the first is 0."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(*shape, generator=gen, device="cuda").mul_(1e-3).add_(1)
    x[:, 0] = 0
    dy = torch.randn(*shape, generator=gen, device="cuda")
    compare(x, G, dy, [0, shape[0] - 1])


@pytest.mark.parametrize("row", [0, 5, 700, 2999])
@pytest.mark.parametrize("far", [-30.0, 3000.0])
def test_a_row_far_from_the_others(row, far):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, dy = torch.randn(230, 3000, 200, generator=gen, device="cuda"), torch.randn(230, 3000, 200, generator=gen, device="cuda")
    x[:, row] += far
    compare(x, 4, dy, [0, 229])


def test_constant_gradients_of_long_samples():
    x = torch.randn(149, 60_001, 194, device="cuda", dtype=BF)
    dy = torch.full_like(x, 0.3)
    b = torch.zeros(194, device="cuda")
    db = run(x, 2, None, b, 1e-5, False, dy)[2].double()
    want = 149 * 60_001 * float(dy[0, 0, 0])
    assert float((db - want).abs().max()) <= (1024 + 1) * 2.0 ** -24 * want  # (and rounded once)


def test_constant_gradients_of_many_rows():
    x = torch.randn(4_500_000, 512, device="cuda", dtype=BF)
    dy = torch.full_like(x, 0.3)
    b = torch.zeros(512, device="cuda")
    db = run(x, 512, None, b, 1e-5, False, dy)[2].double()
    want = 4_500_000 * float(dy[0, 0])
    assert float((db - want).abs().max()) <= (1024 + 1) * 2.0 ** -24 * want
