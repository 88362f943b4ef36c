"""How many samples and groups group_norm takes."""
import ctypes as C

import pytest
import torch


def _scratch(N, S, channels, groups):
    from openkimi_b200 import _lib

    fb, bb = C.c_size_t(), C.c_size_t()
    return _lib.load().kda_group_norm_scratch_bytes(N, S, channels, groups, 1, C.byref(fb), C.byref(bb)), fb.value, bb.value


def test_samples_that_the_entry_point_takes():
    """Grids count samples times slices of a sample, and many samples have one slice each."""
    for N in (9_000_000, 2 ** 31 - 1):
        assert _scratch(N, 2, 8, 1) == (0, N * 8 * 9, N * 8 * 9)
    assert _scratch(2 ** 31, 2, 8, 1)[0] == 2
    assert _scratch(2 ** 31 - 1, 2 ** 20, 8, 1)[0] == 2  # two slices a sample
    assert _scratch(1, 2 ** 50, 512, 1)[0] == 2
    assert _scratch(2, 3, 24576, 24576)[0] == 0 and _scratch(2, 3, 24577, 24577)[0] == 2
    assert _scratch(3, 1, 2 ** 20, 2 ** 20)[0] == 0


@pytest.mark.gpu
def test_samples_and_groups():
    from openkimi_b200 import group_norm

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(9_000_000, 2, 8, generator=gen, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = group_norm(x, 1, activation="silu")
    (dx,) = torch.autograd.grad(y, x, y.detach())
    # (other samples at once: other slices, the same FP32 statistics of 16 values)
    end = x.detach()[-300:].clone().requires_grad_()
    y2 = group_norm(end, 1, activation="silu")
    (dx2,) = torch.autograd.grad(y2, end, y2.detach())
    assert torch.equal(y[-300:], y2) and torch.equal(dx[-300:], dx2)
    z = torch.zeros(1, 2, 24577, device="cuda")
    with pytest.raises(ValueError, match="at most 24576 groups"):
        group_norm(z, 24577)
    assert group_norm(z[:, 0], 24577).shape == (1, 24577)
    assert torch.equal(group_norm(z[..., :24576] + 3, 24576), torch.zeros_like(z[..., :24576]))


def test_channels_that_32_bits_count_twice():
    assert _scratch(1, 1, 2 ** 30, 2 ** 20)[0] == 0
    assert _scratch(1, 1, 2 ** 31 - 1024, 2 ** 21 - 1)[0] == 2 and _scratch(1, 3, 2 ** 31 - 1, 1)[0] == 2
