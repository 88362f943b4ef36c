"""The gated delta rule's calls under forward-mode differentiation, and after a failure on the device."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def _inputs():
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    return dict(q=r(2, 3, 1, 64), k=r(2, 3, 1, 64), v=r(2, 3, 2, 64), g=-r(2, 3, 2).abs(), beta=r(2, 3, 2).sigmoid(), initial_state=r(2, 2, 64, 64))


def _calls():
    import openkimi_b200 as kimi

    def step(q, k, v, g, beta, initial_state):
        return kimi.recurrent_gated_delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], initial_state)

    return kimi.chunk_gated_delta_rule, kimi.fused_recurrent_gated_delta_rule, step


@pytest.mark.parametrize("call", range(3))
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "initial_state"])
def test_tangents_are_refused(call, name):
    """An input's tangent is refused, not dropped."""
    x = _inputs()
    with fwd.dual_level():
        x[name] = fwd.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            _calls()[call](**x)


@pytest.mark.parametrize("call", range(3))
def test_a_failure_on_the_device_surfaces_in_the_next_call(call):
    """What a kernel's given-up wait leaves in the words of status: the next call raises, the one after it answers."""
    from openkimi_b200.ops import _DeviceStatus

    x = _inputs()
    want = _calls()[call](**x)
    torch.cuda.synchronize()
    words = _DeviceStatus.get(torch.device("cuda", torch.cuda.current_device()))
    words.dev.fill_(32)
    words.host.fill_(32)
    with pytest.raises(RuntimeError, match="bounded device-side wait gave up"):
        _calls()[call](**x)
    assert torch.equal(_calls()[call](**x)[0], want[0])
