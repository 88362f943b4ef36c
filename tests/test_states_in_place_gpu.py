"""A state that a decoding step updates in place, as autograd sees it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(rule, state, inplace=True):
    from openkimi_b200 import recurrent_gated_delta_rule_step, recurrent_kda_step

    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    q, k, v, beta = r(3, 2, 64), r(3, 2, 64), r(3, 2, 64), r(3, 2).sigmoid()
    if rule == "kda":
        return recurrent_kda_step(q, k, v, -r(3, 2, 64).abs(), beta, state, inplace=inplace)
    return recurrent_gated_delta_rule_step(q, k, v, -r(3, 2).abs(), beta, state, inplace=inplace)


@pytest.mark.parametrize("rule", ["kda", "gdr"])
def test_a_saved_state_that_is_updated_is_noticed(rule):
    """What autograd has saved of a state is not used after a step has changed it."""
    w = torch.randn(3, 2, 64, 64, device="cuda", requires_grad=True)
    state = torch.randn(3, 2, 64, 64, device="cuda")
    loss = (w * state).sum()
    _step(rule, state)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    loss = (w * state).sum()
    _step(rule, state, inplace=False)
    loss.backward()
    assert torch.equal(w.grad, state)


@pytest.mark.parametrize("rule", ["kda", "gdr"])
def test_states_of_every_mode(rule):
    """Made under inference mode, under no_grad, as a leaf with a gradient: updated alike."""
    first = torch.randn(3, 2, 64, 64, device="cuda")
    want = _step(rule, first, inplace=False)
    with torch.inference_mode():
        made = first.clone()
        inner = first.clone()
        assert torch.equal(_step(rule, inner)[1], want[1])
    for state in (made, first.clone(), first.clone().requires_grad_()):
        place = state.data_ptr()
        o, s = _step(rule, state)
        assert s.data_ptr() == place and torch.equal(s, want[1]) and torch.equal(o, want[0]) and torch.equal(state, want[1])
