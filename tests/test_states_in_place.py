"""States that a decode step writes in place: autograd sees the write, so a graph that saved the state
before it refuses its backward instead of using the new values."""

import pytest
import torch

DEV = "cuda"


def _recurrence_step(state, batch=2, channels=24):
    from metal_kernelops.cv import gated_recurrence_update
    x = torch.randn(batch, channels, device=state.device)
    return gated_recurrence_update(state, x, x, x, x[0].clone(), out_state=state)


# --------------------------------------------------------------------------- CPU: the launch replaced


def test_an_update_in_place_moves_the_version(monkeypatch):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_recurrence
    monkeypatch.setattr(gated_recurrence.__globals__["nat"], "launch", lambda *a: None)
    monkeypatch.setitem(gated_recurrence.__globals__, "_require_gpu", lambda t: None)
    state = torch.randn(2, 24)
    leaf = torch.ones(2, 24, requires_grad=True)
    loss = (leaf * state).sum()
    before = state._version
    with torch.no_grad():
        assert _recurrence_step(state)[1] is state
    assert state._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():  # such tensors have no version
        _recurrence_step(torch.zeros(2, 24))
    assert nat.written(state) is None


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
def test_a_scan_whose_state_was_overwritten_refuses_its_backward():
    from metal_kernelops.cv import gated_recurrence
    x = torch.randn(2, 70, 24, device=DEV)
    gate = torch.randn(2, 70, 24, device=DEV, requires_grad=True)
    state = torch.randn(2, 24, device=DEV)
    y = gated_recurrence(x, x, gate, x[0, 0].clone(), initial_state=state)
    with torch.no_grad():
        _recurrence_step(state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.inference_mode():
        held = torch.zeros(2, 24, device=DEV)
        assert torch.isfinite(_recurrence_step(held)[1]).all()
