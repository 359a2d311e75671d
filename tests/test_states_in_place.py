"""States that a decode step writes in place: autograd sees the write, so a graph that saved the state
before it refuses its backward instead of using the new values."""

import pytest
import torch

DEV = "cuda"


def _recurrence_step(state, batch=2, channels=24):
    from metal_kernelops.cv import gated_recurrence_update
    x = torch.randn(batch, channels, device=state.device)
    return gated_recurrence_update(state, x, x, x, x[0].clone(), out_state=state)


def _ssm_step(state, **kw):
    from metal_kernelops.cv import mamba2_state_update
    (b, h, d, n), dev = state.shape, state.device
    x, B = torch.randn(b, h, d, device=dev), torch.randn(b, 1, n, device=dev)
    return mamba2_state_update(state, x, torch.rand(b, h, device=dev), -torch.rand(h, device=dev), B, B, **kw)


# --------------------------------------------------------------------------- CPU: the launch replaced


def test_an_update_in_place_moves_the_version(monkeypatch):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_recurrence
    monkeypatch.setattr(nat, "launch", lambda *a: None)
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("alias", ["itself", "data", "detached"])
def test_a_recorded_update_keeps_the_entering_state(monkeypatch, alias, dtype):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_recurrence, gated_recurrence_update
    kept = []
    monkeypatch.setattr(nat, "launch", lambda name, p, device: kept.append((name, p.initial)))
    monkeypatch.setitem(gated_recurrence.__globals__, "_require_gpu", lambda t: None)
    state = torch.randn(2, 24).to(dtype)
    if alias != "itself":
        state.requires_grad_(True)
    out = {"itself": state, "data": state.data, "detached": state.detach()}[alias]
    x = torch.randn(2, 24, requires_grad=True)
    y, new = gated_recurrence_update(state, x, x, x, torch.randn(24), out_state=out)
    assert new is out and not new.requires_grad
    y.sum().backward()
    assert [name for name, _ in kept] == ["mko_recur_fwd", "mko_recur_bwd"]
    assert kept[0][1] == kept[1][1] != out.data_ptr()  # both read the state from memory of its own
    assert x.grad is not None and (alias == "itself" or state.grad.dtype == dtype)


@pytest.mark.parametrize("shift", [0, 1, -1, 3])
def test_a_shifted_destination_is_not_read(monkeypatch, shift):
    """Rows of one buffer moved by ``shift`` rows: the kernel reads a copy unless they are the same."""
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_recurrence, gated_recurrence_update
    seen = []
    monkeypatch.setattr(nat, "launch", lambda name, p, device: seen.append((p.state, p.new_state)))
    monkeypatch.setitem(gated_recurrence.__globals__, "_require_gpu", lambda t: None)
    buffer, x = torch.zeros(9, 24), torch.zeros(3, 24)
    state, out = buffer[3:6], buffer[3 + shift:6 + shift]
    gated_recurrence_update(state, x, x, x, x[0], out_state=out)
    read, wrote = seen[0]
    assert wrote == out.data_ptr()
    assert (read == state.data_ptr()) == (shift in (0, 3))  # three rows on is another place altogether


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("alias", ["itself", "data"])
def test_gradients_of_an_update_in_place(alias, dtype):
    """Those of the same call with a destination of its own, bit for bit."""
    from metal_kernelops.cv import gated_recurrence_update
    x, ig, rg = (torch.randn(3, 40, device=DEV) for _ in range(3))
    start, decay, dy = torch.randn(3, 40, device=DEV).to(dtype), torch.randn(40, device=DEV), torch.randn(3, 40, device=DEV)

    def run(in_place):
        state = start.clone().requires_grad_(alias == "data")
        leaves = [t.clone().requires_grad_(True) for t in (x, ig, rg, decay)]
        out = (state.data if alias == "data" else state) if in_place else None
        y, new = gated_recurrence_update(state, *leaves, out_state=out)
        grads = torch.autograd.grad(y, leaves + ([state] if alias == "data" else []), dy)
        assert out is None or new is out
        return [y.detach(), new.detach(), *grads]

    assert all(torch.equal(a, b) for a, b in zip(run(True), run(False)))


@pytest.mark.gpu
def test_a_destination_shifted_against_the_state():
    from metal_kernelops.cv import gated_recurrence_update
    buffer, x = torch.randn(600, 520, device=DEV), torch.randn(599, 520, device=DEV)
    decay = torch.randn(520, device=DEV)
    want = gated_recurrence_update(buffer[:-1].clone(), x, x, x, decay)
    got = gated_recurrence_update(buffer[:-1], x, x, x, decay, out_state=buffer[1:])
    assert torch.equal(got[0], want[0]) and torch.equal(buffer[1:], want[1])


def test_only_shifted_memory_is_copied():
    from metal_kernelops import _native as nat
    t = torch.zeros(9, 24)
    for shift in range(-3, 4):
        state, out = t[3:6], t[3 + shift:6 + shift]
        assert (nat.unshifted(state, out) is state) == (shift in (0, 3, -3))


@pytest.mark.gpu
def test_an_ssm_destination_shifted_against_the_state():
    from metal_kernelops.cv import mamba2_state_update
    buffer, x = torch.randn(300, 4, 8, 16, device=DEV), torch.randn(299, 4, 8, device=DEV)
    dt, A, B = torch.rand(299, 4, device=DEV), -torch.rand(4, device=DEV), torch.randn(299, 1, 16, device=DEV)
    want = mamba2_state_update(buffer[:-1].clone(), x, dt, A, B, B)
    got = mamba2_state_update(buffer[:-1], x, dt, A, B, B, out_state=buffer[1:])
    assert torch.equal(got[0], want[0]) and torch.equal(buffer[1:], want[1])


@pytest.mark.gpu
def test_an_ssm_state_in_place_moves_the_version():
    state = torch.randn(2, 4, 8, 16, device=DEV)
    dt = torch.rand(2, 4, device=DEV, requires_grad=True)
    from metal_kernelops.cv import mamba2_state_update
    x, B = torch.randn(2, 4, 8, device=DEV), torch.randn(2, 1, 16, device=DEV)
    y, _ = mamba2_state_update(state, x, dt, -torch.rand(4, device=DEV), B, B)
    with torch.no_grad():
        assert _ssm_step(state, out_state=state)[1] is state
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.inference_mode():
        held = torch.zeros(2, 4, 8, 16, device=DEV)
        assert torch.isfinite(_ssm_step(held, out_state=held)[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("alias", ["itself", "data"])
def test_gradients_of_an_ssm_update_in_place(alias):
    from metal_kernelops.cv import mamba2_state_update
    start, x, dt = (torch.randn(s, device=DEV) for s in ((2, 4, 8, 16), (2, 4, 8), (2, 4)))
    A, B, dy = -torch.rand(4, device=DEV), torch.randn(2, 1, 16, device=DEV), torch.randn(2, 4, 8, device=DEV)

    def run(in_place):
        state = start.clone().requires_grad_(alias == "data")
        leaves = [t.clone().requires_grad_(True) for t in (x, dt, A, B)]
        out = (state.data if alias == "data" else state) if in_place else None
        y, new = mamba2_state_update(state, *leaves, leaves[-1], out_state=out)
        grads = torch.autograd.grad(y, leaves + ([state] if alias == "data" else []), dy)
        assert out is None or new is out
        return [y.detach(), new.detach(), *grads]

    assert all(torch.equal(a, b) for a, b in zip(run(True), run(False)))
