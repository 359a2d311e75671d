"""The gated delta rule and the layer norm at the edges of what their calls allow: the largest launches, empty axes,
values that a padded lane turns into NaN, and gradients that are zero by the formulas."""

import ctypes

import pytest
import torch

from test_gated_delta import DEV, _params


# --------------------------------------------------------------------------- CPU: the largest calls


@pytest.mark.parametrize("name", ["mko_delta_fwd", "mko_delta_bwd"])
@pytest.mark.parametrize("kw", [{"batch": 1 << 13, "heads": 1 << 10}, {"batch": 1 << 10, "length": 64 << 13},
                                {"batch": 1 << 9, "heads": 2, "value": 16 << 13}])
def test_c_entries_refuse_more_threads_than_a_launch_has(name, kw):
    """Workgroups have up to 512 threads and a launch below 2^32, so it has room for fewer than 2^23 of them; one
    sequence less and the next check is reached."""
    from metal_kernelops import _native as nat
    lib = nat.lib()
    kw = {"length": 64, "heads": 1, "value": 16, "workspace_bytes": 64, **kw}
    assert getattr(lib, name)(ctypes.byref(_params(**kw)), None) == 3  # MKO_EUNSUPPORTED
    assert b"2^23" in lib.mko_last_error()
    kw["batch"] -= 1
    assert getattr(lib, name)(ctypes.byref(_params(**kw)), None) == 4  # MKO_EWORKSPACE


@pytest.mark.parametrize("name", ["mko_delta_fwd", "mko_delta_bwd"])
def test_c_entries_refuse_wide_values(name):
    from metal_kernelops import _native as nat
    assert getattr(nat.lib(), name)(ctypes.byref(_params(value=1 << 20)), None) == 3
    assert b"2^20" in nat.lib().mko_last_error()


def test_calls_refuse_what_the_launches_do_not_take(monkeypatch):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_delta, gated_delta_rule
    monkeypatch.setattr(gated_delta, "_require_gpu", lambda t: None)
    monkeypatch.setattr(nat, "launch", lambda *args: pytest.fail("launched"))
    monkeypatch.setattr(torch, "empty", lambda *args, **kw: pytest.fail("allocated"))
    one = torch.zeros(1)
    for batch, length, heads, value, text in [(1 << 13, 1, 1 << 10, 1, r"2\^23"), (1, 1 << 29, 1, 1, r"2\^23"),
                                              (1, 1, 1, 1 << 20, r"2\^20")]:
        q, v, gate = (one.expand(s) for s in ((batch, length, 1, 1), (batch, length, heads, value), (batch, length, heads)))
        with pytest.raises(ValueError, match=text):
            gated_delta_rule(q, q, v, gate, gate)
