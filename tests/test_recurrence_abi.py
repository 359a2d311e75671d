"""Argument checks of the recurrence's C entries that come before any launch: nothing here runs a kernel."""

import ctypes

import pytest


def _params(**kw):
    """A problem of two chunks at made-up addresses."""
    from metal_kernelops import _native as nat
    names = ("x", "input_gate", "decay_gate", "decay", "y", "states", "dy", "dx", "dinput_gate", "ddecay_gate", "workspace")
    at = {n: 1 << 20 for n in names}
    return nat.RecurParams(**{**at, "workspace_bytes": 1 << 20, "batch": 1, "length": 65, "channels": 8, "scale": 8.0,
                              "dtype": 0, **kw})


@pytest.mark.parametrize("name,field", [("mko_recur_fwd", "workspace"), ("mko_recur_fwd", "states"),
                                        ("mko_recur_bwd", "workspace")])
@pytest.mark.parametrize("off", [1, 4, 8])
def test_unaligned_cells_are_refused(name, field, off):
    """The chunks' cells are cleared in 16-byte stores and a map is a 64-bit atomic word."""
    from metal_kernelops import _native as nat
    lib = nat.lib()
    p = _params(**{field: (1 << 20) + off})
    assert getattr(lib, name)(ctypes.byref(p), None) == 1 and b"16 bytes" in lib.mko_last_error()
