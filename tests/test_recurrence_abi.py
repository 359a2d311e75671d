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


@pytest.mark.parametrize("sizes", [(1 << 15, 1 << 31, 1 << 31), (1 << 14, 1 << 31, 1 << 31), (65535, 1 << 31, 1 << 31),
                                   (1, 1 << 31, 1 << 31), (1, (1 << 28) + 1, 1), (8, 1 << 25, 129)])
def test_sizes_past_the_launch_are_refused(sizes):
    """The count of workgroups of the first passes 64 bits and would wrap to zero."""
    from metal_kernelops import _native as nat
    lib = nat.lib()
    batch, length, channels = sizes
    p = _params(batch=batch, length=length, channels=channels)
    for name in ("mko_recur_fwd", "mko_recur_bwd"):
        assert getattr(lib, name)(ctypes.byref(p), None) == 3 and b"2^22" in lib.mko_last_error()
    assert lib.mko_recur_states_size(ctypes.byref(p)) == 0


def test_the_largest_problem_has_its_sizes():
    from metal_kernelops import _native as nat
    lib = nat.lib()
    p = _params(batch=8, length=64 << 10, channels=512 * 128)  # 4096 chains of 1024 chunks: 2^22 workgroups
    cells = 8 * (1 << 10) * 512 * 128
    assert lib.mko_recur_states_size(ctypes.byref(p)) == cells * 4
    assert lib.mko_recur_fwd_workspace_size(ctypes.byref(p)) == cells * 8 + 1024
