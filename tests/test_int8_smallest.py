"""8-bit integers at their smallest and strangest: rows without features, a padding alone, NaN and infinities."""

import ctypes

import pytest
import torch

DEV = "cuda"


def test_a_padding_without_memory_is_refused():
    """Before any launch: the kernel would clear the padding through the null pointer."""
    from metal_kernelops import _native as nat
    lib = nat.lib()
    scale = torch.empty(2)
    p = nat.QuantizeParams(scale=scale.data_ptr(), rows=2, features=0, q_stride=16, dtype=0)
    assert lib.mko_quantize_int8(ctypes.byref(p), None) == 1 and b"required" in lib.mko_last_error()
    p.q_stride, p.scale = 0, None
    assert lib.mko_quantize_int8(ctypes.byref(p), None) == 1  # their scales are written
    p.rows = 0
    assert lib.mko_quantize_int8(ctypes.byref(p), None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pitch", [0, 16, 40])
def test_rows_without_features(pitch):
    """Their scales are 0 and their padding is cleared, as the C entry says."""
    from metal_kernelops import _native as nat
    scale = torch.full((300,), 7.0, device=DEV)
    q = torch.full((300, pitch + 1), 7, dtype=torch.int8, device=DEV)
    p = nat.QuantizeParams(q=q.data_ptr() if pitch else None, scale=scale.data_ptr(), rows=299, features=0, q_stride=pitch,
                           dtype=2)
    nat.launch("mko_quantize_int8", p, scale.device)
    assert (scale[:299] == 0).all() and scale[299] == 7
    flat = q.flatten()
    assert (flat[:299 * pitch] == 0).all() and (flat[299 * pitch:] == 7).all()


@pytest.mark.gpu
def test_rows_without_features_from_torch():
    from metal_kernelops.cv import quantize_int8
    for shape in ((3, 0), (2, 5, 0), (0,), (0, 0)):
        q, scale = quantize_int8(torch.empty(shape, device=DEV))
        assert q.shape == shape and torch.equal(scale, torch.zeros(shape[:-1], device=DEV))
