"""Projections in 8-bit integers: oracle pins on the CPU, HIP parity on the GPU.

Tolerances.  Quantisation is two IEEE roundings that the oracle makes too: bit for bit.  The
product's sum is exact; its conversion to float32, two scales and the bias are at most four
roundings of 2^-24 of the larger addend, then the output's own half unit (2^-24, 2^-11, 2^-8).
"""

import pytest
import torch

from oracle import recurrent_layer as oracle

DEV = "cuda"
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# (rows, inner, outer): single values, inner lengths around 16-byte loads and the kernels' k steps,
# rows and outer widths around every tile, ragged and odd ones
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 2560, 5120), (2, 15, 33), (3, 17, 64), (5, 1000, 4099), (15, 64, 17),
          (16, 128, 256), (17, 129, 255), (31, 777, 100), (32, 256, 48), (33, 512, 1000), (63, 1023, 65),
          (64, 1024, 64), (65, 100, 129), (100, 4096, 32), (127, 144, 127), (128, 128, 128), (129, 272, 257),
          (200, 2560, 300), (255, 260, 255), (256, 256, 256), (257, 48, 513), (300, 384, 4099), (513, 1000, 520),
          (1000, 1, 40), (1030, 640, 770), (2048, 768, 1536)]


def quantised(rows, inner, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (rows, inner), generator=g, dtype=torch.int8), \
        torch.rand(rows, generator=g) * 0.02 + 1e-3


def bound(want, dtype, *addends):
    largest = torch.stack([want.abs(), *[a.abs().expand_as(want) for a in addends]]).amax(0)
    return 4 * 2.0 ** -24 * largest + (HALF_ULP[dtype] * 1.001) * want.abs() + 1e-30


def check(q, qs, w, ws, bias, dtype, views=None):
    """The product of q and w, or of `views` that hold the same values on the GPU."""
    from metal_kernelops.cv import int8_linear
    dq, dw = views if views is not None else (q.to(DEV), w.to(DEV))
    out = int8_linear(dq, qs.to(DEV), dw, ws.to(DEV), bias=None if bias is None else bias.to(DEV),
                      out_dtype=dtype)
    want = oracle.int8_linear(q, qs, w, ws, bias)
    plain = oracle.int8_linear(q, qs, w, ws)
    assert out.shape == want.shape and out.dtype == dtype
    off = (out.cpu().double() - want).abs()
    extra = 2.0 ** -25 if dtype == torch.float16 else 0.0  # float16's smallest steps
    assert (off <= bound(want, dtype, plain, *(() if bias is None else (bias.double(),))) + extra).all()
    return out


# --------------------------------------------------------------------------- CPU: oracle pins


def test_oracle_product_equals_integers():
    q, qs = quantised(7, 40, 1)
    w, ws = quantised(9, 40, 2)
    acc = (q.long()[:, None] * w.long()[None]).sum(-1)
    want = acc.double() * qs.double()[:, None] * ws.double()
    assert torch.equal(oracle.int8_linear(q, qs, w, ws), want)


def test_oracle_quantisation_is_within_half_a_step():
    x = torch.randn(20, 100, generator=torch.Generator().manual_seed(4))
    x[3] = 0.0
    q, scale = oracle.quantize_int8(x)
    assert (q[3] == 0).all() and scale[3] == 0
    assert ((q.double() * scale.double()[:, None] - x.double()).abs() <= scale.double()[:, None] * 0.50001).all()
    assert (q.abs().amax(-1)[scale > 0] == 127).all()


def test_reference_twins_match_the_oracle():
    from metal_kernelops.cv import int8_linear_reference, quantize_int8_reference
    x = torch.randn(6, 50, generator=torch.Generator().manual_seed(5))
    x[2] = 0.0
    q, scale = quantize_int8_reference(x)
    oq, oscale = oracle.quantize_int8(x)
    assert (q.int() - oq.int()).abs().max() <= 1 and (scale - oscale).abs().max() <= 2.0 ** -24 * oscale.max()
    w, ws = quantised(8, 50, 6)
    bias = torch.randn(8)
    got = int8_linear_reference(q, scale, w, ws, bias, torch.float32)
    assert torch.equal(got, oracle.int8_linear(q, scale, w, ws, bias).float())


def test_native_argument_checks_without_a_gpu():
    import ctypes

    from metal_kernelops import _native as nat
    lib = nat.lib()
    p = nat.Int8LinearParams(rows=2, inner=8, outer=4, dtype=3)
    assert lib.mko_int8_linear(ctypes.byref(p), None) == 1 and b"dtype" in lib.mko_last_error()
    p.dtype = 2
    assert lib.mko_int8_linear(ctypes.byref(p), None) == 1 and b"required" in lib.mko_last_error()
    p.inner = 1 << 17
    assert lib.mko_int8_linear(ctypes.byref(p), None) == 3 and b"inner" in lib.mko_last_error()
    p.inner = -1
    assert lib.mko_int8_linear(ctypes.byref(p), None) == 1
    p.inner, p.rows = 8, 0
    assert lib.mko_int8_linear(ctypes.byref(p), None) == 0
    z = nat.QuantizeParams(rows=2, features=8, q_stride=4, dtype=0)
    assert lib.mko_quantize_int8(ctypes.byref(z), None) == 1


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_product(shape):
    rows, inner, outer = shape
    q, qs = quantised(rows, inner, rows + inner)
    w, ws = quantised(outer, inner, outer)
    bias = torch.randn(outer, generator=torch.Generator().manual_seed(outer))
    for dtype in DTYPES:
        check(q, qs, w, ws, bias, dtype)
    check(q, qs, w, ws, None, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("inner", [96, 100, 257])
@pytest.mark.parametrize("rows,outer", [(700, 600), (2048, 4352), (4100, 4099), (4090, 4096)])
def test_every_tile(rows, outer, inner):
    """Sizes that each tile is chosen for, 64 x 64 to 256 x 256, with direct loads and without."""
    q, qs = quantised(rows, inner, rows)
    w, ws = quantised(outer, inner, outer)
    bias = torch.randn(outer, generator=torch.Generator().manual_seed(1))
    check(q, qs, w, ws, bias, torch.bfloat16 if inner == 96 else torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 150, 700])
def test_largest_values_stay_exact(rows):
    """-128 and 127 throughout, at the longest sum that int32 holds."""
    inner = 131071
    q = torch.full((rows, inner), -128, dtype=torch.int8)
    w = torch.full((5, inner), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(rows), torch.ones(5)
    check(q, one[0], w, one[1], None, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 90, 300])
@pytest.mark.parametrize("inner", [64, 1000, 1001])
def test_strides_offsets_and_poison(rows, inner):
    """Rows inside wider tensors, at odd byte offsets, with other values on every side."""
    outer = 140
    q, qs = quantised(rows, inner, 1)
    w, ws = quantised(outer, inner, 2)
    for lead, pitch in ((0, inner + 16), (1, inner + 3), (16, inner + 32), (4, inner + 4)):
        wide_q = torch.full((rows + 2, lead + pitch), 77, dtype=torch.int8, device=DEV)
        wide_w = torch.full((outer + 2, lead + pitch), -99, dtype=torch.int8, device=DEV)
        vq, vw = wide_q[1:-1, lead:lead + inner], wide_w[1:-1, lead:lead + inner]
        vq.copy_(q)
        vw.copy_(w)
        check(q, qs, w, ws, None, torch.float32, (vq, vw))
    check(q, qs, w, ws, None, torch.float32, (q.t().to(DEV).contiguous().t(), w.t().to(DEV).contiguous().t()))
    check(q[:1].expand(rows, -1), qs, w, ws, None, torch.float32, (q[:1].to(DEV).expand(rows, -1), w.to(DEV)))


@pytest.mark.gpu
@pytest.mark.parametrize("inner", [1, 15, 17, 100, 127, 1000, 1001])
@pytest.mark.parametrize("rows,outer", [(30, 70), (100, 1500), (700, 600), (2048, 4352), (4090, 4096)])
def test_aligned_rows_of_odd_lengths(rows, outer, inner):
    """Rows at multiples of 16 bytes, as the quantisations write them, with other values after their end."""
    pitch = -(-inner // 16) * 16
    q, qs = quantised(rows, inner, 7)
    w, ws = quantised(outer, inner, 8)
    wide_q = torch.full((rows, pitch), 77, dtype=torch.int8, device=DEV)
    wide_w = torch.full((outer, pitch), -99, dtype=torch.int8, device=DEV)
    vq, vw = wide_q[:, :inner], wide_w[:, :inner]
    vq.copy_(q)
    vw.copy_(w)
    check(q, qs, w, ws, None, torch.float32, (vq, vw))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 30, 128, 520])
def test_the_end_of_an_allocation(rows):
    """Operands whose last byte is the last of their memory."""
    for inner in (1, 15, 100, 1001):
        q, qs = quantised(rows, inner, 3)
        w, ws = quantised(37, inner, 4)
        check(q, qs, w, ws, None, torch.float32)


@pytest.mark.gpu
def test_scales_that_are_zero_or_not_finite():
    from metal_kernelops.cv import int8_linear
    for rows in (6, 200):
        q, qs = quantised(rows, 64, 5)
        w, ws = quantised(20, 64, 6)
        qs[1], qs[2], qs[3] = 0.0, float("inf"), float("nan")
        q[2] = 0
        out = int8_linear(q.to(DEV), qs.to(DEV), w.to(DEV), ws.to(DEV), out_dtype=torch.float32).cpu()
        assert (out[1] == 0).all() and torch.isnan(out[2]).all() and torch.isnan(out[3]).all()
        assert torch.isfinite(out[4:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features", [1, 7, 64, 77, 520, 1000, 1001, 2560, 4099, 8192, 40000])
def test_quantise(features, dtype):
    from metal_kernelops.cv import quantize_int8
    rows = 5 if features < 8192 else 2
    x = (torch.randn(rows, features, generator=torch.Generator().manual_seed(features)) * 3).to(dtype)
    if rows > 2:
        x[2] = 0.0
    q, scale = quantize_int8(x.to(DEV))
    want, want_scale = oracle.quantize_int8(x)
    assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu(), want_scale)
    assert q.stride(0) % 16 == 0
    whole = torch.empty(0, dtype=torch.int8, device=DEV).set_(q.untyped_storage()).view(rows, -1)
    assert (whole[:, features:] == 0).all()
    wide = torch.full((rows, features + 9), 1e4, device=DEV).to(dtype)
    wide[:, 3:3 + features] = x.to(DEV)
    assert torch.equal(quantize_int8(wide[:, 3:3 + features])[0].cpu(), want)


@pytest.mark.gpu
def test_quantise_many_rows_and_odd_values():
    from metal_kernelops.cv import quantize_int8
    x = torch.randn(3000, 300, generator=torch.Generator().manual_seed(8))
    q, scale = quantize_int8(x.to(DEV))
    want, want_scale = oracle.quantize_int8(x)
    assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu(), want_scale)
    y = torch.randn(6, 40, generator=torch.Generator().manual_seed(9))
    y[0, 3], y[1, 3], y[2], y[3, 0] = float("inf"), float("nan"), 1e-38, -float("inf")
    q, scale = quantize_int8(y.to(DEV))
    assert not torch.isfinite(scale[[0, 1, 3]]).any() and scale[2] == 0 and (q[2] == 0).all()
    assert torch.equal(q[4:].cpu(), oracle.quantize_int8(y[4:])[0])
    ties = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]])
    assert quantize_int8(ties.to(DEV))[0].tolist() == [[127, 0, 2, 2, 0, -2, -2, 126]]
    z = quantize_int8(torch._neg_view(x[:4].to(DEV)))[0]
    assert torch.equal(z.cpu(), oracle.quantize_int8(-x[:4])[0])


@pytest.mark.gpu
def test_shapes_and_empty_sizes():
    from metal_kernelops.cv import int8_linear, quantize_int8
    g = torch.Generator().manual_seed(10)
    x, w = torch.randn(2, 3, 50, generator=g).to(DEV), torch.randn(8, 50, generator=g).to(DEV)
    q, s = quantize_int8(x)
    wq, ws = quantize_int8(w)
    out = int8_linear(q, s, wq, ws, out_dtype=torch.float32)
    assert out.shape == (2, 3, 8)
    assert torch.equal(out[1, 2], int8_linear(q[1, 2], s[1, 2], wq, ws, out_dtype=torch.float32))
    assert torch.equal(out.transpose(0, 1),
                       int8_linear(q.transpose(0, 1), s.transpose(0, 1), wq, ws, out_dtype=torch.float32))
    bias = torch.randn(8, generator=g).to(DEV)
    assert int8_linear(q[:0], s[:0], wq, ws).shape == (0, 3, 8)
    assert int8_linear(q, s, wq[:0], ws[:0]).shape == (2, 3, 0)
    empty = int8_linear(*quantize_int8(x[..., :0]), *quantize_int8(w[:, :0]), bias=bias, out_dtype=torch.float32)
    assert torch.equal(empty, bias.expand(2, 3, 8))
    assert quantize_int8(x[:0])[0].shape == (0, 3, 50)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    from metal_kernelops.cv import int8_linear, quantize_int8
    for rows in (3, 70, 300):
        x = torch.randn(rows, 512, generator=torch.Generator().manual_seed(11)).to(DEV)
        w, ws = quantised(700, 512, 12)
        w, ws = w.to(DEV), ws.to(DEV)

        def step():
            return int8_linear(*quantize_int8(x), w, ws, out_dtype=torch.float32)

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = step()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(there, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for k in range(3):
            x.copy_(torch.randn(rows, 512, generator=torch.Generator().manual_seed(k)))
            graph.replay()
            assert torch.equal(held, step())


@pytest.mark.gpu
def test_refusals():
    from metal_kernelops.cv import int8_linear, quantize_int8
    q, w = torch.zeros(3, 8, dtype=torch.int8, device=DEV), torch.zeros(4, 8, dtype=torch.int8, device=DEV)
    s, ws = torch.ones(3, device=DEV), torch.ones(4, device=DEV)
    bad = [((q[:, :7], s, w, ws), {}), ((q, s[:2], w, ws), {}), ((q, s, w[0], ws), {}), ((q, s, w, ws[:3]), {}),
           ((q.cpu(), s.cpu(), w.cpu(), ws.cpu()), {}), ((q, s.cpu(), w, ws), {}), ((q.float(), s, w, ws), {}),
           ((q, s, w.int(), ws), {}), ((q, s.int(), w, ws), {}), ((q, s, w, ws), {"bias": ws[:2]}),
           ((q, s, w, ws), {"bias": ws.cpu()}), ((q, s, w, ws), {"out_dtype": torch.float64}),
           ((q, s, w, ws), {"bias": ws.clone().requires_grad_(True)})]
    for args, kw in bad:
        with pytest.raises(ValueError, match="int8_linear|ROCm GPU"):
            int8_linear(*args, **kw)
    wide = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="131071"):
        int8_linear(wide, s[:1], wide, ws[:1])
    for x in (torch.zeros(3, 4), torch.zeros(3, 4, device=DEV, dtype=torch.float64), torch.zeros((), device=DEV),
              torch.zeros(3, 4, device=DEV, requires_grad=True)):
        with pytest.raises(ValueError):
            quantize_int8(x)
