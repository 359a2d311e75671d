"""RMS norm of the residual stream: oracle pins on the CPU, HIP parity on the GPU.

Tolerances.  Float32, relative error of the global norm: a mean of squares and a dot product in
float32, each summed in blocks (errors below 8 * 2^-24 relative), and four roundings an element:
1e-6.  ``dweight`` sums rows, with the same terms.  16-bit outputs add their rounding, at most half
a unit in the last place: 2^-11 for float16, 2^-8 for bfloat16.  The stream is one rounded sum and
is compared bit for bit.  An 8-bit value is off by half a step, and by 1e-4 of a step for the
float32 value that was rounded.
"""

import pytest
import torch

from oracle import recurrent_layer as oracle

DEV = "cuda"
F32_TOL = 1e-6
TOL = {torch.float32: F32_TOL, torch.float16: F32_TOL + 2.0 ** -11, torch.bfloat16: F32_TOL + 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
# one feature, around a wavefront's and a workgroup's vectors, odd widths, and beyond what any
# workgroup holds in registers
FEATURES = [1, 7, 64, 77, 512, 520, 1000, 1001, 2560, 4099, 8192, 40000]


def problem(rows, features, dtype, stream, seed=0, wdtype=F32):
    g = torch.Generator().manual_seed(seed * 77 + rows + features)

    def r(*shape):
        return torch.randn(shape, generator=g)

    return {"x": r(rows, features).to(dtype), "residual": (2 * r(rows, features)).to(stream),
            "weight": (1 + 0.1 * r(features)).to(wdtype), "dout": r(rows, features).to(dtype),
            "dstream": r(rows, features).to(stream)}


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    scale = want.norm().item()
    return (got - want).norm().item() / (scale if scale else 1.0)


def to_dev(p):
    return {k: None if v is None else v.to(DEV) for k, v in p.items()}


def check(p, residual=True, use=("out", "stream"), eps=1e-5):
    from metal_kernelops.cv import rmsnorm_residual
    d = to_dev(p)
    names = ["x", "weight"] + (["residual"] if residual else [])
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in names}
    out, stream = rmsnorm_residual(leaves["x"], leaves["weight"], leaves.get("residual"), eps=eps)
    want, want_stream = oracle.rmsnorm_residual(p["x"], p["weight"], p["residual"] if residual else None, eps)
    assert out.dtype == p["x"].dtype and rel(out, want) <= TOL[out.dtype]
    assert torch.equal(stream.detach().cpu().double(), want_stream)
    pairs = {"out": (out, d["dout"]), "stream": (stream, d["dstream"].to(stream.dtype))}
    grads = torch.autograd.grad([pairs[u][0] for u in use], list(leaves.values()), [pairs[u][1] for u in use],
                                allow_unused=True)
    dout = p["dout"] if "out" in use else torch.zeros_like(p["dout"])
    ds, dw = oracle.rmsnorm_residual_bwd(dout, p["dstream"].to(stream.dtype) if "stream" in use else None, want_stream,
                                         p["weight"], eps)
    got = dict(zip(names, grads))
    if residual:
        assert rel(got["x"], ds) <= TOL[p["x"].dtype]
        assert rel(got["residual"], ds) <= TOL[p["residual"].dtype]
    elif use == ("out",):
        assert rel(got["x"], ds) <= TOL[p["x"].dtype]
    if "out" in use:
        assert got["weight"].dtype == p["weight"].dtype and rel(got["weight"], dw) <= TOL[p["weight"].dtype]
    with torch.no_grad():
        plain, plain_stream = rmsnorm_residual(d["x"], d["weight"], d["residual"] if residual else None, eps=eps)
    assert torch.equal(plain, out) and torch.equal(plain_stream, stream)


# --------------------------------------------------------------------------- CPU: oracle pins


def test_oracle_backward_equals_autograd_and_differences():
    p = {k: v.double() for k, v in problem(3, 9, F32, F32).items()}
    x, w = p["x"].requires_grad_(True), p["weight"].requires_grad_(True)
    out, stream = oracle.rmsnorm_residual(x, w, p["residual"], 1e-3)
    loss = (out * p["dout"]).sum() + (stream * p["dstream"]).sum()
    gx, gw = torch.autograd.grad(loss, (x, w))
    ds, dw = oracle.rmsnorm_residual_bwd(p["dout"], p["dstream"], stream.detach(), w.detach(), 1e-3)
    assert (gx - ds).abs().max() < 1e-12 and (gw - dw).abs().max() < 1e-12
    step = 1e-6
    for i in range(0, 27, 4):
        e = torch.zeros(27, dtype=torch.float64)
        e[i] = step
        e = e.reshape(3, 9)

        def at(v):
            o, s = oracle.rmsnorm_residual(v, w.detach(), p["residual"], 1e-3)
            return (o * p["dout"]).sum() + (s * p["dstream"]).sum()

        assert abs((at(x.detach() + e) - at(x.detach() - e)) / (2 * step) - ds.reshape(-1)[i]) < 1e-7


def test_reference_twins_match_the_oracle():
    from metal_kernelops.cv import rmsnorm_residual_int8_reference, rmsnorm_residual_reference
    p = problem(4, 33, BF16, BF16)
    out, stream = rmsnorm_residual_reference(p["x"], p["weight"], p["residual"])
    want, want_stream = oracle.rmsnorm_residual(p["x"], p["weight"], p["residual"])
    assert torch.equal(out, want.to(BF16)) and torch.equal(stream.double(), want_stream)
    q, scale, s8 = rmsnorm_residual_int8_reference(p["x"], p["weight"], p["residual"])
    assert torch.equal(s8, stream) and q.dtype == torch.int8
    assert ((q.double() * scale.double()[:, None] - want).abs() <= scale.double()[:, None] * 0.5001).all()


def test_native_argument_checks_without_a_gpu():
    import ctypes

    from metal_kernelops import _native as nat
    lib = nat.lib()
    p = nat.ResnormParams(rows=2, features=8, dtype=2, stream_dtype=1, wdtype=0)
    assert lib.mko_resnorm_fwd(ctypes.byref(p), None) == 1 and b"stream" in lib.mko_last_error()
    p.stream_dtype = 2
    assert lib.mko_resnorm_fwd(ctypes.byref(p), None) == 1 and b"required" in lib.mko_last_error()
    assert lib.mko_resnorm_bwd(ctypes.byref(p), None) == 1
    p.rows = -1
    assert lib.mko_resnorm_fwd(ctypes.byref(p), None) == 1 and b"negative" in lib.mko_last_error()
    p.rows = 0
    assert lib.mko_resnorm_fwd(ctypes.byref(p), None) == 0


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,stream", PAIRS)
@pytest.mark.parametrize("features", FEATURES)
def test_forward_and_gradients(features, dtype, stream):
    check(problem(3 if features < 8192 else 2, features, dtype, stream))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 63, 300, 1025])
def test_rows(rows):
    check(problem(rows, 520, BF16, BF16))
    check(problem(rows, 77, BF16, F32))


@pytest.mark.gpu
def test_training_sizes():
    """Several row blocks of every workgroup, whole and ragged."""
    check(problem(4100, 2560, BF16, BF16))
    check(problem(1500, 1001, F16, F32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_residual_and_one_output_used(dtype):
    p = problem(5, 300, dtype, dtype)
    check(p, residual=False, use=("out",))
    check(p, use=("out",))
    check(p, use=("stream",))


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", [F32, F16, BF16])
def test_weight_dtypes_and_eps(wdtype):
    check(problem(5, 300, BF16, BF16, wdtype=wdtype), eps=1e-2)
    check(problem(5, 301, F32, F32, wdtype=wdtype), eps=1e-2)


@pytest.mark.gpu
def test_slices_shapes_and_negated_views():
    from metal_kernelops.cv import rmsnorm_residual
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 5, 1 + 2 * 77, generator=g).to(BF16).to(DEV)
    w = torch.randn(77, generator=g).to(DEV)
    x, res = wide[..., 1:78], wide[..., 78:]
    want = rmsnorm_residual(x.contiguous(), w, res.contiguous())
    for got in (rmsnorm_residual(x, w, res), rmsnorm_residual(x.transpose(0, 1), w, res.transpose(0, 1))):
        got = [t if t.shape == x.shape else t.transpose(0, 1) for t in got]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(rmsnorm_residual(torch._neg_view(x), w, res)[0], rmsnorm_residual(-x, w, res)[0])
    one = rmsnorm_residual(x[0, 0], w, res[0, 0])
    assert torch.equal(one[0], want[0][0, 0]) and torch.equal(one[1], want[1][0, 0])
    lead = rmsnorm_residual(x[:1, :1].expand(2, 5, 77), w, res)[1]
    assert torch.equal(lead, (x[:1, :1].float() + res.float()).to(BF16))


@pytest.mark.gpu
def test_shared_gradient_tensor_is_not_shared_by_leaves():
    """x and the residual of one dtype get one gradient; their .grad tensors are separate."""
    from metal_kernelops.cv import rmsnorm_residual
    p = to_dev(problem(4, 64, F32, F32))
    x, r = p["x"].requires_grad_(True), p["residual"].requires_grad_(True)
    rmsnorm_residual(x, p["weight"], r)[0].sum().backward()
    before = r.grad.clone()
    x.grad.add_(1.0)
    assert torch.equal(r.grad, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,stream", PAIRS)
@pytest.mark.parametrize("features", FEATURES)
def test_int8_output(features, dtype, stream):
    from metal_kernelops.cv import rmsnorm_residual_int8
    p = problem(3, features, dtype, stream)
    d = to_dev(p)
    q, scale, s = rmsnorm_residual_int8(d["x"], d["weight"], d["residual"])
    want, want_stream = oracle.rmsnorm_residual(p["x"], p["weight"], p["residual"])
    assert torch.equal(s.cpu().double(), want_stream)
    amax = want.abs().amax(-1)
    assert rel(scale, amax / 127) <= F32_TOL
    assert q.shape == p["x"].shape and q.stride(0) % 16 == 0 and q.abs().max() == 127
    step = (amax / 127)[:, None]
    assert ((q.cpu().double() * step - want).abs() <= step * (0.5 + 1e-4)).all()
    q2, scale2, s2 = rmsnorm_residual_int8(d["x"], d["weight"])
    want2, _ = oracle.rmsnorm_residual(p["x"], p["weight"])
    step = (want2.abs().amax(-1) / 127)[:, None]
    assert s2 is d["x"] and ((q2.cpu().double() * step - want2).abs() <= step * (0.5 + 1e-4)).all()


@pytest.mark.gpu
def test_int8_rows_of_zeros_infinities_and_nan():
    from metal_kernelops.cv import rmsnorm_residual_int8
    x = torch.randn(6, 130, generator=torch.Generator().manual_seed(1)).to(DEV)
    x[1] = 0.0
    x[2, 5], x[3, 129], x[4] = float("inf"), float("nan"), 1e-30
    q, scale, _ = rmsnorm_residual_int8(x, torch.ones(130, device=DEV))
    assert (q[1] == 0).all() and scale[1] == 0
    assert not torch.isfinite(scale[2:4]).any()
    assert torch.isfinite(scale[[0, 4, 5]]).all() and (q[[0, 5]].abs().amax(-1) == 127).all()


@pytest.mark.gpu
def test_weight_gradient_repeats_bit_for_bit():
    from metal_kernelops.cv import rmsnorm_residual
    p = to_dev(problem(3000, 1536, BF16, BF16))
    w = p["weight"].requires_grad_(True)
    grads = [torch.autograd.grad(rmsnorm_residual(p["x"], w, p["residual"])[0], w, p["dout"])[0] for _ in range(3)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.gpu
def test_empty_sizes():
    from metal_kernelops.cv import rmsnorm_residual, rmsnorm_residual_int8
    for shape in ((0, 8), (3, 0), (2, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[-1], device=DEV, requires_grad=True)
        out, stream = rmsnorm_residual(x, w, torch.zeros(shape, device=DEV))
        assert out.shape == shape and stream.shape == shape
        gx, gw = torch.autograd.grad(out.sum() + stream.sum(), (x, w))
        assert gx.shape == shape and torch.equal(gw, torch.zeros_like(w))
        with torch.no_grad():
            q, scale, _ = rmsnorm_residual_int8(x, w)
        assert q.shape == shape and scale.shape == shape[:-1]


@pytest.mark.gpu
def test_captured_graph_replays():
    from metal_kernelops.cv import rmsnorm_residual
    p = to_dev(problem(700, 520, BF16, BF16))
    leaves = [p[n].requires_grad_(True) for n in ("x", "weight", "residual")]

    def step():
        out, stream = rmsnorm_residual(*leaves)
        return (out, stream, *torch.autograd.grad([out, stream], leaves, [p["dout"], p["dstream"]]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            p["x"].copy_(torch.randn(p["x"].shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_refusals():
    from metal_kernelops.cv import rmsnorm_residual, rmsnorm_residual_int8
    x, w = torch.zeros(2, 8, device=DEV), torch.ones(8, device=DEV)
    for args in [(x, w[:7]), (x, w, x[:1]), (x.cpu(), w.cpu()), (x, w.cpu()), (x, w, x.cpu()), (x.double(), w),
                 (x, w.double()), (x, w, x.half()), (x.half(), w, x.to(BF16)), (torch.zeros((), device=DEV), w)]:
        for fn in (rmsnorm_residual, rmsnorm_residual_int8):
            with pytest.raises(ValueError):
                fn(*args)
    with pytest.raises(ValueError, match="no_grad"):
        rmsnorm_residual_int8(x, w.clone().requires_grad_(True))
