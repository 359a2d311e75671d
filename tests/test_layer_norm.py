"""Layer norm of the residual stream: oracle pins and refusals on the CPU, HIP parity on the GPU.

Tolerances, relative error of the global norm.  Float32: a mean, the squares of the differences from it
and two dot products, each summed in blocks (errors below 8 * 2^-24 relative to the sum of the terms'
magnitudes), and five roundings an element: 1e-6, and for rows whose mean is m deviations away the
mean's error of 8 * 2^-24 m beside it.  A row of few features can lie close together: its rounded
differences come back times r, 4 * 2^-24 r.  ``dweight`` and ``dbias`` sum rows in blocks, with the same terms.
16-bit outputs add their rounding, at most half a unit in the last place: 2^-11 for float16, 2^-8 for
bfloat16.  The stream is one rounded sum and is compared bit for bit.
"""

import ctypes

import pytest
import torch

from oracle import layer_norm as oracle

DEV = "cuda"
F32_TOL = 1e-6
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
TOL = {F32: F32_TOL, F16: F32_TOL + 2.0 ** -11, BF16: F32_TOL + 2.0 ** -8}
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
# one feature, around a quarter, a half and whole wavefronts' vectors, odd widths, several vectors a lane,
# and beyond what a team of lanes holds
FEATURES = [2, 7, 64, 77, 96, 128, 129, 256, 260, 512, 520, 1001, 1536, 2560, 4099, 5120, 8192, 10240, 13000, 40000]
NAMES = ("x", "weight", "bias", "residual")


def problem(rows, features, dtype, stream, seed=0, wdtype=F32, mean=0.5):
    g = torch.Generator().manual_seed(seed * 77 + rows + features)

    def r(*shape):
        return torch.randn(shape, generator=g)

    return {"x": r(rows, features).to(dtype), "residual": (2 * r(rows, features) + mean).to(stream),
            "weight": (1 + 0.1 * r(features)).to(wdtype), "bias": (0.1 * r(features)).to(wdtype),
            "dout": r(rows, features).to(dtype), "dstream": r(rows, features).to(stream)}


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    scale = want.norm().item()
    return (got - want).norm().item() / (scale if scale else 1.0)


def to_dev(p):
    return {k: None if v is None else v.to(DEV) for k, v in p.items()}


def call(a, eps=1e-5):
    from metal_kernelops.cv import layernorm_residual
    return layernorm_residual(a["x"], a["weight"], a.get("bias"), a.get("residual"), eps=eps)


def check(p, residual=True, bias=True, use=("out", "stream"), eps=1e-5, extra=0.0):
    d = to_dev(p)
    names = [n for n in NAMES if (residual or n != "residual") and (bias or n != "bias")]
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in names}
    out, stream = call(leaves, eps)
    want, want_stream = oracle.layernorm_residual(p["x"], p["weight"], p["bias"] if bias else None,
                                                  p["residual"] if residual else None, eps)
    assert out.dtype == p["x"].dtype and rel(out, want) <= TOL[out.dtype] + extra
    assert torch.equal(stream.detach().cpu().double(), want_stream)
    pairs = {"out": (out, d["dout"]), "stream": (stream, d["dstream"].to(stream.dtype))}
    grads = dict(zip(names, torch.autograd.grad([pairs[u][0] for u in use], list(leaves.values()),
                                                [pairs[u][1] for u in use], allow_unused=True)))
    ds, dw, db = oracle.layernorm_residual_bwd(p["dout"] if "out" in use else torch.zeros_like(p["dout"]),
                                               p["dstream"].to(stream.dtype) if "stream" in use else None, want_stream,
                                               p["weight"], eps)
    if residual:
        assert rel(grads["x"], ds) <= TOL[p["x"].dtype] + extra
        assert rel(grads["residual"], ds) <= TOL[p["residual"].dtype] + extra
    elif use == ("out",):
        assert rel(grads["x"], ds) <= TOL[p["x"].dtype] + extra
    if "out" in use:
        assert grads["weight"].dtype == p["weight"].dtype and rel(grads["weight"], dw) <= TOL[p["weight"].dtype] + extra
        if bias:
            assert grads["bias"].dtype == p["bias"].dtype and rel(grads["bias"], db) <= TOL[p["bias"].dtype]
    else:
        assert grads["weight"] is None
    with torch.no_grad():
        plain, plain_stream = call({n: d[n] for n in names}, eps)
    assert torch.equal(plain, out) and torch.equal(plain_stream, stream)


# --------------------------------------------------------------------------- CPU: oracle pins and refusals


def test_oracle_gradients_equal_autograd_and_differences():
    p = {k: v.double() for k, v in problem(3, 9, F32, F32).items()}
    leaves = {n: p[n].requires_grad_(True) for n in ("x", "weight", "bias")}

    def loss(a):
        out, stream = oracle.layernorm_residual(a["x"], a["weight"], a["bias"], p["residual"], 1e-3)
        return (out * p["dout"]).sum() + (stream * p["dstream"]).sum()

    want = torch.autograd.grad(loss(leaves), list(leaves.values()))
    got = oracle.layernorm_residual_bwd(p["dout"], p["dstream"], (p["x"] + p["residual"]).detach(), p["weight"].detach(), 1e-3)
    g = torch.Generator().manual_seed(2)
    for name, a, b in zip(leaves, got, want):
        assert (a - b).abs().max() < 1e-12, name
        d, step = torch.randn(b.shape, generator=g, dtype=F64), 1e-6
        ends = [loss({**leaves, name: leaves[name] + s * step * d}) for s in (1, -1)]
        assert abs((ends[0] - ends[1]).item() / (2 * step) - (b * d).sum().item()) < 1e-7, name


def test_reference_twin_matches_the_oracle():
    from metal_kernelops.cv import layernorm_residual_reference
    p = problem(4, 33, BF16, BF16)
    out, stream = layernorm_residual_reference(p["x"], p["weight"], p["bias"], p["residual"])
    want, want_stream = oracle.layernorm_residual(p["x"], p["weight"], p["bias"], p["residual"])
    assert rel(out, want) <= TOL[BF16] and torch.equal(stream.double(), want_stream)


def test_native_argument_checks_without_a_gpu():
    from metal_kernelops import _native as nat
    lib = nat.lib()
    for kw, status, text in [({"dtype": 2, "stream_dtype": 1}, 1, b"stream"), ({"dtype": 7}, 1, b"dtype"), ({}, 1, b"required"),
                             ({"rows": -1}, 1, b"negative"), ({"rows": 1 << 22}, 3, b"2^22"),
                             ({"features": 1 << 30}, 3, b"2^30")]:
        p = nat.LayernormParams(**{"rows": 2, "features": 8, **kw})
        for name in ("mko_layernorm_fwd", "mko_layernorm_bwd"):
            assert getattr(lib, name)(ctypes.byref(p), None) == status and text in lib.mko_last_error()
    at = {n: 1 << 20 for n in ("stream", "weight", "stats", "dout", "dx", "dweight")}
    p = nat.LayernormParams(**at, rows=300, features=1000)
    assert lib.mko_layernorm_bwd(ctypes.byref(p), None) != 0 and b"workspace" in lib.mko_last_error()
    at = {n: 1 << 20 for n in ("x", "weight", "out")}
    p = nat.LayernormParams(**at, rows=3, features=8, dtype=2, stream_dtype=0)
    assert lib.mko_layernorm_fwd(ctypes.byref(p), None) == 1 and b"without a residual" in lib.mko_last_error()
    p.rows = 0
    assert lib.mko_layernorm_fwd(ctypes.byref(p), None) == 0 and lib.mko_layernorm_bwd(ctypes.byref(p), None) == 0


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,stream", PAIRS)
@pytest.mark.parametrize("features", FEATURES)
def test_forward_and_gradients(features, dtype, stream):
    p = problem(3 if features < 8192 else 2, features, dtype, stream)
    r = (p["x"].double() + p["residual"].double()).var(-1, unbiased=False).min() ** -0.5
    check(p, extra=4 * 2.0 ** -24 * r.item() if features < 8 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 63, 300, 1025, 4100])
def test_rows(rows):
    check(problem(rows, 520, BF16, BF16))
    check(problem(rows, 77, BF16, F32))
    check(problem(rows, 250, F32, F32))


@pytest.mark.gpu
def test_training_sizes():
    """Several rows of every team, whole and ragged."""
    check(problem(4100, 2560, BF16, BF16))
    check(problem(1500, 1001, F16, F32))
    check(problem(50_000, 96, BF16, BF16))
    check(problem(700, 13_000, BF16, BF16))


@pytest.mark.gpu
def test_one_feature():
    """The difference from the mean is zero: the output is the bias, and x's gradient the stream's."""
    p = problem(5, 1, F32, F32)
    d = to_dev(p)
    leaves = {n: d[n].clone().requires_grad_(True) for n in NAMES}
    out, stream = call(leaves)
    assert torch.equal(out, d["bias"].expand(5, 1))
    grads = torch.autograd.grad([out, stream], list(leaves.values()), [d["dout"], d["dstream"]])
    assert torch.equal(grads[0], d["dstream"]) and torch.equal(grads[3], d["dstream"])
    assert grads[1].item() == 0 and abs(grads[2].item() - d["dout"].sum().item()) < 1e-6 * 5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_parts_left_out(dtype):
    p = problem(5, 300, dtype, dtype)
    check(p, residual=False, use=("out",))
    check(p, residual=False, bias=False, use=("out",))
    check(p, bias=False)
    check(p, use=("out",))
    check(p, use=("stream",))


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", [F32, F16, BF16])
def test_weight_dtypes_and_eps(wdtype):
    check(problem(5, 300, BF16, BF16, wdtype=wdtype), eps=1e-2)
    check(problem(5, 301, F32, F32, wdtype=wdtype), eps=1e-2)
    p = problem(5, 96, F32, F32)
    p["bias"] = p["bias"].to(wdtype)
    check(p)


@pytest.mark.gpu
@pytest.mark.parametrize("features", [64, 1001, 40000])
def test_rows_far_from_zero(features):
    """A mean of 1000 deviations: the variance is that of the differences, not of squares that cancel."""
    check(problem(7, features, F32, F32, mean=2000.0), extra=8 * 2.0 ** -24 * 1000)


@pytest.mark.gpu
def test_constant_rows_infinities_and_nan():
    x = torch.randn(5, 130, generator=torch.Generator().manual_seed(1)).to(DEV)
    w, b = torch.ones(130, device=DEV), torch.full((130,), 0.25, device=DEV)
    clean = call({"x": x, "weight": w, "bias": b})[0]
    x[1], x[2, 5], x[3, 129] = 3.0, float("inf"), float("nan")
    out = call({"x": x, "weight": w, "bias": b})[0]
    assert torch.equal(out[1], b) and torch.isnan(out[2:4]).all()
    assert torch.equal(out[[0, 4]], clean[[0, 4]])


@pytest.mark.gpu
def test_slices_shapes_and_negated_views():
    from metal_kernelops.cv import layernorm_residual
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 5, 1 + 2 * 77, generator=g).to(BF16).to(DEV)
    w, b = torch.randn(77, generator=g).to(DEV), torch.randn(77, generator=g).to(DEV)
    x, res = wide[..., 1:78], wide[..., 78:]
    want = layernorm_residual(x.contiguous(), w, b, res.contiguous())
    for got in (layernorm_residual(x, w, b, res), layernorm_residual(x.transpose(0, 1), w, b, res.transpose(0, 1))):
        got = [t if t.shape == x.shape else t.transpose(0, 1) for t in got]
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert torch.equal(layernorm_residual(torch._neg_view(x), w, b, res)[0], layernorm_residual(-x, w, b, res)[0])
    one = layernorm_residual(x[0, 0], w, b, res[0, 0])
    assert torch.equal(one[0], want[0][0, 0]) and torch.equal(one[1], want[1][0, 0])
    strided = torch.stack([w, b], -1)
    assert torch.equal(layernorm_residual(x, strided[:, 0], strided[:, 1], res)[0], want[0])
    lead = layernorm_residual(x[:1, :1].expand(2, 5, 77), w, b, res)[1]
    assert torch.equal(lead, (x[:1, :1].float() + res.float()).to(BF16))
    grid = torch.randn(1, 4, 6, 96, generator=g).to(DEV).requires_grad_(True)  # a map of positions, as a vision block has it
    out, stream = layernorm_residual(grid, torch.ones(96, device=DEV))
    assert stream is grid
    out.sum().backward()
    assert grid.grad.shape == grid.shape and grid.grad.abs().max() < 1e-4  # a constant gradient is taken out


@pytest.mark.gpu
def test_a_tensor_in_two_roles_and_broadcast_parameters():
    from metal_kernelops.cv import layernorm_residual
    p = problem(9, 130, F32, F32)
    d = to_dev(p)
    leaf = d["x"].clone().requires_grad_(True)
    one = torch.full((1,), 0.5, device=DEV, requires_grad=True)
    both = one.expand(130)
    out, stream = layernorm_residual(leaf, both, both, leaf)
    torch.autograd.backward([out, stream], [d["dout"], d["dstream"]])
    ds, dw, db = oracle.layernorm_residual_bwd(p["dout"], p["dstream"], 2 * p["x"].double(), torch.full((130,), 0.5))
    assert rel(leaf.grad, 2 * ds) <= 2e-6
    assert abs(one.grad.item() - (dw.sum() + db.sum()).item()) <= 1e-6 * (dw.norm() + db.norm()).item() * 130 ** 0.5
    x, r = d["x"].clone().requires_grad_(True), d["residual"].clone().requires_grad_(True)
    layernorm_residual(x, d["weight"], d["bias"], r)[0].sum().backward()
    before = r.grad.clone()
    x.grad.add_(1.0)  # one gradient for both, but not one tensor
    assert torch.equal(r.grad, before)


@pytest.mark.gpu
@pytest.mark.parametrize("features", [96, 1536, 40000])
def test_results_repeat_and_do_not_depend_on_old_memory(features):
    d = to_dev(problem(300 if features > 2000 else 3000, features, BF16, BF16))
    leaves = [d[n].requires_grad_(True) for n in NAMES]

    def run(fill):
        before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
        torch.use_deterministic_algorithms(fill)
        torch.utils.deterministic.fill_uninitialized_memory = fill
        try:
            out, stream = call(d)
            return [out, stream, *torch.autograd.grad([out, stream], leaves, [d["dout"], d["dstream"]])]
        finally:
            torch.use_deterministic_algorithms(before[0])
            torch.utils.deterministic.fill_uninitialized_memory = before[1]

    for a, b, c in zip(run(False), run(True), run(False)):
        assert torch.isfinite(b.float()).all() and torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_empty_sizes():
    from metal_kernelops.cv import layernorm_residual
    for shape in ((0, 8), (3, 0), (2, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
        out, stream = layernorm_residual(x, w, b, torch.zeros(shape, device=DEV))
        assert out.shape == shape and stream.shape == shape
        gx, gw, gb = torch.autograd.grad(out.sum() + stream.sum(), (x, w, b))
        assert gx.shape == shape and (gw == 0).all() and (gb == 0).all()


@pytest.mark.gpu
def test_captured_graph_replays():
    d = to_dev(problem(700, 520, BF16, BF16))
    leaves = [d[n].requires_grad_(True) for n in NAMES]

    def step():
        out, stream = call(d)
        return (out, stream, *torch.autograd.grad([out, stream], leaves, [d["dout"], d["dstream"]]))

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
            d["x"].copy_(torch.randn(d["x"].shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows beyond 2^32 bytes against the same rows alone.  How a row is split over lanes goes by the number of
    rows, so two calls on the same row are each within the tolerance of the exact one: twice that apart."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(900_000, 2560, dtype=BF16, device=DEV).normal_(generator=g).requires_grad_(True)
    w, b = torch.full((2560,), 1.5, device=DEV), torch.full((2560,), 0.5, device=DEV)
    tail = x.detach()[-50:].clone().requires_grad_(True)
    out, stream = call({"x": x, "weight": w, "bias": b, "residual": x.detach()})
    last, last_stream = call({"x": tail, "weight": w, "bias": b, "residual": tail.detach()})
    assert rel(out[-50:], last) <= 2 * TOL[BF16] and torch.equal(stream[-50:], last_stream)
    dx, = torch.autograd.grad(out, x, x.detach())
    dlast, = torch.autograd.grad(last, tail, tail.detach())
    # the gradient of a row along itself is taken out but for eps: what is left of terms r dout w, here
    # 0.5 * 1.5 |x|, is their float32 roundings, 8 * 2^-24 of the largest in each call; a row read elsewhere gives
    # the terms themselves
    largest = 0.75 * tail.detach().abs().max().item()
    assert (dx[-50:] - dlast).abs().max().item() <= 2 * 8 * 2.0 ** -24 * largest * 1.1
    assert dlast.abs().max().item() <= 1e-4 * largest


@pytest.mark.gpu
def test_a_second_derivative_and_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwd
    d = to_dev(problem(3, 40, F32, F32))
    x = d["x"].clone().requires_grad_(True)
    grad, = torch.autograd.grad(call({**d, "x": x})[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), x)
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        call({**d, "x": fwd.make_dual(d["x"], d["x"])})


@pytest.mark.gpu
def test_refusals():
    from metal_kernelops.cv import layernorm_residual
    x, w = torch.zeros(2, 8, device=DEV), torch.ones(8, device=DEV)
    for args in [(x, w[:7]), (x, w, w[:7]), (x, w, w, x[:1]), (x.cpu(), w.cpu()), (x, w.cpu()), (x, w, w.cpu()),
                 (x, w, w, x.cpu()), (x.double(), w), (x, w.double()), (x, w, w.double()), (x, w, w, x.half()),
                 (x.half(), w, w, x.to(BF16)), (torch.zeros((), device=DEV), w)]:
        with pytest.raises(ValueError):
            layernorm_residual(*args)
