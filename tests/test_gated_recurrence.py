"""Gated linear recurrence: oracle pins on the CPU, HIP parity on the GPU.

Tolerances.  Float32, relative error of the global norm: a step multiplies the state by a decay
computed to a few units of 2^-24, errors that differ from step to step; over the memory of the
longest channels here (a = 0.999, a thousand steps) they add to sqrt(1000) * 4 * 2^-24 = 8e-6, so
1e-5; the sums of ddecay have the same terms.  16-bit outputs add their rounding, of relative norm
at most half a unit in the last place: 2^-11 for float16 and 2^-8 for bfloat16.
"""

import pytest
import torch

from oracle import recurrent_layer as oracle

DEV = "cuda"
F32_TOL = 1e-5
TOL = {torch.float32: F32_TOL, torch.float16: F32_TOL + 2.0 ** -11, torch.bfloat16: F32_TOL + 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# one step, one channel; lengths around two chunks of 64 steps and their fractions; many chunks;
# channel counts around a wavefront's and odd ones
SHAPES = [(1, 1, 1), (2, 1, 64), (1, 2, 130), (3, 15, 65), (2, 127, 3), (1, 128, 64), (2, 129, 129), (1, 257, 200),
          (5, 64, 31), (2, 1000, 77), (1, 4500, 40)]


def problem(batch, length, channels, dtype, seed=0, initial=True, reset=None):
    g = torch.Generator().manual_seed(seed * 1000 + batch + length + channels)

    def r(*shape):
        return torch.randn(shape, generator=g)

    rate = -torch.log(torch.rand(channels, generator=g) * 0.099 + 0.9) / 8.0
    p = {"x": r(batch, length, channels).to(dtype), "input_gate": r(batch, length, channels).to(dtype),
         "decay_gate": r(batch, length, channels).to(dtype), "decay": torch.log(torch.expm1(rate)),
         "initial": r(batch, channels) if initial else None, "reset": None,
         "dy": r(batch, length, channels).to(dtype), "dfinal": r(batch, channels)}
    if reset == "some":
        p["reset"] = torch.rand(batch, length, generator=g) < 0.05
    elif reset == "edges":  # the first and last step, and both sides of the chunks' ends
        p["reset"] = torch.zeros(batch, length, dtype=torch.bool)
        for t in (0, 15, 16, 127, 128, 255, 256, length - 1):
            if t < length:
                p["reset"][:, t] = True
    elif reset == "all":
        p["reset"] = torch.ones(batch, length, dtype=torch.bool)
    return p


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    scale = want.norm().item()
    return (got - want).norm().item() / (scale if scale else 1.0)


def to_dev(p):
    return {k: None if v is None else v.to(DEV) for k, v in p.items()}


def run_grads(p, use=("y", "final")):
    """Outputs and gradients of the public function on the GPU."""
    from metal_kernelops.cv import gated_recurrence
    d = to_dev(p)
    names = [n for n in ("x", "input_gate", "decay_gate", "decay", "initial") if d[n] is not None]
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in names}
    y, final = gated_recurrence(leaves["x"], leaves["input_gate"], leaves["decay_gate"], leaves["decay"],
                                initial_state=leaves.get("initial"), reset=d["reset"], return_final_state=True)
    outs = {"y": (y, d["dy"]), "final": (final, d["dfinal"])}
    grads = torch.autograd.grad([outs[u][0] for u in use], list(leaves.values()), [outs[u][1] for u in use])
    return y, final, dict(zip(names, grads))


def check(p, use=("y", "final")):
    y, final, grads = run_grads(p, use)
    args = [p[k] for k in ("x", "input_gate", "decay_gate", "decay", "initial", "reset")]
    want_y, want_final = oracle.gated_recurrence(*args)
    dtype = p["x"].dtype
    assert rel(y, want_y) <= TOL[dtype]
    assert rel(final, want_final) <= F32_TOL
    dy = p["dy"] if "y" in use else torch.zeros_like(p["dy"])
    want = oracle.gated_recurrence_bwd(dy, p["dfinal"] if "final" in use else None, *args)
    for name, w in zip(("x", "input_gate", "decay_gate", "decay", "initial"), want):
        if name in grads:
            tol = TOL[dtype] if name in ("x", "input_gate", "decay_gate") else F32_TOL
            assert rel(grads[name], w) <= tol, name


# --------------------------------------------------------------------------- CPU: oracle pins


@pytest.mark.parametrize("reset", [None, "some", "edges", "all"])
@pytest.mark.parametrize("initial", [False, True])
def test_oracle_backward_equals_autograd(reset, initial):
    p = problem(2, 21, 5, torch.float64, initial=initial, reset=reset)
    leaves = [p[k].double().requires_grad_(True) for k in ("x", "input_gate", "decay_gate", "decay")]
    h0 = p["initial"].double().requires_grad_(True) if initial else None
    y, final = oracle.gated_recurrence(*leaves, h0, p["reset"])
    loss = (y * p["dy"]).sum() + (final * p["dfinal"]).sum()
    want = torch.autograd.grad(loss, leaves + ([h0] if initial else []))
    got = oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *[t.detach() for t in leaves],
                                      None if h0 is None else h0.detach(), p["reset"])
    for a, b in zip(got, want):
        assert (a - b).abs().max() < 1e-12


def test_oracle_backward_equals_central_differences():
    p = problem(1, 9, 2, torch.float64, reset="some")
    args = [p[k].double() for k in ("x", "input_gate", "decay_gate", "decay", "initial")]
    got = oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *args, p["reset"])

    def loss(values):
        y, final = oracle.gated_recurrence(*values, p["reset"])
        return (y * p["dy"]).sum() + (final * p["dfinal"]).sum()

    step = 1e-6
    for k, value in enumerate(args):
        for i in range(0, value.numel(), 3):
            e = torch.zeros(value.numel(), dtype=torch.float64)
            e[i] = step
            e = e.reshape(value.shape)
            up = loss([v + e if j == k else v for j, v in enumerate(args)])
            down = loss([v - e if j == k else v for j, v in enumerate(args)])
            assert abs((up - down) / (2 * step) - got[k].reshape(-1)[i]) < 1e-6


@pytest.mark.parametrize("reset", [None, "some"])
def test_reference_twins_match_the_oracle(reset):
    from metal_kernelops.cv import gated_recurrence_reference, gated_recurrence_update_reference
    p = problem(2, 13, 6, torch.float64, reset=reset)
    args = [p[k].double() for k in ("x", "input_gate", "decay_gate", "decay")]
    y, final = gated_recurrence_reference(*args, initial_state=p["initial"].double(), reset=p["reset"],
                                          return_final_state=True)
    want, want_final = oracle.gated_recurrence(*args, p["initial"], p["reset"])
    assert (y - want).abs().max() < 1e-12 and (final - want_final).abs().max() < 1e-12
    if reset is None:
        h = p["initial"].double()
        for t in range(13):
            step, h = gated_recurrence_update_reference(h, args[0][:, t], args[1][:, t], args[2][:, t], args[3])
            assert (step - want[:, t]).abs().max() < 1e-12
    assert gated_recurrence_reference(*(a[:, :0] for a in args[:3]), args[3]).shape == (2, 0, 6)


def test_native_argument_checks_without_a_gpu():
    import ctypes

    from metal_kernelops import _native as nat
    lib = nat.lib()
    p = nat.RecurParams(batch=1, length=4, channels=8, dtype=3, scale=8.0)
    assert lib.mko_recur_fwd(ctypes.byref(p), None) == 1 and b"dtype" in lib.mko_last_error()
    p.dtype = 0
    assert lib.mko_recur_fwd(ctypes.byref(p), None) == 1  # no pointers
    assert lib.mko_recur_bwd(ctypes.byref(p), None) == 1
    p.length = -1
    assert lib.mko_recur_fwd(ctypes.byref(p), None) == 1 and b"negative" in lib.mko_last_error()
    p.length = 0
    assert lib.mko_recur_fwd(ctypes.byref(p), None) == 0 and lib.mko_recur_bwd(ctypes.byref(p), None) == 0
    u = nat.RecurUpdateParams(batch=1, channels=8, dtype=0, state_dtype=9)
    assert lib.mko_recur_update(ctypes.byref(u), None) == 1


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    check(problem(*shape, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("reset", ["some", "edges", "all"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 129, 66), (2, 700, 33)])
def test_resets(shape, dtype, reset):
    check(problem(*shape, dtype, reset=reset))


@pytest.mark.gpu
@pytest.mark.parametrize("use", [("y",), ("final",)])
def test_no_initial_state_and_one_output_used(use):
    check(problem(2, 300, 70, torch.float32, initial=False), use)
    check(problem(2, 300, 70, torch.bfloat16, initial=True), use)


@pytest.mark.gpu
@pytest.mark.parametrize("reset", [None, "some"])
def test_many_sequences_of_many_chunks(reset):
    """More workgroups than the chip holds at once, each waiting on the one before it."""
    check(problem(6, 1500, 1536, torch.bfloat16, reset=reset))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slices_broadcasts_and_offsets(dtype):
    """Slices of one projection, inputs broadcast over the batch, rows at odd offsets, and a
    transposed input, against the same values in dense tensors."""
    from metal_kernelops.cv import gated_recurrence
    b, length, c = 3, 200, 77
    g = torch.Generator().manual_seed(5)
    proj = torch.randn(b, length, 3 * c + 1, generator=g).to(dtype).to(DEV)
    decay = torch.randn(c, generator=g).to(DEV) - 3
    parts = [proj[..., 1 + i * c:1 + (i + 1) * c] for i in range(3)]
    want = gated_recurrence(*(t.contiguous() for t in parts), decay)
    assert torch.equal(gated_recurrence(*parts, decay), want)
    one = proj[:1, :, :c]
    dense = gated_recurrence(one.expand(b, -1, -1).contiguous(), *(t.contiguous() for t in parts[1:]), decay)
    leaf = one.detach().clone().requires_grad_(True)
    out = gated_recurrence(leaf.expand(b, -1, -1), *parts[1:], decay)
    assert torch.equal(out, dense)
    copy = one.expand(b, -1, -1).contiguous().requires_grad_(True)
    dy = torch.randn(b, length, c, generator=g).to(dtype).to(DEV)
    (gc,) = torch.autograd.grad(gated_recurrence(copy, *parts[1:], decay), copy, dy)
    (gl,) = torch.autograd.grad(out, leaf, dy)
    assert rel(gl, gc.double().sum(0, keepdim=True)) <= TOL[dtype] * 2
    turned = parts[0].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(gated_recurrence(turned, *parts[1:], decay), want)
    assert torch.equal(gated_recurrence(-parts[0], *parts[1:], decay),
                       gated_recurrence(torch._neg_view(parts[0]), *parts[1:], decay))
    by_dim = gated_recurrence(parts[0][..., :1].expand(-1, -1, c), *parts[1:], decay)
    assert torch.equal(by_dim, gated_recurrence(parts[0][..., :1].repeat(1, 1, c), *parts[1:], decay))


@pytest.mark.gpu
def test_extreme_gates():
    """Gates at +-100 and the infinities: a full decay, a full hold (m = 0), a closed input; every
    output and gradient is finite and the oracle's."""
    p = problem(2, 140, 64, torch.float32)
    for i, v in enumerate((100.0, -100.0, float("inf"), -float("inf"), -30.0, 12.0)):
        p["decay_gate"][:, i::7] = v
        p["input_gate"][:, :, i::9] = v
    p["decay"][:8] = torch.tensor([30.0, 21.0, 19.0, -40.0, -80.0, 5.0, 0.0, -10.0])
    y, final, grads = run_grads(p)
    args = [p[k] for k in ("x", "input_gate", "decay_gate", "decay", "initial", "reset")]
    want_y, _ = oracle.gated_recurrence(*args)
    want = oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *args)
    assert torch.isfinite(y).all() and rel(y, want_y) <= F32_TOL
    for name, w in zip(("x", "input_gate", "decay_gate", "decay", "initial"), want):
        assert torch.isfinite(grads[name]).all(), name
        if name != "decay":  # a held step's term of ddecay is a limit whose value m = 0 leaves open
            assert rel(grads[name], w) <= F32_TOL, name


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["x", "dy"])
def test_nan_stays_in_its_document(where):
    """A NaN or an infinity reaches no step of another document, forward or backward."""
    p = problem(2, 400, 70, torch.float32)
    p["reset"] = torch.zeros(2, 400, dtype=torch.bool)
    p["reset"][:, 150] = p["reset"][:, 290] = True
    clean = run_grads(p)
    p[where][0, 200, :35] = float("nan")
    p[where][0, 201, 35:] = float("inf")
    p["decay_gate"][0, 150] = float("nan") if where == "x" else p["decay_gate"][0, 150]
    got = run_grads(p)
    others = [slice(0, 150), slice(290, 400)]
    for s in others:
        assert torch.equal(got[0][:, s], clean[0][:, s])
        for n in ("x", "input_gate", "decay_gate"):
            assert torch.equal(got[2][n][:, s], clean[2][n][:, s]), n
    assert torch.equal(got[1], clean[1])
    if where == "x":
        assert not torch.isfinite(got[0][0, 201:290]).any()
    assert torch.equal(got[0][1], clean[0][1])


@pytest.mark.gpu
def test_a_nan_state_never_decays_away():
    """Without a reset a NaN stays in the state, however strong the decay."""
    from metal_kernelops.cv import gated_recurrence
    p = to_dev(problem(1, 600, 64, torch.float32))
    p["x"][0, 10, 3] = float("nan")
    p["decay_gate"] += 50.0
    p["decay"][:] = 10.0
    y = gated_recurrence(p["x"], p["input_gate"], p["decay_gate"], p["decay"])
    assert torch.isnan(y[0, 10:, 3]).all() and not torch.isnan(y[0, :, 4:]).any()


@pytest.mark.gpu
def test_runs_repeat_bit_for_bit():
    for dtype in (torch.float32, torch.bfloat16):
        p = problem(3, 900, 160, dtype, reset="some")
        a, b = run_grads(p), run_grads(p)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert all(torch.equal(a[2][k], b[2][k]) for k in a[2])


@pytest.mark.gpu
def test_a_sequence_in_pieces_is_the_sequence():
    """Prompt pieces with the state carried, then single tokens, against one call."""
    from metal_kernelops.cv import gated_recurrence, gated_recurrence_update
    p = to_dev(problem(2, 333, 90, torch.float32))
    args = [p[k] for k in ("x", "input_gate", "decay_gate")]
    want, want_final = gated_recurrence(*args, p["decay"], initial_state=p["initial"], return_final_state=True)
    state, out = p["initial"], []
    for lo, hi in ((0, 1), (1, 130), (130, 325)):
        y, state = gated_recurrence(*(t[:, lo:hi] for t in args), p["decay"], initial_state=state,
                                    return_final_state=True)
        out.append(y)
    for t in range(325, 333):
        y, state = gated_recurrence_update(state, *(a[:, t] for a in args), p["decay"], out_state=state)
        out.append(y[:, None])
    assert rel(torch.cat(out, 1), want) <= F32_TOL and rel(state, want_final) <= F32_TOL


@pytest.mark.gpu
def test_empty_sizes():
    from metal_kernelops.cv import gated_recurrence, gated_recurrence_update
    d = torch.zeros(4, device=DEV)
    for shape in ((2, 0, 4), (0, 3, 4)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        h0 = torch.randn(shape[0], 4, device=DEV, requires_grad=True)
        y, final = gated_recurrence(x, x, x, d, initial_state=h0, return_final_state=True)
        assert y.shape == shape and torch.equal(final, h0)
        gx, gh = torch.autograd.grad(y.sum() + final.sum(), (x, h0))
        assert gx.shape == shape and torch.equal(gh, torch.ones_like(h0))
    y, final = gated_recurrence(*(torch.zeros(2, 0, 4, device=DEV) for _ in range(3)), d, return_final_state=True)
    assert torch.equal(final, torch.zeros(2, 4, device=DEV))
    x = torch.zeros(2, 3, 0, device=DEV)
    assert gated_recurrence(x, x, x, torch.zeros(0, device=DEV)).shape == (2, 3, 0)
    x = torch.zeros(0, 4, device=DEV)
    assert gated_recurrence_update(x, x, x, x, d)[0].shape == (0, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("state_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 65), (2, 1001), (17, 256)])
def test_update(shape, dtype, state_dtype):
    from metal_kernelops.cv import gated_recurrence_update
    b, c = shape
    p = problem(b, 1, c, dtype)
    state = p["initial"].to(state_dtype)
    d = to_dev(p)
    dev_state = state.to(DEV)
    y, new = gated_recurrence_update(dev_state, *(d[k][:, 0] for k in ("x", "input_gate", "decay_gate")), d["decay"])
    want, _ = oracle.gated_recurrence(p["x"], p["input_gate"], p["decay_gate"], p["decay"], state)
    assert y.dtype == dtype and new.dtype == state_dtype
    assert rel(y, want[:, 0]) <= TOL[dtype] and rel(new, want[:, 0]) <= TOL[state_dtype]
    assert torch.equal(dev_state.cpu(), state)
    wide = torch.randn(b, 3 * c + 1, device=DEV).to(dtype)
    wide[:, 1:] = torch.cat([d[k][:, 0] for k in ("x", "input_gate", "decay_gate")], 1)
    parts = [wide[:, 1 + i * c:1 + (i + 1) * c] for i in range(3)]
    y2, new2 = gated_recurrence_update(dev_state, *parts, d["decay"], out_state=dev_state)
    assert new2 is dev_state and torch.equal(y2, y) and torch.equal(dev_state, new)


@pytest.mark.gpu
def test_update_differentiates_like_one_step():
    from metal_kernelops.cv import gated_recurrence_update
    p = problem(2, 1, 40, torch.float32)
    d = to_dev(p)
    leaves = [d["initial"], d["x"][:, 0], d["input_gate"][:, 0], d["decay_gate"][:, 0], d["decay"]]
    leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
    y, new = gated_recurrence_update(*leaves)
    grads = torch.autograd.grad([y, new], leaves, [d["dy"][:, 0], d["dfinal"]])
    args = [p[k] for k in ("x", "input_gate", "decay_gate", "decay", "initial")]
    dx, dig, drg, dd, dh = oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *args)
    for got, want in zip(grads, (dh, dx[:, 0], dig[:, 0], drg[:, 0], dd)):
        assert rel(got, want) <= F32_TOL


@pytest.mark.gpu
def test_gradients_against_differences_of_the_forward():
    """Central differences of the kernel's own float32 forward, summed in float64.  The truncation
    error is (2^-6)^2 of the third derivative, the rounding error the outputs' 2^-24 times sqrt of
    their number over the step, 3e-5 of the directional derivative's terms: 1e-3 of their norm."""
    from metal_kernelops.cv import gated_recurrence
    p = problem(1, 150, 48, torch.float32)
    y, final, grads = run_grads(p)
    d = to_dev(p)
    names = ("x", "input_gate", "decay_gate", "decay", "initial")

    def loss(v):
        out, last = gated_recurrence(v["x"], v["input_gate"], v["decay_gate"], v["decay"], initial_state=v["initial"],
                                     return_final_state=True)
        return ((out.double() * d["dy"].double()).sum() + (last.double() * d["dfinal"].double()).sum()).item()

    g = torch.Generator().manual_seed(9)
    for n in names:
        e = torch.randn(p[n].shape, generator=g).to(DEV)
        step = 2.0 ** -6
        up, down = dict(d), dict(d)
        up[n], down[n] = d[n] + step * e, d[n] - step * e
        got = (loss(up) - loss(down)) / (2 * step)
        want = (grads[n].double() * e.double()).sum().item()
        scale = (grads[n].double() * e.double()).norm().item() + abs(want)
        assert abs(got - want) <= 1e-2 * scale, n


@pytest.mark.gpu
def test_on_another_stream():
    from metal_kernelops.cv import gated_recurrence
    p = to_dev(problem(2, 500, 130, torch.bfloat16))
    args = [p[k] for k in ("x", "input_gate", "decay_gate", "decay")]
    want = gated_recurrence(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [gated_recurrence(*args) for _ in range(3)]
    here = [gated_recurrence(*args) for _ in range(3)]  # both streams at once
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs + here)


@pytest.mark.gpu
def test_captured_graph_replays():
    """Forward and backward in one captured graph, replayed with other work between, give the eager
    bits every time."""
    from metal_kernelops.cv import gated_recurrence
    p = to_dev(problem(2, 400, 96, torch.bfloat16, reset="some"))
    names = ("x", "input_gate", "decay_gate", "decay", "initial")
    leaves = [p[n].requires_grad_(True) for n in names]

    def step():
        y, final = gated_recurrence(*leaves[:4], initial_state=leaves[4], reset=p["reset"], return_final_state=True)
        return (y, final, *torch.autograd.grad([y, final], leaves, [p["dy"], p["dfinal"]]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            p["x"].copy_(torch.randn(p["x"].shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_refusals():
    from metal_kernelops.cv import gated_recurrence, gated_recurrence_update
    x = torch.zeros(2, 3, 4, device=DEV)
    d, h = torch.zeros(4, device=DEV), torch.zeros(2, 4, device=DEV)
    bad = [
        ((x[0], x, x, d), {}), ((x, x[:1], x, d), {}), ((x, x, x[..., :3], d), {}), ((x, x, x, d[:3]), {}),
        ((x.cpu(), x.cpu(), x.cpu(), d.cpu()), {}), ((x, x.cpu(), x, d), {}), ((x, x.half(), x, d), {}),
        ((x.double(), x.double(), x.double(), d), {}), ((x, x, x, d.int()), {}), ((x, x, x, d), {"scale": 0.0}),
        ((x, x, x, d), {"initial_state": h[:1]}), ((x, x, x, d), {"initial_state": h.int()}),
        ((x, x, x, d), {"reset": torch.zeros(2, 3, device=DEV)}),
        ((x, x, x, d), {"reset": torch.zeros(2, 4, dtype=torch.bool, device=DEV)}),
        ((x, x, x, d), {"reset": torch.zeros(2, 3, dtype=torch.bool)}),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError, match="gated_recurrence|ROCm GPU"):
            gated_recurrence(*args, **kw)
    r = x[:, 0]
    for args, kw in [((h[:1], r, r, r, d), {}), ((h.double(), r, r, r, d), {}), ((h, x, x, x, d), {}),
                     ((h, r, r.half(), r, d), {}), ((h, r, r, r, d), {"out_state": h.half()}),
                     ((h, r, r, r, d), {"out_state": torch.zeros(2, 8, device=DEV)[:, ::2]}),
                     ((h, r, r, r, d), {"out_state": h.clone().requires_grad_(True)})]:
        with pytest.raises(ValueError, match="gated_recurrence_update"):
            gated_recurrence_update(*args, **kw)
    y = gated_recurrence(x.clone().requires_grad_(True), x, x, d)
    (g,) = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
