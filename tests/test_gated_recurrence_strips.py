"""Gated linear recurrence at the kernels' own seams: whole strips of 128 channels, which take the vector
loads and stores, in every type; lengths and resets around a wavefront's run of 8 steps and a chunk's
64; and gradients against differences of the forward.

Tolerances as in ``test_gated_recurrence.py``: 1e-5 of the global norm in float32, beside half a unit of a
16-bit output."""

import pytest
import torch

from oracle import recurrent_layer as oracle
from test_gated_recurrence import DEV, DTYPES, F32_TOL, check, problem, rel, run_grads, to_dev

LENGTHS = [7, 8, 9, 63, 64, 65, 129]
EDGES = (0, 7, 8, 63, 64, 65, 127, 128)


def with_edges(p):
    """Resets on both sides of every seam."""
    batch, length, _ = p["x"].shape
    p["reset"] = torch.zeros(batch, length, dtype=torch.bool)
    for t in EDGES:
        if t < length:
            p["reset"][t % batch, t] = True
            p["reset"][-1, t] = True
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("reset", [None, "edges", "all"])
@pytest.mark.parametrize("initial", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [128, 256, 384])
def test_whole_strips(channels, dtype, initial, reset):
    for length in (1, 65, 200):
        p = problem(3, length, channels, dtype, initial=initial, reset="all" if reset == "all" else None)
        check(with_edges(p) if reset == "edges" else p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [72, 128])
@pytest.mark.parametrize("length", LENGTHS)
def test_lengths_around_a_run_and_a_chunk(length, channels, dtype):
    check(problem(2, length, channels, dtype))
    check(with_edges(problem(2, length, channels, dtype, seed=1)))


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [72, 128])
@pytest.mark.parametrize("at", EDGES)
def test_one_reset_at_a_seam(at, channels):
    """A single reset, and in the other sequence a NaN just before it that must not pass."""
    p = problem(2, 140, channels, torch.float32)
    p["reset"] = torch.zeros(2, 140, dtype=torch.bool)
    p["reset"][:, at] = True
    check(p)
    if at:
        clean = run_grads(p)
        p["x"][1, at - 1] = float("nan")
        got = run_grads(p)
        assert torch.equal(got[0][:, at:], clean[0][:, at:]) and torch.equal(got[0][0], clean[0][0])
        assert torch.isnan(got[0][1, at - 1]).all()
        for name in ("x", "input_gate", "decay_gate"):
            assert torch.equal(got[2][name][:, at:], clean[2][name][:, at:]), name


@pytest.mark.gpu
@pytest.mark.parametrize("use", [("y",), ("final",)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_whole_strips_with_one_output_used(dtype, use):
    check(problem(2, 150, 128, dtype, initial=False), use)
    check(problem(2, 150, 128, dtype, reset="some"), use)


@pytest.mark.gpu
def test_extreme_gates_in_whole_strips():
    """Gates at +-100 and the infinities, as in the narrow strips' test."""
    p = problem(2, 140, 128, torch.float32)
    for i, v in enumerate((100.0, -100.0, float("inf"), -float("inf"), -30.0, 12.0)):
        p["decay_gate"][:, i::7] = v
        p["input_gate"][:, :, i::9] = v
    p["decay"][:8] = torch.tensor([30.0, 21.0, 19.0, -40.0, -80.0, 5.0, 0.0, -10.0])
    y, final, grads = run_grads(p)
    args = [p[k] for k in ("x", "input_gate", "decay_gate", "decay", "initial", "reset")]
    want_y, want_final = oracle.gated_recurrence(*args)
    want = oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *args)
    assert rel(y, want_y) <= F32_TOL and rel(final, want_final) <= F32_TOL
    for name, w in zip(("x", "input_gate", "decay_gate", "decay", "initial"), want):
        assert torch.isfinite(grads[name]).all(), name
        if name != "decay":  # a held step's term of ddecay is a limit whose value m = 0 leaves open
            assert rel(grads[name], w) <= F32_TOL, name


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["x", "dy"])
def test_nan_stays_in_its_document_in_whole_strips(where):
    p = problem(2, 300, 256, torch.float32)
    p["reset"] = torch.zeros(2, 300, dtype=torch.bool)
    p["reset"][:, 64] = p["reset"][:, 200] = True
    clean = run_grads(p)
    p[where][0, 130, :200] = float("nan")
    p[where][0, 131, 200:] = float("inf")
    got = run_grads(p)
    for s in (slice(0, 64), slice(200, 300)):
        assert torch.equal(got[0][:, s], clean[0][:, s])
        for n in ("x", "input_gate", "decay_gate"):
            assert torch.equal(got[2][n][:, s], clean[2][n][:, s]), n
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0][1], clean[0][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_of_one_projection_at_odd_offsets(dtype):
    """Whole strips read in place from rows that no vector load is aligned to."""
    from metal_kernelops.cv import gated_recurrence
    wide = torch.randn(2, 100, 3 * 128 + 1, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    decay = torch.randn(128, generator=torch.Generator().manual_seed(3)).to(DEV) - 3
    parts = [wide[..., 1 + 128 * i:129 + 128 * i] for i in range(3)]
    assert torch.equal(gated_recurrence(*parts, decay), gated_recurrence(*(t.contiguous() for t in parts), decay))


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [48, 128])
def test_gradients_against_differences(channels):
    """Central differences of the kernel's own float32 forward, summed in float64, against its gradients.

    With a step s in the direction e the difference is the derivative, plus a truncation error that the
    float64 oracle's own difference at the same points gives, plus rounding.  Rounding: over the 150
    steps here an output is off by sqrt(150) * 4 * 2^-24 = 3e-6 of itself, independently from output to
    output and on both sides, so the difference by sqrt(2) * 3e-6 / (2 s) of |dy y|; four times that,
    at s = 1/8, is 7e-5 of the norm of dy * y.  The gradients themselves may be off by 1e-5 of their
    norm: four times that of grad * e."""
    from metal_kernelops.cv import gated_recurrence
    step = 2.0 ** -3
    p = problem(1, 150, channels, torch.float32)
    y, final, grads = run_grads(p)
    names = ("x", "input_gate", "decay_gate", "decay", "initial")
    d = to_dev(p)

    def weighed(out, last, q):
        return (out.double() * q["dy"].double()).sum().item() + (last.double() * q["dfinal"].double()).sum().item()

    def loss(v):
        out = gated_recurrence(v["x"], v["input_gate"], v["decay_gate"], v["decay"], initial_state=v["initial"],
                               return_final_state=True)
        return weighed(*out, d)

    def exact_loss(v):
        return weighed(*oracle.gated_recurrence(*(v[n] for n in names)), p)

    want = dict(zip(names, oracle.gated_recurrence_bwd(p["dy"], p["dfinal"], *(p[n] for n in names))))
    terms = ((y.detach().cpu().double() * p["dy"]).square().sum() + (final.detach().cpu().double() * p["dfinal"]).square().sum()) ** 0.5
    g = torch.Generator().manual_seed(9)
    for n in names:
        e = torch.randn(p[n].shape, generator=g)
        # both sides see the same float32 points
        up, down = p[n] + step * e, p[n] - step * e
        e = (up.double() - down.double()) / (2 * step)
        got = (loss({**d, n: up.to(DEV)}) - loss({**d, n: down.to(DEV)})) / (2 * step)
        exact = (exact_loss({**p, n: up}) - exact_loss({**p, n: down})) / (2 * step)
        truncation = exact - (want[n] * e).sum().item()
        along = grads[n].cpu().double() * e
        bound = 7e-5 * terms.item() + 4e-5 * along.norm().item()
        assert abs(got - along.sum().item() - truncation) <= bound, n
