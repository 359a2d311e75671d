"""The gated delta rule and its one-token update: oracle pins and refusals on the CPU, HIP parity on the GPU.

Tolerances, relative error of the global norm, with u half a unit in the last place (2^-8 for
bfloat16, 2^-11 for float16).  In 16 bits the forward rounds S, V - K S^T, T, P, E, the weighted E and
the output, seven operands of contractions whose terms are about as large as their sums: 8 u.  The
backward adds the saved S and E, G, dE, X, the decayed dY and X, dP and dA: 16 u.  Float32 products
of at most 256 keys and 64 tokens, carried from chunk to chunk by a state that forgets: 1e-5, as the
other recurrences have it.  The one-token update computes in float32 and rounds twice: 1e-6 and u.
"""

import ctypes

import pytest
import torch

from oracle import delta_rule as oracle

DEV = "cuda"
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
FWD = {F32: 1e-5, F16: 8 * U[F16], BF16: 8 * U[BF16]}
BWD = {F32: 1e-5, F16: 16 * U[F16], BF16: 16 * U[BF16]}
NAMES = ("q", "k", "v", "log_decay", "beta", "initial")


def problem(batch, length, key_heads, heads, key, value, dtype=F32, initial=True, seed=0, gates=None, state=None):
    """Keys of norm one, a state that keeps 0.9 to 0.999 a token, and both outputs' gradients."""
    g = torch.Generator().manual_seed(1000 * seed + 7 * length + key + value)

    def r(*shape):
        return torch.randn(shape, generator=g)

    def unit(*shape):
        return torch.nn.functional.normalize(r(*shape), dim=-1).to(dtype)

    rate = -torch.log(0.9 + 0.099 * torch.rand(heads, generator=g))
    p = {"q": unit(batch, length, key_heads, key), "k": unit(batch, length, key_heads, key),
         "v": r(batch, length, heads, value).to(dtype),
         "log_decay": (-rate * (0.5 + torch.rand(batch, length, heads, generator=g))).to(gates or dtype),
         "beta": torch.sigmoid(r(batch, length, heads)).to(gates or dtype),
         "initial": (0.3 * r(batch, heads, value, key)).to(state or dtype) if initial else None}
    p["dy"], p["dfinal"] = r(batch, length, heads, value).to(dtype), (0.1 * r(batch, heads, value, key)).to(
        (state or dtype) if initial else dtype)
    return p


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    scale = want.norm().item()
    if scale < 2.0 ** -126:  # below float32's normal numbers: a gradient through 1500 tokens of decays, each 0.9 to
        want, scale = torch.zeros_like(want), 0.0  # 0.999, is exp(-75) to exp(-150), and zero where it has no number
    return (got - want).norm().item() / (scale if scale else 1.0)


def to_dev(p):
    return {k: None if v is None else v.to(DEV) for k, v in p.items()}


def call(d, final=True, **kw):
    from metal_kernelops.cv import gated_delta_rule
    return gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["initial"], return_final_state=final, **kw)


def gradients(d, use=("y", "final"), **kw):
    """Outputs and the gradients of what is there."""
    d = dict(d)
    leaves = {n: d[n].detach().requires_grad_(True) for n in NAMES if d[n] is not None}
    d.update(leaves)
    outs = dict(zip(("y", "final"), call(d, **kw)))
    dys = {"y": d["dy"], "final": d["dfinal"]}
    grads = torch.autograd.grad([outs[n] for n in use], list(leaves.values()), [dys[n] for n in use])
    return outs, dict(zip(leaves, grads))


def check(p, use=("y", "final"), scale=None, times=1):
    """Inference, the training forward and every gradient against the oracle; ``times`` the tolerances."""
    dtype, d = p["q"].dtype, to_dev(p)
    fwd, bwd = times * FWD[dtype], times * BWD[dtype]
    args = [p[n] for n in NAMES[:5]]
    y, final = oracle.gated_delta_rule(*args, scale=scale, initial=p["initial"])
    with torch.no_grad():
        plain_y, plain_final = call(d, scale=scale)
    assert plain_y.dtype == dtype and plain_final.dtype == p["dfinal"].dtype
    assert rel(plain_y, y) <= fwd and rel(plain_final, final) <= fwd + U[p["dfinal"].dtype]
    outs, grads = gradients(d, use, scale=scale)
    assert torch.equal(outs["y"], plain_y) and torch.equal(outs["final"], plain_final)
    want = oracle.gated_delta_rule_bwd(p["dy"] if "y" in use else torch.zeros_like(p["dy"]),
                                       p["dfinal"] if "final" in use else None, *args, scale=scale, initial=p["initial"])
    for name, w in zip(NAMES, want):
        if name in grads:
            assert grads[name].dtype == p[name].dtype
            assert rel(grads[name], w) <= bwd + U[p[name].dtype], name


# --------------------------------------------------------------------------- CPU: oracle pins and refusals


def test_oracle_gradients_equal_autograd_and_differences():
    p = {n: t.to(F64) for n, t in problem(2, 9, 1, 2, 5, 4).items()}
    args = {n: p[n].requires_grad_(True) for n in NAMES}

    def loss(a):
        y, final = oracle.gated_delta_rule(*(a[n] for n in NAMES[:5]), initial=a["initial"])
        return (y * p["dy"]).sum() + (final * p["dfinal"]).sum()

    want = torch.autograd.grad(loss(args), list(args.values()))
    got = oracle.gated_delta_rule_bwd(p["dy"], p["dfinal"], *(args[n] for n in NAMES[:5]), initial=args["initial"])
    g = torch.Generator().manual_seed(5)
    for name, a, b in zip(NAMES, got, want):
        assert rel(a, b) < 1e-12, name
        d, step = torch.randn(b.shape, generator=g, dtype=F64), 1e-5
        ends = [loss({**args, name: args[name] + s * step * d}) for s in (1, -1)]
        assert abs((ends[0] - ends[1]).item() / (2 * step) - (b * d).sum().item()) < 1e-7 * (1 + b.norm().item()), name


def test_reference_twins_match_the_oracle():
    from metal_kernelops.cv import gated_delta_rule_reference, gated_delta_rule_update_reference
    p = {n: t.double() for n, t in problem(2, 11, 2, 4, 6, 5).items()}
    args = [p[n] for n in NAMES[:5]]
    want = oracle.gated_delta_rule(*args, initial=p["initial"])
    got = gated_delta_rule_reference(*args, initial_state=p["initial"], return_final_state=True)
    assert all(rel(a, b) < 1e-12 for a, b in zip(got, want))
    want = oracle.gated_delta_rule(*(a[:, :1] for a in args), scale=0.5, initial=p["initial"])
    got = gated_delta_rule_update_reference(p["initial"], *(a[:, 0] for a in args), scale=0.5)
    assert rel(got[0], want[0][:, 0]) < 1e-12 and rel(got[1], want[1]) < 1e-12
    assert gated_delta_rule_reference(*(a[:, :0] for a in args)).shape == (2, 0, 4, 5)


def _params(**kw):
    """A problem of two chunks at made-up addresses."""
    from metal_kernelops import _native as nat
    names = ("q", "k", "v", "log_decay", "beta", "y", "saved", "dy", "dq", "dk", "dv", "dlog_decay", "dbeta", "workspace")
    at = {n: 1 << 20 for n in names}
    return nat.DeltaParams(**{**at, "workspace_bytes": 1 << 40, "batch": 1, "length": 65, "key_heads": 1, "heads": 2, "key": 8,
                              "value": 8, **kw})


@pytest.mark.parametrize("name", ["mko_delta_fwd", "mko_delta_bwd"])
@pytest.mark.parametrize("kw,status,text", [
    ({"batch": -1}, 1, b"negative"), ({"dtype": 9}, 1, b"dtypes"), ({"state_dtype": 7}, 1, b"dtypes"),
    ({"key_heads": 0}, 1, b"key_heads"), ({"key_heads": 2, "heads": 3}, 1, b"key_heads"), ({"key": 0}, 1, b"key"),
    ({"key": 257}, 3, b"at most"), ({"workspace_bytes": 64}, 2, b"workspace"), ({"q": None}, 1, b"required"),
    ({"workspace": (1 << 20) + 8}, 1, b"16 bytes"), ({"saved": (1 << 20) + 4}, 1, b"16 bytes"),
    ({"length": 1 << 30}, 3, b"2^24"), ({"batch": 1 << 12, "heads": 1 << 12}, 3, b"2^24"),
    ({"batch": 1 << 40, "heads": 1 << 40}, 3, b"2^24"), ({"length": 1 << 29, "batch": 2}, 3, b"2^24"),
    ({"value": 1 << 19, "heads": 1 << 9}, 3, b"2^24"),
])
def test_c_entries_refuse(name, kw, status, text):
    from metal_kernelops import _native as nat
    lib = nat.lib()
    got = getattr(lib, name)(ctypes.byref(_params(**kw)), None)
    names = {1: "MKO_EINVAL", 2: "MKO_EWORKSPACE", 3: "MKO_EUNSUPPORTED"}
    assert got != 0 and text in lib.mko_last_error(), (names[status], lib.mko_last_error())


def test_c_update_refuses():
    from metal_kernelops import _native as nat
    lib = nat.lib()
    at = {n: 1 << 20 for n in ("q", "k", "v", "log_decay", "beta", "state", "new_state", "y")}
    good = {**at, "batch": 2, "key_heads": 1, "heads": 2, "key": 8, "value": 8}
    for kw, text in [({"key": 257}, b"at most"), ({"heads": 3, "key_heads": 2}, b"key_heads"), ({"y": None}, b"required"),
                     ({"batch": -2}, b"negative"), ({"dtype": 5}, b"dtypes"), ({"value": 1 << 26}, b"2^24"),
                     ({"batch": 1 << 40, "heads": 1 << 40}, b"2^24")]:
        assert lib.mko_delta_update(ctypes.byref(nat.DeltaUpdateParams(**{**good, **kw})), None) != 0
        assert text in lib.mko_last_error()
    assert lib.mko_delta_update(ctypes.byref(nat.DeltaUpdateParams(**{**good, "batch": 0})), None) == 0


def test_sizes_agree_with_the_fake_op():
    """What a trace allocates for the saved tensor is what the library asks for."""
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_delta
    from torch._subclasses.fake_tensor import FakeTensorMode
    for dtype in (F32, BF16):
        for b, l, hk, h, k, v in [(1, 1, 1, 1, 1, 1), (2, 130, 2, 6, 33, 50), (1, 64, 1, 2, 128, 128)]:
            want = gated_delta._sizes(b, l, hk, h, k, v, nat.code(dtype), True)[0]
            with FakeTensorMode():
                a = [torch.empty(s, dtype=dtype, device=DEV) for s in ((b, l, hk, k), (b, l, hk, k), (b, l, h, v), (b, l, h),
                                                                       (b, l, h))]
                saved = torch.ops.mko.delta_fwd(*a, None, 1.0, False, True)[2]
            assert saved.numel() == want


def test_cpu_tensors_and_shapes_are_refused():
    from metal_kernelops.cv import gated_delta_rule, gated_delta_rule_update
    p = problem(2, 5, 2, 4, 8, 6)
    args = [p[n] for n in NAMES[:5]]
    with pytest.raises(ValueError, match="GPU"):
        gated_delta_rule(*args)
    with pytest.raises(ValueError, match="GPU"):
        gated_delta_rule_update(p["initial"], *(a[:, 0] for a in args))
    bad = [(0, args[0][0]), (1, args[1][..., :7]), (1, args[1][:, :4]), (2, args[2][:1]), (2, args[2][:, :, :3]),
           (2, args[2][:, :, 0]), (3, args[3][..., :1]), (4, args[4][:, 1:]), (0, torch.zeros(2, 5, 2, 0)),
           (0, torch.zeros(2, 5, 2, 257))]
    for i, t in bad:
        with pytest.raises(ValueError):
            gated_delta_rule(*(t if j == i or (j == 1 and i == 0 and t.dim() == 4) else a for j, a in enumerate(args)))


def _update_without_a_launch(monkeypatch, seen):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_delta
    monkeypatch.setattr(nat, "launch", lambda name, p, device: seen.append((name, p)))
    monkeypatch.setattr(gated_delta, "_require_gpu", lambda t: None)


@pytest.mark.parametrize("shift", [0, 1, -1, 3])
def test_an_update_in_place(monkeypatch, shift):
    """The version moves, and a destination shifted against its state is not read by the kernel."""
    from metal_kernelops.cv import gated_delta_rule_update
    seen = []
    _update_without_a_launch(monkeypatch, seen)
    buffer, one = torch.zeros(9, 2, 4, 8), torch.zeros(3, 2, 8)
    state, out = buffer[3:6], buffer[3 + shift:6 + shift]
    before = out._version
    y, new = gated_delta_rule_update(state, one, one, one[..., :4], one[..., 0], one[..., 0], out_state=out)
    assert new is out and out._version > before
    p = seen[0][1]
    assert p.new_state == out.data_ptr() and (p.state == state.data_ptr()) == (shift in (0, 3))


@pytest.mark.parametrize("alias", ["itself", "data", "none"])
def test_a_recorded_update_keeps_the_entering_state(monkeypatch, alias):
    from metal_kernelops.cv import gated_delta_rule_update
    seen = []
    _update_without_a_launch(monkeypatch, seen)
    state, one = torch.zeros(3, 2, 4, 8), torch.zeros(3, 2, 8, requires_grad=True)
    if alias != "itself":
        state.requires_grad_(True)
    out = {"itself": state, "data": state.data, "none": None}[alias]
    y, new = gated_delta_rule_update(state, one, one, one[..., :4], one[..., 0], one[..., 0], out_state=out)
    y.sum().backward()
    assert [name for name, _ in seen] == ["mko_delta_fwd", "mko_delta_bwd"]
    assert seen[0][1].initial and (out is None or seen[0][1].initial != out.data_ptr())
    assert one.grad is not None


# --------------------------------------------------------------------------- GPU: parity


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 129, 500])
def test_lengths(length, dtype):
    check(problem(2, length, 1, 2, 64, 48, dtype, initial=length % 2 == 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("key,value", [(1, 1), (7, 5), (8, 16), (32, 31), (33, 64), (40, 50), (64, 128), (96, 96), (100, 17),
                                       (128, 128), (129, 33), (128, 300), (200, 128), (256, 64), (256, 256)])
def test_widths(key, value, dtype):
    check(problem(1, 131, 1, 2, key, value, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,key_heads,heads", [(1, 1, 1), (3, 2, 2), (2, 2, 6), (1, 1, 4), (2, 3, 9)])
def test_heads(batch, key_heads, heads, dtype):
    check(problem(batch, 70, key_heads, heads, 32, 24, dtype))
    check(problem(batch, 150, key_heads, heads, 128, 64, dtype, initial=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gates,state", [(F32, F32), (BF16, F16), (F16, BF16)])
def test_other_dtypes_of_the_gates_and_the_state(dtype, gates, state):
    check(problem(2, 77, 2, 4, 64, 64, dtype, gates=gates, state=state))
    check(problem(1, 77, 2, 4, 24, 20, F32, gates=gates, state=state))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("use", [("y",), ("final",)])
def test_one_output_used(use, dtype):
    check(problem(1, 100, 1, 2, 40, 32, dtype), use=use)
    check(problem(1, 100, 1, 2, 40, 32, dtype, initial=False), use=use, scale=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_long_sequences(dtype):
    """Many chunks a sequence, few sequences and heads, which run in segments side by side: whole and ragged."""
    check(problem(1, 4096, 1, 1, 64, 64, dtype))
    check(problem(1, 2500, 1, 2, 128, 128, dtype, initial=False))
    check(problem(2, 3001, 1, 1, 96, 40, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [24 * 64 - 1, 24 * 64, 24 * 64 + 1, 25 * 64, 1727])
def test_lengths_at_the_seams_of_segments(length):
    """24 chunks are the fewest that are cut; the last segment has from one token to all of its chunks."""
    check(problem(1, length, 1, 2, 32, 24, BF16, initial=length % 2 == 0))
    check(problem(1, length, 1, 2, 256, 40, BF16), use=("final",))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_long_sequence_of_unaligned_rows(dtype):
    """It is not cut, whatever the workspace has room for."""
    p = problem(1, 2000, 1, 2, 64, 32, dtype)
    d = to_dev(p)
    wide = torch.zeros(1, 2000, 1, 2 * 64 + 1, dtype=dtype, device=DEV)
    wide[..., 1:65], wide[..., 65:] = d["q"], d["k"]
    with torch.no_grad():
        y, final = call({**d, "q": wide[..., 1:65], "k": wide[..., 65:]})
    want = oracle.gated_delta_rule(*(p[n] for n in NAMES[:5]), initial=p["initial"])
    assert rel(y, want[0]) <= FWD[dtype] and rel(final, want[1]) <= FWD[dtype] + U[dtype]


@pytest.mark.gpu
def test_documents_and_nan_in_a_cut_sequence():
    """A log decay of -inf drops what earlier segments left, and a NaN leaves the segments before it alone."""
    p = problem(1, 2048, 1, 2, 64, 32, BF16)
    p["log_decay"][:, 1000] = -float("inf")
    d = to_dev(p)
    with torch.no_grad():
        y, final = call(d)
        tail = {n: t[:, 1000:] if n in NAMES[:5] else t for n, t in p.items()}
        tail["log_decay"] = torch.where(torch.isinf(tail["log_decay"]), 0.0, tail["log_decay"])
        want = oracle.gated_delta_rule(*(tail[n] for n in NAMES[:5]))
        assert rel(y[:, 1000:], want[0]) <= FWD[BF16] and rel(final, want[1]) <= FWD[BF16] + U[BF16]
        d["v"][0, 1500, 1, 3] = float("nan")
        got, last = call(d)
    assert torch.equal(got[:, :1472], y[:, :1472]) and torch.equal(got[:, :, 0], y[:, :, 0])
    assert torch.isnan(got[0, 1500:, 1].float()).any(-1).all() and torch.isnan(last[0, 1, 3].float()).all()
    assert torch.isfinite(got[0, :, 1, :3].float()).all()  # the other value rows have states of their own


@pytest.mark.gpu
@pytest.mark.parametrize("key_heads,heads", [(2, 4), (4, 12)])
def test_many_chunks_of_shared_key_heads(key_heads, heads):
    """From 256 key-head chunks on the value heads of a key head are summed by one workgroup."""
    for dtype in (F32, BF16):
        check(problem(3, 64 * 45, key_heads, heads, 32, 40, dtype))
    check(problem(2, 64 * 70 - 5, 2, 4, 128, 24, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays_of_zero_and_strong_ones(dtype):
    """No forgetting, and decays whose exponentials differ by more than a float holds within a chunk."""
    p = problem(1, 200, 1, 2, 64, 32, dtype)
    p["log_decay"] = torch.zeros_like(p["log_decay"])
    check(p)
    p["log_decay"] = torch.full_like(p["log_decay"], -20.0)
    p["log_decay"][:, ::7] = 0.0
    p["log_decay"][:, 40:90] = 0.0
    check(p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_keys_and_betas_at_the_ends(dtype):
    """One key throughout, the largest triangular system; corrections of zero and of the whole error.  Here
    the state is a telescoping sum of the chunk's 64 corrections, which their roundings do not share:
    independent ones add to sqrt(64) times one of them."""
    p = problem(1, 150, 1, 2, 32, 32, dtype)
    p["k"] = p["k"][:, :1].expand_as(p["k"]).contiguous()
    p["log_decay"] = torch.zeros_like(p["log_decay"])
    p["beta"][:, ::3], p["beta"][:, 1::3] = 0.0, 1.0
    check(p, times=1 if dtype == F32 else 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_documents_in_one_row(dtype):
    """A log decay of -inf drops the state: outputs and gradients are those of the documents alone."""
    p = problem(1, 210, 1, 2, 64, 64, dtype, initial=False)
    cuts = [0, 10, 64, 140, 210]
    for c in cuts[1:-1]:
        p["log_decay"][:, c] = -float("inf")
    d = to_dev(p)
    outs, grads = gradients(d, ("y",))
    assert all(torch.isfinite(t.float()).all() for t in grads.values())
    for a, b in zip(cuts, cuts[1:]):
        part = {n: t[:, a:b] if n in ("q", "k", "v", "log_decay", "beta", "dy") else t for n, t in p.items() if t is not None}
        part["log_decay"] = torch.where(torch.isinf(part["log_decay"]), 0.0, part["log_decay"])
        args = [part[n] for n in NAMES[:5]]
        y, _ = oracle.gated_delta_rule(*args)
        want = oracle.gated_delta_rule_bwd(part["dy"], None, *args)
        assert rel(outs["y"][:, a:b], y) <= FWD[dtype]
        for name, w in zip(NAMES[:5], want):
            if name == "log_decay":  # the first token's decay meets no state
                assert rel(grads[name][:, a + 1:b], w[:, 1:]) <= BWD[dtype] + U[dtype]
                assert grads[name][:, a].abs().max() <= BWD[dtype] * w.abs().max()
            else:
                assert rel(grads[name][:, a:b], w) <= BWD[dtype] + U[dtype], name


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["v", "k", "log_decay", "beta"])
def test_what_is_not_finite_stays_in_its_head_and_behind(where):
    p = problem(2, 200, 2, 4, 64, 32, BF16)
    with torch.no_grad():
        clean = call(to_dev(p))
        p[where][1, 100, 1] = float("nan")
        y, final = call(to_dev(p))
    heads = [2, 3] if where == "k" else [1]
    others = [h for h in range(4) if h not in heads]
    assert torch.equal(y[0], clean[0][0]) and torch.equal(y[1][:, others], clean[0][1][:, others])
    assert torch.equal(y[1, :64], clean[0][1, :64])
    assert torch.isnan(y[1, 100:, heads].float()).any(-1).all() and torch.isnan(final[1, heads].float()).any()
    assert torch.equal(final[1, others], clean[1][1, others])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients_against_differences(dtype):
    """Those of the oracle in 64 bits along a direction; its step's third-order term is below 1e-7."""
    p = problem(1, 90, 1, 2, 32, 16, dtype)
    _, grads = gradients(to_dev(p))
    wide = {n: t.to(F64) for n, t in p.items()}
    g = torch.Generator().manual_seed(3)
    for name in NAMES:
        d, step = torch.randn(p[name].shape, generator=g, dtype=F64), 1e-5

        def loss(s):
            a = {**wide, name: wide[name] + s * step * d}
            y, final = oracle.gated_delta_rule(*(a[n] for n in NAMES[:5]), initial=a["initial"])
            return (y * wide["dy"]).sum() + (final * wide["dfinal"]).sum()

        want = ((loss(1) - loss(-1)) / (2 * step)).item()
        got = (grads[name].double().cpu() * d).sum().item()
        # an error vector of the bound's norm, all of it along the direction
        assert abs(got - want) <= (BWD[dtype] + U[dtype]) * grads[name].double().norm().item() * d.norm().item() + 1e-5, name


# --------------------------------------------------------------------------- GPU: layouts and callers


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_slices_of_one_projection(offset, dtype):
    """q, k and v inside one wider tensor, at any alignment, transposed and negated views of them."""
    p = problem(2, 100, 2, 4, 32, 24, dtype)
    parts = [p[n].flatten(2) for n in ("q", "k", "v")]
    wide = torch.cat([torch.full((2, 100, offset), float("nan"), dtype=dtype), *parts], -1).to(DEV)
    d = to_dev(p)
    at, sliced = offset, dict(d)
    for n, part in zip(("q", "k", "v"), parts):
        sliced[n] = wide[..., at:at + part.shape[2]].unflatten(2, d[n].shape[2:])
        at += part.shape[2]
    want, want_grads = gradients(d)
    got, got_grads = gradients(sliced)
    exact = offset % 8 == 0 or dtype == F32  # another alignment may take another path of the same arithmetic
    for a, b in [*zip(got.values(), want.values()), *zip(got_grads.values(), want_grads.values())]:
        assert torch.equal(a, b) if exact else rel(a, b) <= BWD[dtype]
    moved = dict(d)
    for n in ("q", "k", "v"):
        moved[n] = d[n].transpose(1, 2).contiguous().transpose(1, 2)
    moved["log_decay"], moved["beta"] = (d[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("log_decay", "beta"))
    got, got_grads = gradients(moved)
    assert all(torch.equal(a, b) for a, b in zip([*got.values(), *got_grads.values()], [*want.values(), *want_grads.values()]))
    with torch.no_grad():
        negated = call({**d, "q": torch._neg_view(-d["q"]), "initial": torch._neg_view(-d["initial"])})
        assert torch.equal(negated[0], want["y"]) and torch.equal(negated[1], want["final"])


@pytest.mark.gpu
def test_broadcast_inputs_and_one_tensor_in_two_roles():
    p = problem(2, 80, 1, 2, 32, 32)
    d = to_dev(p)
    one = torch.full((1,), 0.5, device=DEV, requires_grad=True)
    row = d["log_decay"][:1, :1].clone().requires_grad_(True)
    both = d["k"].clone().requires_grad_(True)
    y = call({**d, "q": both, "k": both, "beta": one.expand(2, 80, 2), "log_decay": row.expand(2, 80, 2)}, final=False)
    y.backward(d["dy"])
    beta, decay = torch.full((2, 80, 2), 0.5), p["log_decay"][:1, :1].expand(2, 80, 2)
    want = oracle.gated_delta_rule_bwd(p["dy"], None, p["k"], p["k"], p["v"], decay, beta, initial=p["initial"])
    assert rel(both.grad, want[0] + want[1]) <= 2e-5
    assert rel(row.grad, want[3].sum((0, 1), keepdim=True)) <= 1e-5 * 160 ** 0.5
    assert abs(one.grad.item() - want[4].sum().item()) <= 1e-5 * want[4].norm().item() * 320 ** 0.5


@pytest.mark.gpu
def test_gradients_of_some_inputs():
    d = to_dev(problem(1, 90, 1, 2, 32, 32, BF16))
    _, every = gradients(d)
    for name in NAMES:
        leaf = d[name].clone().requires_grad_(True)
        y, final = call({**d, name: leaf})
        got, = torch.autograd.grad([y, final], leaf, [d["dy"], d["dfinal"]])
        assert torch.equal(got, every[name]), name


@pytest.mark.gpu
def test_empty_sizes():
    for sizes in [(0, 5, 1, 2, 8, 8), (2, 0, 1, 2, 8, 8), (2, 5, 1, 2, 8, 0)]:
        p = problem(*sizes)
        outs, grads = gradients(to_dev(p))
        assert outs["y"].shape == p["v"].shape
        if sizes[1] == 0:
            assert torch.equal(outs["final"].cpu(), p["initial"]) and torch.equal(grads["initial"].cpu(), p["dfinal"])
        else:
            assert all((g == 0).all() for g in grads.values())
        _, bare = call({**to_dev(p), "initial": None})
        assert (bare == 0).all() and bare.shape == p["initial"].shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", [(2, 300, 2, 4, 128, 64), (1, 1500, 1, 2, 96, 96)])
def test_results_repeat_and_do_not_depend_on_old_memory(sizes, dtype):
    d = to_dev(problem(*sizes, dtype))

    def run(fill):
        before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
        torch.use_deterministic_algorithms(fill)  # fills what torch.empty allocates with NaN
        torch.utils.deterministic.fill_uninitialized_memory = fill
        try:
            outs, grads = gradients(d)
            with torch.no_grad():
                plain = call(d)
                step = _update(d)
        finally:
            torch.use_deterministic_algorithms(before[0])
            torch.utils.deterministic.fill_uninitialized_memory = before[1]
        return [*outs.values(), *grads.values(), *plain, *step]

    first = run(False)
    for k, (a, b, c) in enumerate(zip(first, run(True), run(False))):
        assert torch.isfinite(b.float()).all() and torch.equal(a, b) and torch.equal(a, c), k


def _graph_of(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    return graph, held


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [(2, 200, 1, 2, 64, 64), (1, 1300, 1, 1, 64, 32)])
def test_captured_training_replays(sizes):
    d = to_dev(problem(*sizes, BF16))

    def step():
        outs, grads = gradients(d)
        return [*(t.detach() for t in outs.values()), *grads.values()]

    graph, held = _graph_of(step)
    for k in range(3):
        d["v"].copy_(torch.randn(d["v"].shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_two_captured_graphs_and_streams_at_once():
    """Graphs and streams keep to their own workspaces."""
    ds = [to_dev(problem(1, 700 + i, 1, 2, 64, 64, BF16, seed=i)) for i in range(2)]
    with torch.no_grad():
        want = [call(d) for d in ds]
        graphs = [_graph_of(lambda d=d: call(d)) for d in ds]
        streams = [torch.cuda.Stream() for _ in ds]
        torch.cuda.synchronize()
        outs = [[], []]
        for _ in range(3):
            for i, (s, (graph, _)) in enumerate(zip(streams, graphs)):
                with torch.cuda.stream(s):
                    graph.replay()
                    outs[i].append(call(ds[i]))
        torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i]))
        assert all(torch.equal(a, b) for o in outs[i] for a, b in zip(o, want[i]))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The second sequence of a batch whose keys pass 2^32 bytes, against the sequence alone."""
    g = torch.Generator(device=DEV).manual_seed(0)
    b, l, h, k, v = 2, 80_000, 64, 256, 32
    q = torch.empty(b, l, h, k, dtype=BF16, device=DEV).normal_(generator=g).mul_(k ** -0.5)
    val = torch.empty(b, l, h, v, dtype=BF16, device=DEV).normal_(generator=g)
    decay = torch.full((1, 1, 1), -0.05, dtype=BF16, device=DEV).expand(b, l, h)
    beta = torch.full((1, 1, 1), 0.5, dtype=BF16, device=DEV).expand(b, l, h)
    with torch.no_grad():
        from metal_kernelops.cv import gated_delta_rule
        y, final = gated_delta_rule(q, q, val, decay, beta, return_final_state=True)
        one, last = gated_delta_rule(q[1:], q[1:], val[1:], decay[1:], beta[1:], return_final_state=True)
    assert torch.isfinite(one.float()).all()
    assert rel(y[1], one[0]) <= FWD[BF16] and rel(final[1], last[0]) <= FWD[BF16]


@pytest.mark.gpu
def test_a_second_derivative_and_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwd
    d = to_dev(problem(1, 20, 1, 1, 8, 8))
    q = d["q"].clone().requires_grad_(True)
    grad, = torch.autograd.grad(call({**d, "q": q}, final=False).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), q)
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        call({**d, "q": fwd.make_dual(d["q"], d["q"])})


@pytest.mark.gpu
def test_refusals():
    from metal_kernelops.cv import gated_delta_rule, gated_delta_rule_update
    d = to_dev(problem(2, 5, 1, 2, 8, 6))
    args = [d[n] for n in NAMES[:5]]
    for i in range(5):
        for t in (args[i].double(), args[i].cpu()):
            with pytest.raises(ValueError):
                gated_delta_rule(*(t if j == i else a for j, a in enumerate(args)))
    with pytest.raises(ValueError):
        gated_delta_rule(args[0].half(), *args[1:])
    for s in (d["initial"][:1], d["initial"].cpu(), d["initial"].double(), d["initial"].transpose(2, 3)):
        with pytest.raises(ValueError):
            gated_delta_rule(*args, initial_state=s)
        with pytest.raises(ValueError):
            gated_delta_rule_update(s, *(a[:, 0] for a in args))
    one = [a[:, 0] for a in args]
    for out in (d["initial"][:1], d["initial"].half(), d["initial"].cpu(), torch._neg_view(d["initial"]),
                d["initial"].transpose(2, 3).contiguous().transpose(2, 3), d["initial"].clone().requires_grad_(True)):
        with pytest.raises(ValueError):
            gated_delta_rule_update(d["initial"], *one, out_state=out)


# --------------------------------------------------------------------------- GPU: one token


def _update(d, state=None, t=0, **kw):
    from metal_kernelops.cv import gated_delta_rule_update
    return gated_delta_rule_update(d["initial"] if state is None else state, *(d[n][:, t] for n in NAMES[:5]), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,state", [(F32, F32), (BF16, F32), (F16, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 1), (1, 2, 4, 128, 128), (3, 1, 2, 7, 5), (2, 2, 2, 40, 33), (2, 1, 3, 64, 300),
                                   (1, 2, 2, 256, 17), (2, 1, 1, 100, 50), (40, 4, 16, 128, 128)])
def test_update(sizes, dtype, state):
    batch, key_heads, heads, key, value = sizes
    p = problem(batch, 1, key_heads, heads, key, value, dtype, state=state)
    want = oracle.gated_delta_rule(*(p[n] for n in NAMES[:5]), scale=0.3, initial=p["initial"])
    with torch.no_grad():
        y, new = _update(to_dev(p), scale=0.3)
    assert y.dtype == dtype and new.dtype == state
    assert rel(y, want[0][:, 0]) <= 1e-6 + U[dtype] and rel(new, want[1]) <= 1e-6 + U[state]


@pytest.mark.gpu
def test_updates_follow_the_scan_in_place():
    d = to_dev(problem(2, 100, 2, 4, 64, 32))
    with torch.no_grad():
        want, final = call(d)
        state, ys = d["initial"].clone(), []
        for t in range(100):
            y, new = _update(d, state, t, out_state=state)
            assert new is state
            ys.append(y)
    assert rel(torch.stack(ys, 1), want) <= 2e-5 and rel(state, final) <= 2e-5


@pytest.mark.gpu
def test_update_destinations_slices_and_cleared_states():
    d = to_dev(problem(3, 1, 2, 4, 40, 24, BF16, state=F32))
    with torch.no_grad():
        want = _update(d)
        before, out = d["initial"].clone(), torch.empty_like(d["initial"])
        got = _update(d, out_state=out)
        assert got[1] is out and torch.equal(out, want[1]) and torch.equal(got[0], want[0])
        assert torch.equal(d["initial"], before)
        buffer = torch.cat([torch.full_like(before[:1], 7.0), before, torch.full_like(before[:1], 9.0)])
        got = _update(d, buffer[1:4], out_state=buffer[2:5])  # moved by one user
        assert torch.equal(got[1], want[1]) and (buffer[0] == 7).all() and torch.equal(buffer[1], before[0])
        wide = torch.cat([d["q"][:, 0].flatten(1), d["v"][:, 0].flatten(1)[:, :1], d["k"][:, 0].flatten(1)], -1)
        odd = {**d, "k": wide[:, 81:].unflatten(1, (2, 40))[:, None]}
        got = _update(odd)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        y, new = _update({**d, "log_decay": torch.full_like(d["log_decay"], -float("inf"))})
        alone = _update({**d, "log_decay": torch.zeros_like(d["log_decay"])}, torch.zeros_like(before))
        assert torch.equal(y, alone[0]) and torch.equal(new, alone[1])


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
def test_update_gradients_are_those_of_a_scan_of_one(in_place):
    p = problem(2, 1, 1, 2, 32, 24)
    d = to_dev(p)
    leaves = {n: d[n].clone().requires_grad_(True) for n in NAMES if not (in_place and n == "initial")}
    held = {**d, **leaves}
    y, new = _update(held, out_state=held["initial"] if in_place else None)
    outs, dys = ([y], [d["dy"][:, 0]]) if in_place else ([y, new], [d["dy"][:, 0], d["dfinal"]])
    got = torch.autograd.grad(outs, list(leaves.values()), dys)
    want = oracle.gated_delta_rule_bwd(p["dy"], None if in_place else p["dfinal"], *(p[n] for n in NAMES[:5]),
                                       initial=p["initial"])
    for name, a, w in zip(leaves, got, want):
        assert rel(a, w) <= 1e-5, name


@pytest.mark.gpu
def test_captured_updates_replay():
    d = to_dev(problem(4, 1, 2, 4, 64, 64, BF16, state=F32))
    state = d["initial"].clone()
    with torch.no_grad():
        graph, held = _graph_of(lambda: _update(d, state, out_state=state))
        state.copy_(d["initial"])
        eager = d["initial"].clone()
        for k in range(4):
            d["v"].copy_(torch.randn(d["v"].shape, generator=torch.Generator().manual_seed(k)))
            graph.replay()
            y, _ = _update(d, eager, out_state=eager)
            torch.cuda.synchronize()
            assert torch.equal(held[0], y) and torch.equal(state, eager)
