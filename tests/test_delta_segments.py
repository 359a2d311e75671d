"""The gated delta rule on sequences that run in segments side by side, where the state outlives a segment: what is
kept passes in float32, and every chunk is compared by itself.

Tolerances, with u half a unit in the last place of the activations (2^-8 for bfloat16, 2^-11 for float16).  The part of
the state that is only kept is a product of one factor a chunk: a float32 exponential (one unit, at most 2^-24 of a
number just below one) and a float32 product (2^-24), and two more products a segment, of which there is at most one for
eight chunks: 3 * 2^-24 a chunk.  What corrections have written or taken away carries eight 16-bit roundings: 8 u of its
norm, as the rule's own tests count them.  Compared by chunks, where a fault of one chunk is as large as the output, the
roundings of different operands are independent and add by their squares: the forward's eight to sqrt(8) u, the
backward's sixteen to 4 u, and u for storing a gradient.  Float32: 1e-5, and the same a chunk for what is kept.
"""

import ctypes
import math

import pytest
import torch

from oracle import delta_rule as oracle
from test_gated_delta import BF16, DEV, F16, F32, NAMES, U, call, gradients, problem, to_dev

FWD = {F32: 1e-5, F16: math.sqrt(8) * U[F16], BF16: math.sqrt(8) * U[BF16]}
BWD = {F32: 1e-5, F16: 5 * U[F16], BF16: 5 * U[BF16]}
CORRECTED = {F32: 1e-5, F16: 8 * U[F16], BF16: 8 * U[BF16]}


def kept(length):
    return 3 * 2.0 ** -24 * -(-length // 64)


def slow(batch, length, key_heads, heads, key, value, dtype, decay, beta, seed=0):
    """A problem whose tokens forget ``exp(decay)`` and correct by ``beta``, each varied by half, with gates and
    states in float32."""
    p = problem(batch, length, key_heads, heads, key, value, dtype, seed=seed, gates=F32, state=F32)
    g = torch.Generator().manual_seed(length + seed)
    for name, mean in (("log_decay", decay), ("beta", beta)):
        p[name] = mean * (0.5 + torch.rand(p[name].shape, generator=g))
    return p


def exact(p):
    return oracle.gated_delta_rule(*(p[n] for n in NAMES[:5]), initial=p["initial"])


def by_chunks(got, want):
    """The largest relative error of a chunk of 64 tokens of a head of a sequence."""
    got, want = got.detach().double().cpu(), want.detach().double()
    return max(((a - b).norm(dim=(1, 3)) / b.norm(dim=(1, 3))).max().item()
               for a, b in zip(got.split(64, 1), want.split(64, 1)))


def segments(length, heads, key, value, dtype):
    """Of one sequence, from the workspace that the library asks for: T and P, the decays, and beside them what the
    segments but the last one leave."""
    from metal_kernelops import _native as nat
    p = nat.DeltaParams(batch=1, length=length, key_heads=1, heads=heads, key=key, value=value, dtype=nat.code(dtype))
    size, cells = 4 if dtype == F32 else 2, heads * -(-length // 64)
    more = nat.lib().mko_delta_fwd_workspace_size(ctypes.byref(p)) - cells * (2 * 6 * 512 * size + 64 * 24)
    each = heads * 4 * (value * key + key * key + 1)
    return 1 + round(more / each)  # whole, but for the alignment of the arrays


@pytest.mark.parametrize("dtype,key,value,chunks,heads,want", [
    (BF16, 128, 128, 24, 1, 1), (BF16, 64, 64, 40, 2, 1), (BF16, 128, 128, 64, 21, 1), (F16, 32, 32, 80, 84, 1),
    (BF16, 128, 128, 48, 1, 6), (BF16, 64, 64, 50, 2, 6), (BF16, 128, 128, 64, 16, 4), (BF16, 128, 128, 512, 16, 4),
    (F16, 64, 64, 512, 1, 22), (BF16, 256, 128, 24, 1, 3), (BF16, 256, 128, 64, 21, 3), (F32, 64, 64, 24, 2, 3),
    (F32, 64, 64, 64, 42, 3), (F32, 32, 32, 24, 4, 1), (F32, 32, 32, 40, 4, 5), (F32, 32, 32, 160, 84, 1),
    (BF16, 128, 128, 512, 22, 1), (BF16, 60, 64, 512, 2, 1)])
def test_sequences_are_cut_where_it_pays(dtype, key, value, chunks, heads, want):
    """The sizes that the rule was measured at, on both of its sides."""
    assert segments(chunks * 64, heads, key, value, dtype) == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("sizes", [(1, 4096, 1, 1, 64, 64), (1, 4001, 1, 2, 128, 40), (2, 3300, 1, 1, 24, 8), (1, 1600, 1, 1, 256, 16)])
def test_a_state_that_nothing_changes_comes_back_bit_for_bit(sizes, dtype):
    """No forgetting and no correction: every output reads the initial state."""
    p = slow(*sizes, dtype, 0.0, 0.0)
    with torch.no_grad():
        y, final = call(to_dev(p))
    assert torch.equal(final.cpu(), p["initial"])
    assert by_chunks(y, exact(p)[0]) <= FWD[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("length,decay,beta", [(16384, -1e-5, 5e-4), (16384, -1e-6, 5e-5), (32768, -1.2e-6, 0.0),
                                               (5000, -1e-3, 1e-4), (5000, 0.0, 1e-2)])
def test_a_state_that_forgets_slowly(length, decay, beta, dtype):
    p = slow(1, length, 1, 1, 64, 64, dtype, decay, beta)
    want, last = exact(p)
    with torch.no_grad():
        y, final = call(to_dev(p))
    start = p["initial"].double()
    left = p["log_decay"].double().sum(1).exp()[..., None, None] * start
    bound = kept(length) * left.norm().item() + CORRECTED[dtype] * (last - left).norm().item()
    assert (final.cpu().double() - last).norm().item() <= bound
    # the state's error reaches an output beside the output's own roundings
    assert by_chunks(y, want) <= FWD[dtype] + bound / min(last.norm().item(), start.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("length", [24 * 64 - 1, 24 * 64 + 1, 47 * 64 + 1, 50 * 64, 50 * 64 + 1])
def test_chunks_and_gradients_at_the_seams(length, dtype):
    """States that reach across several segments (the shorter sequences are cut in float32, the longer in every type):
    outputs and gradients chunk by chunk, the last one's single token among them, and the whole gradient of the initial
    state."""
    p = slow(1, length, 1, 2, 64, 48, dtype, -5e-4, 0.02)
    args = [p[n] for n in NAMES[:5]]
    want, last = exact(p)
    outs, grads = gradients(to_dev(p))
    assert by_chunks(outs["y"], want) <= FWD[dtype]
    assert (outs["final"].detach().cpu().double() - last).norm().item() <= FWD[dtype] * last.norm().item()
    exact_grads = dict(zip(NAMES, oracle.gated_delta_rule_bwd(p["dy"], p["dfinal"], *args, initial=p["initial"])))
    for name in ("q", "k", "v"):
        assert by_chunks(grads[name], exact_grads[name]) <= BWD[dtype], name
    for name in ("beta", "initial"):  # a number a token, and one gradient
        w = exact_grads[name]
        assert w.norm().item() > 0.1  # it is there
        assert (grads[name].cpu().double() - w).norm().item() <= BWD[dtype] * w.norm().item(), name


def check_chunks(p, fwd, bwd):
    """Outputs and the gradients of q, k and v chunk by chunk, the others whole."""
    args = [p[n] for n in NAMES[:5]]
    want, last = exact(p)
    outs, grads = gradients(to_dev(p))
    assert by_chunks(outs["y"], want) <= fwd
    assert (outs["final"].detach().cpu().double() - last).norm().item() <= (fwd + U[p["dfinal"].dtype]) * last.norm().item()
    exact_grads = dict(zip(NAMES, oracle.gated_delta_rule_bwd(p["dy"], p["dfinal"], *args, initial=p["initial"])))
    for name in ("q", "k", "v"):
        assert by_chunks(grads[name], exact_grads[name]) <= bwd, name
    for name in ("beta", "initial"):
        w = exact_grads[name]
        assert (grads[name].cpu().double() - w).norm().item() <= bwd * w.norm().item(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("sizes", [(2, 1, 1, 2, 64, 48), (2, 129, 1, 2, 64, 48), (1, 200, 2, 2, 128, 128), (1, 131, 1, 2, 256, 64),
                                   (1, 131, 1, 2, 33, 31), (2, 150, 1, 4, 128, 64), (3, 64 * 43 + 1, 2, 4, 32, 40)])
def test_every_chunk_is_as_near_as_its_roundings(sizes, dtype):
    """Sequences that are not cut: one token, whole and ragged chunks, wide and odd rows, shared key heads."""
    check_chunks(problem(*sizes, dtype), FWD[dtype], BWD[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_equal_keys_in_every_type(dtype):
    """One key throughout and no forgetting: a state is a telescoping sum of the chunk's 64 corrections, whose
    roundings are independent and add to sqrt(64) times one of them."""
    p = problem(1, 150, 1, 2, 32, 32, dtype)
    p["k"] = p["k"][:, :1].expand_as(p["k"]).contiguous()
    p["log_decay"] = torch.zeros_like(p["log_decay"])
    p["beta"][:, ::3], p["beta"][:, 1::3] = 0.0, 1.0
    times = 1 if dtype == F32 else 8
    y, _ = exact(p)
    outs, grads = gradients(to_dev(p))
    assert (outs["y"].detach().cpu().double() - y).norm().item() <= times * FWD[dtype] * y.norm().item()
    want = oracle.gated_delta_rule_bwd(p["dy"], p["dfinal"], *(p[n] for n in NAMES[:5]), initial=p["initial"])
    for name, w in zip(NAMES, want):
        assert (grads[name].cpu().double() - w).norm().item() <= times * BWD[dtype] * w.norm().item(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_two_captured_cut_sequences_replay(dtype):
    """Each graph has segments of its own, and a replay with other values those values' results."""
    ds = [to_dev(slow(1, 3200, 1, 2, 64, 48, dtype, -5e-4, 0.02, seed=i)) for i in range(2)]
    with torch.no_grad():
        graphs = []
        for d in ds:
            call(d)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = call(d)
            graphs.append((graph, held))
        for k in range(3):
            for d in ds:
                d["v"].copy_(torch.randn(d["v"].shape, generator=torch.Generator().manual_seed(k)))
            want = [call(d) for d in ds]
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for (_, held), w in zip(graphs, want):
                assert all(torch.equal(a, b) for a, b in zip(held, w))
