"""The gated delta rule against its definition, frame by frame in 64 bits.

Tolerances.  The state is a contraction of what it was (its factor f (1 - w k k') has a norm of 1 at most, as k has length one), so a rounding error made in one frame
does not grow afterwards: an output has the errors of a sum of ``terms`` products, those of a chunk's triangular system and of the frames a state lasts,
each 2^-24 of the size of what is added up.  That size is that of the result, up to a factor (``spread``) for what cancels: 4 for values and states, 16 for the gates'
gradients, which are differences of sums over a chunk.  Bounds are on the 2-norm over a tensor, and 64 times as wide, of the root mean square, on every value.
Values of 16 bits are rounded once more, by 2^-8 at most."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8
DTYPES = [torch.float32, torch.bfloat16]
NAMES = ("q", "k", "v", "gate", "beta", "initial")


STREAMS = {}


def stream_of(name):
    """One stream for a name: streams share a few hardware queues, and what else runs in this process should find them as free as it can."""
    if name not in STREAMS:
        STREAMS[name] = torch.cuda.Stream()
    return STREAMS[name]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def problem(B, T, H, G, K, V, dtype, seed=1, lens=None, initial=True):
    g = gen(seed)
    values = {"q": torch.randn((B, T, G, K), generator=g, device="cuda"), "v": torch.randn((B, T, H, V), generator=g, device="cuda")}
    values["k"] = torch.randn((B, T, G, K), generator=g, device="cuda") + 0.5
    values["gate"] = torch.randn((B, T, H), generator=g, device="cuda") + torch.linspace(0.0, 5.0, H, device="cuda")
    values["beta"] = torch.randn((B, T, H), generator=g, device="cuda")
    p = {n: values[n].to(dtype) for n in NAMES[:5]}
    p["initial"] = torch.randn((B, H, K, V), generator=g, device="cuda") if initial else None
    p["lens"] = None if lens == "all" else torch.tensor(lens, dtype=torch.int32, device="cuda") if lens is not None else torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    p["grad_o"] = torch.randn((B, T, H, V), generator=g, device="cuda").to(dtype)
    p["grad_last"] = torch.randn((B, H, K, V), generator=g, device="cuda")
    return p


def expected(p, grads=True):
    """By autograd through the recurrence in 64 bits, on the CPU."""
    B, T, H, V = p["v"].shape
    G = p["k"].shape[2]
    leaves = {n: p[n].detach().double().cpu().requires_grad_(grads) if p[n] is not None else None for n in NAMES}
    lens = (p["lens"].long().cpu() if p["lens"] is not None else torch.full((B,), T)).clamp(0, T)

    def unit(x):
        return (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(H // G, dim=2)

    # frames behind the end may hold anything
    live = torch.arange(T)[None, :] < lens[:, None]
    inputs = {n: torch.where(live.view(B, T, *[1] * (leaves[n].dim() - 2)), leaves[n], 0.0) for n in NAMES[:5]}
    q, k = unit(inputs["q"]), unit(inputs["k"])
    f, w = torch.sigmoid(inputs["gate"]), torch.sigmoid(inputs["beta"])
    S = leaves["initial"] if leaves["initial"] is not None else torch.zeros(B, H, p["k"].shape[3], V, dtype=torch.float64)
    o = []
    for t in range(T):
        kept = f[:, t, :, None, None] * S
        u = w[:, t, :, None] * (inputs["v"][:, t] - (kept * k[:, t, :, :, None]).sum(2))
        on = (t < lens).view(B, 1, 1, 1)
        S = torch.where(on, kept + k[:, t, :, :, None] * u[:, :, None, :], S)
        o.append((S * q[:, t, :, :, None]).sum(2) * on[..., 0])
    out = {"o": torch.stack(o, 1), "last": S}
    if not grads:
        return {n: x.cuda() for n, x in out.items()}
    loss = (out["o"] * torch.where(live[:, :, None, None], p["grad_o"].double().cpu(), 0.0)).sum() + (out["last"] * p["grad_last"].double().cpu()).sum()
    names = [n for n in NAMES if leaves[n] is not None]
    out |= dict(zip(names, torch.autograd.grad(loss, [leaves[n] for n in names])))
    return {n: x.detach().cuda() for n, x in out.items()}


def run(p, grads=True):
    from i6_native_ops_amd.training import gated_delta_rule
    leaves = {n: p[n].detach().requires_grad_(grads) if p[n] is not None else None for n in NAMES}
    o, last = gated_delta_rule(*(leaves[n] for n in NAMES[:5]), seq_lens=p["lens"], initial_state=leaves["initial"])
    out = {"o": o.detach(), "last": last.detach()}
    if grads:
        names = [n for n in NAMES if leaves[n] is not None]
        out |= dict(zip(names, torch.autograd.grad([o, last], [leaves[n] for n in names], [p["grad_o"], p["grad_last"]])))
    return out


def check(p, got, want):
    K, V = p["k"].shape[3], p["v"].shape[3]
    f = torch.sigmoid(torch.nan_to_num(p["gate"].float())).max()
    lasts = min(p["k"].shape[1], 1.0 / max(1e-4, 1.0 - float(f)))
    terms = K + V + 4 * 32 + lasts
    for n, x in got.items():
        w = want[n]
        assert x.shape == w.shape and x.dtype == (torch.float32 if n in ("last", "initial") else p["v"].dtype), n
        bound = (16 if n in ("gate", "beta") else 4) * terms * EPS32
        out = EPS16 if x.dtype == torch.bfloat16 else 0.0
        d, rms = (x.double() - w).abs(), float(w.square().mean().sqrt())
        assert torch.isfinite(x).all(), n
        assert float(d.norm()) <= (bound + out) * float(w.norm()) + 1e-30, (n, float(d.norm() / w.norm()), bound + out)
        assert (d <= 64 * bound * (rms + w.abs()) + out * w.abs() + 1e-30).all(), (n, float(d.max()), rms)


SIZES = [
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 1, 33, 65), (3, 31, 2, 2, 16, 16), (3, 32, 1, 1, 32, 32), (2, 33, 4, 2, 40, 72), (2, 64, 3, 3, 64, 64), (2, 65, 2, 1, 128, 128),
    (5, 97, 3, 1, 100, 127), (2, 150, 8, 2, 24, 20), (1, 300, 2, 2, 65, 33), (2, 129, 2, 2, 128, 17), (2, 129, 2, 2, 17, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,G,K,V", SIZES)
def test_outputs_and_gradients(B, T, H, G, K, V, dtype):
    p = problem(B, T, H, G, K, V, dtype, seed=B + T + K + V)
    check(p, run(p), expected(p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 7, 16, 17, 40])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (20, 100)])
def test_without_gradients(T, K, V, dtype):
    p = problem(3, T, 4, 2, K, V, dtype, seed=T, lens=[T, max(0, T - 1), 0])
    got = run(p, grads=False)
    check(p, got, expected(p, grads=False))
    assert torch.equal(got["last"][2], p["initial"][2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_stands_behind_the_end(dtype):
    """Lengths of nothing, of one frame, negative, beyond T; NaN and infinities behind them."""
    p = problem(6, 70, 2, 1, 48, 40, dtype, lens=[0, 70, 1, -3, 99, 37])
    want = expected(p)
    behind = torch.arange(70, device="cuda") >= p["lens"][:, None]
    for n in ("q", "k", "v", "gate", "beta", "grad_o"):
        p[n][behind] = float("nan")
    p["k"][0] = float("inf")
    got = run(p)
    check(p, got, want)
    for n in ("o", "q", "k", "v", "gate", "beta"):
        assert (got[n][behind] == 0).all(), n
    assert torch.equal(got["last"][0], p["initial"][0]) and torch.equal(got["initial"][3], p["grad_last"][3])
    nothing = dict(p, lens=torch.zeros_like(p["lens"]))
    got = run(nothing)
    assert all((got[n] == 0).all() for n in ("o", "q", "k", "v", "gate", "beta")) and torch.equal(got["last"], p["initial"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_lengths_and_initial_states_that_are_missing(dtype):
    p = problem(3, 45, 4, 2, 40, 56, dtype, lens="all", initial=False)
    got = run(p)
    check(p, got, expected(p))
    moved = dict(p)
    wide = torch.zeros((45, 3, 2, 47), dtype=dtype, device="cuda")       # time first, rows that begin at odd places
    wide[..., 3:43] = p["q"].transpose(0, 1)
    moved["q"] = wide.transpose(0, 1)[..., 3:43]
    both = torch.cat([p["k"], p["v"].reshape(3, 45, 2, 112)], dim=-1)    # one projection for all
    moved["k"] = both[..., :40]
    moved["v"] = p["v"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    gates = torch.stack([p["gate"], p["beta"]], dim=-1)
    moved["gate"], moved["beta"] = gates[..., 0], gates[..., 1]
    moved["grad_o"] = p["grad_o"].transpose(1, 2).contiguous().transpose(1, 2)
    again = run(moved)
    moved["v"] = p["v"].transpose(2, 3).contiguous().transpose(2, 3)     # features of any stride
    columns = run(moved)
    for n in got:
        assert torch.equal(got[n], again[n]) and torch.equal(got[n], columns[n]), n
    moved["grad_o"] = torch.ones((1, 1, 1, 1), dtype=dtype, device="cuda").expand(3, 45, 4, 56)
    p["grad_o"] = torch.ones_like(p["grad_o"])
    one, other = run(p), run(moved)
    for n in got:
        assert torch.equal(one[n], other[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_at_their_ends(dtype):
    """f = 0 forgets all in front of a frame, f = 1 nothing; w = 0 writes nothing, w = 1 replaces.  In one chunk, in any order."""
    p = problem(2, 80, 2, 2, 32, 32, dtype, lens="all")
    inf = float("inf")
    p["gate"][0, 5], p["gate"][0, 40:43], p["gate"][1, :, 0], p["gate"][1, 64:, 1] = -inf, -inf, inf, -200.0
    p["beta"][0, 10:20], p["beta"][1, :, 1] = -inf, inf
    p["gate"][0, 20:30] = -60.0
    want = expected(p)
    want["gate"] = torch.nan_to_num(want["gate"])
    got = run(p)
    check(p, got, want)
    # (what f = 0 leaves of a gate's gradient is a difference of sums, right within the bound above)
    assert (got["gate"][1, :, 0] == 0).all() and (got["beta"][0, 10:20] == 0).all() and (got["beta"][1, :, 1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_that_are_alike_and_keys_of_nothing(dtype):
    """The triangular system's inverse has entries of alternating signs that a series would have to find among terms thousands of times larger."""
    p = problem(2, 100, 2, 2, 64, 32, dtype, lens="all")
    p["k"][:] = p["k"][:, :1]
    p["gate"][:], p["beta"][:] = 9.0, 6.0
    check(p, run(p), expected(p))
    p["k"][:, 10:50] = 0.0
    p["q"][:, 20] = 0.0
    check(p, run(p), expected(p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V", [(49, 20, 64), (64, 64, 64), (64, 100, 30), (200, 128, 128), (300, 32, 100)])
def test_frames_that_reach_far(T, K, V, dtype):
    """States that last for a thousand frames: every block of a chunk's matrices counts, the farthest ones too."""
    p = problem(2, T, 2, 1, K, V, dtype, lens="all")
    p["gate"][:] = 7.0
    check(p, run(p), expected(p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,V,lens", [(64, 64, [1300, 1217]), (128, 128, [1300, 640]), (32, 40, [1281, 0]), (128, 64, [1000, 1300]), (64, 128, [1300, 1])])
def test_sequences_in_segments(K, V, lens, dtype):
    """Few heads and many frames: a sequence's parts are worked on at the same time.  Ends at and off a segment's, and sequences that end segments before the longest."""
    p = problem(2, 1300, 2, 1, K, V, dtype, lens=lens)
    p["gate"] += 3
    check(p, run(p), expected(p))


def test_a_strong_gate_among_weak_ones():
    """Sums of log f of thousands in front of differences of less than one."""
    p = problem(1, 64, 1, 1, 16, 16, torch.float32, lens="all")
    p["gate"][:] = 3.0
    p["gate"][0, 2] = -5000.0
    p["gate"][0, 33] = -90.0
    check(p, run(p), expected(p))


@pytest.mark.parametrize("dtype", DTYPES)
def test_frames_go_on_from_a_state(dtype):
    """A sequence in pieces, the pieces one by one, and single frames."""
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(2, 75, 4, 2, 64, 48, dtype, lens="all")
    args = [p[n] for n in NAMES[:5]]
    want = expected(p, grads=False)
    for cut in ([0, 33, 34, 75], [0, 1, 64, 75], list(range(0, 76))):
        state, o = p["initial"], []
        for a, b in zip(cut, cut[1:]):
            part, state = gated_delta_rule(*(x[:, a:b] for x in args), initial_state=state)
            o.append(part)
        check(p, {"o": torch.cat(o, 1), "last": state}, want)


def test_gradients_against_differences():
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(2, 40, 2, 1, 24, 20, torch.float32, lens=[40, 23])
    got = run(p)
    g, h = gen(5), 2.0 ** -7
    for n in NAMES:
        v = torch.randn(p[n].shape, generator=g, device="cuda")
        v /= v.norm()
        sides = []
        for s in (h, -h):
            moved = dict(p, **{n: p[n] + s * v})
            o, last = gated_delta_rule(*(moved[x] for x in NAMES[:5]), seq_lens=p["lens"], initial_state=moved["initial"])
            live = torch.arange(40, device="cuda") < p["lens"][:, None]
            sides.append(((o.double() * p["grad_o"]) * live[:, :, None, None]).sum() + (last.double() * p["grad_last"]).sum())
        slope, want = float((sides[0] - sides[1]) / (2 * h)), float((got[n].double() * v).sum())
        # some thousand values of size 1 rounded to 2^-22 add up to 2^-16 over a step of 2^-6; the third derivative's h^2 / 6 times sums of size 10
        assert abs(slope - want) < 2e-3 * max(1.0, abs(want)), (n, slope, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_single_incoming_gradients_and_repeats(dtype):
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(3, 90, 4, 2, 48, 64, dtype)
    full = run(p)
    again = run(p)
    assert all(torch.equal(full[n], again[n]) for n in full)
    zero = run(dict(p, grad_last=torch.zeros_like(p["grad_last"])))
    leaves = [p[n].detach().requires_grad_() for n in NAMES]
    o, last = gated_delta_rule(*leaves[:5], seq_lens=p["lens"], initial_state=leaves[5])
    for n, x in zip(NAMES, torch.autograd.grad(o, leaves, p["grad_o"], retain_graph=True)):
        assert torch.equal(x, zero[n]), n
    zero = run(dict(p, grad_o=torch.zeros_like(p["grad_o"])))
    for n, x in zip(NAMES, torch.autograd.grad(last, leaves, p["grad_last"])):
        assert torch.equal(x, zero[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,lens", [(70, [70, 41]), (1100, [1100, 700])])
def test_captured_calls(T, lens, dtype):
    """Forward and backward replayed with new inputs, eager calls in between; two graphs in turn.  In one piece, and in segments."""
    p = problem(2, T, 4, 2, 64, 64, dtype, lens=lens)
    leaves = [p[n].detach().clone().requires_grad_() for n in NAMES]
    from i6_native_ops_amd.training import gated_delta_rule

    def step():
        o, last = gated_delta_rule(*leaves[:5], seq_lens=p["lens"], initial_state=leaves[5])
        return (o, last) + torch.autograd.grad([o, last], leaves, [p["grad_o"], p["grad_last"]])

    side = stream_of(dtype)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed in range(3):
        new = problem(2, T, 4, 2, 64, 64, dtype, seed=20 + seed, lens=lens)
        with torch.no_grad():
            for leaf, n in zip(leaves, NAMES):
                leaf.copy_(new[n])
        want = run(dict(new, grad_o=p["grad_o"], grad_last=p["grad_last"]))
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            for n, x in zip(("o", "last") + NAMES, out):
                assert torch.equal(x, want[n]), (seed, n)


@pytest.mark.parametrize("T", [100, 900])
def test_on_another_stream(T):
    p = problem(2, T, 2, 2, 64, 64, torch.bfloat16)
    want = run(p)
    side = stream_of("another")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(p)
    side.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_two_calls_at_once():
    """Calls in flight on two streams have workspaces of their own."""
    p, q = problem(1, 2000, 2, 2, 64, 64, torch.bfloat16, seed=5, lens="all"), problem(3, 700, 4, 4, 128, 128, torch.float32, seed=6, lens="all")
    want = run(p), run(q)
    a, b = stream_of(torch.float32), stream_of(torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            x = run(p)
        with torch.cuda.stream(b):
            y = run(q)
        torch.cuda.synchronize()
        for got, right in zip((x, y), want):
            assert all(torch.equal(got[n], right[n]) for n in right)


def test_second_derivatives_and_tangents_are_refused():
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(1, 8, 1, 1, 8, 8, torch.float32)
    for n in NAMES:
        args = {m: p[m].detach().clone() for m in NAMES}
        args[n].requires_grad_()
        o, _ = gated_delta_rule(*(args[m] for m in NAMES[:5]), initial_state=args["initial"])
        grad, = torch.autograd.grad(o.sum(), args[n], create_graph=True)
        with pytest.raises(RuntimeError, match="gated_delta_rule can be differentiated once"):
            grad.square().sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(p["v"], torch.ones_like(p["v"]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            gated_delta_rule(p["q"], p["k"], dual, p["gate"], p["beta"])


def test_refusals():
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(2, 5, 4, 2, 8, 6, torch.float32)
    good = [p[n] for n in NAMES[:5]]

    def refused(match, at=None, value=None, **more):
        args = list(good)
        if at is not None:
            args[at] = value
        with pytest.raises(RuntimeError, match=match):
            gated_delta_rule(*args, **more)

    refused("q must be a CUDA tensor", 0, p["q"].cpu())
    refused("k must be a CUDA tensor", 1, p["k"].cpu())
    refused("Expected q", 0, p["q"].half())
    refused("Expected k", 1, p["k"].bfloat16())
    refused("Expected gate", 3, p["gate"].bfloat16())
    refused("q must have shape", 0, p["q"][0])
    refused("k must have the shape of q", 1, p["k"][:, :, :1])
    refused("v must have shape", 2, p["v"][:, :4])
    refused("multiple", 2, p["v"][:, :, :3])
    refused("gate must have shape", 3, p["gate"][:, :, :2])
    refused("beta must have shape", 4, p["beta"][:1])
    refused("seq_lens must be", seq_lens=torch.zeros(2, dtype=torch.int64, device="cuda"))
    refused("seq_lens must be", seq_lens=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused("initial_state must be", initial_state=p["initial"][:1])
    refused("initial_state must be", initial_state=p["initial"].bfloat16())
    wide = torch.zeros((2, 5, 2, 129), device="cuda")
    with pytest.raises(RuntimeError, match="larger than this operator takes"):
        gated_delta_rule(wide, wide, *good[2:])
    with pytest.raises(RuntimeError, match="larger than this operator takes"):
        gated_delta_rule(good[0], good[1], torch.zeros((2, 5, 4, 129), device="cuda"), *good[3:])
    with pytest.raises(RuntimeError, match="T > 0"):
        gated_delta_rule(*(x[:, :0] for x in good))
