"""Output layer with cross entropy, gated recurrence and AdamW against plain computations in 64 bits.

Tolerances follow from the number formats: a bound on the rounding of every product and sum is computed next to the
expected value, from the magnitudes that enter it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, EPS_HALVES, EPS16 = 2.0 ** -24, 2.0 ** -22, 2.0 ** -8     # half an ulp of 24 bits, a product of two halves, half an ulp of 8 bits
DTYPES = [torch.float32, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, want, bound, what=""):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / bound)[bad].max()), got[bad][:4], want[bad][:4])


# ------------------------------------------------------------------------------------------------------ cross entropy


def ce_problem(B, T, F, D, dtype, seed=1, lens=None):
    g = gen(seed)
    weight = torch.randn((F, D), generator=g, device="cuda") / math.sqrt(D)
    bias = torch.randn((F,), generator=g, device="cuda")
    targets = torch.randint(0, F, (B, T), generator=g, device="cuda", dtype=torch.int32)
    hidden = torch.randn((B, T, D), generator=g, device="cuda") + weight[targets.long()]
    if lens is None:
        lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[B // 2] = T
    else:
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    grad = torch.randn((B, T), generator=g, device="cuda")
    return hidden.to(dtype), weight.to(dtype), bias.to(dtype), targets, lens, grad


def ce_expected(hidden, weight, bias, targets, lens, grad):
    """Loss and gradients in 64 bits with bounds on what rounding may change."""
    B, T, D = hidden.shape
    F = weight.shape[0]
    x16 = hidden.dtype == torch.bfloat16
    live = (torch.arange(T, device="cuda") < lens[:, None]) & (targets >= 0) & (targets < F)
    h, w, b = hidden[live].double(), weight.double(), bias.double() if bias is not None else torch.zeros(F, dtype=torch.float64, device="cuda")
    y, g = targets[live].long(), grad[live].double()
    z = h @ w.T + b
    # products of bfloat16 are exact; sums of D + 1 terms in 32 bits in any order
    dz = (h.abs() @ w.abs().T + b.abs()) * ((0 if x16 else EPS_HALVES) + (D + 2) * EPS32)
    lse = torch.logsumexp(z, 1) if z.numel() else z.sum(1)
    loss = lse - z.gather(1, y[:, None])[:, 0]
    # exponentials to 2^-21, their arguments (up to |z - lse|) to an ulp, sums of F terms in a tree over tiles
    top = dz.amax(1) if z.numel() else dz.sum(1)
    reach = (z - lse[:, None]).abs()
    dloss = 2 * top + 2.0 ** -20 + 4 * EPS32 * (lse.abs() + loss.abs())
    p = torch.exp(z - lse[:, None])
    G = p * g[:, None]
    dp = p * (2 * top[:, None] + 2.0 ** -20 + 4 * EPS32 * reach)
    dG = dp * g.abs()[:, None]
    G.scatter_add_(1, y[:, None], -g[:, None])
    dG = dG + G.abs() * ((EPS16 if x16 else EPS_HALVES) + EPS32) + 2.0 ** -34 * (g.abs().max() if g.numel() else 0)
    n = max(1, h.shape[0])
    out = EPS16 if x16 else 0.0
    dh = G @ w
    bh = dG @ w.abs() + (G.abs() @ w.abs()) * ((0 if x16 else EPS_HALVES) + (F + 8) * EPS32) + out * dh.abs()
    dw = G.T @ h
    bw = dG.T @ h.abs() + (G.abs().T @ h.abs()) * ((0 if x16 else EPS_HALVES) + (n + 8) * EPS32) + out * dw.abs()
    db = G.sum(0)
    bb = dG.sum(0) + G.abs().sum(0) * (n + 8) * EPS32 + out * db.abs()

    def spread(x):
        full = torch.zeros((B, T) + x.shape[1:], dtype=torch.float64, device="cuda")
        full[live] = x
        return full

    tiny = 1e-30
    return {"loss": (spread(loss), spread(dloss) + tiny), "hidden": (spread(dh), spread(bh) + tiny), "weight": (dw, bw + tiny), "bias": (db, bb + tiny)}


def ce_run(hidden, weight, bias, targets, lens, grad):
    from i6_native_ops_amd.training import linear_cross_entropy
    leaves = [x.detach().requires_grad_() if x is not None else None for x in (hidden, weight, bias)]
    loss = linear_cross_entropy(leaves[0], leaves[1], targets, lens, bias=leaves[2])
    inputs = [x for x in leaves if x is not None]
    grads = torch.autograd.grad(loss, inputs, grad)
    return dict(zip(("loss", "hidden", "weight", "bias"), (loss.detach(),) + grads))


def ce_check(problem):
    want = ce_expected(*problem)
    got = ce_run(*problem)
    for k, x in got.items():
        assert x.dtype == (torch.float32 if k == "loss" else problem[0].dtype)
        close(x, *want[k], k)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,F,D", [
    (1, 1, 1, 1), (1, 1, 2, 3), (2, 50, 10, 64), (3, 7, 129, 65), (5, 61, 127, 128), (4, 130, 700, 33),
    (2, 200, 1201, 200), (8, 129, 264, 512), (300, 2, 40, 16), (1, 1000, 3, 640),
])
def test_cross_entropy_and_gradients(B, T, F, D, dtype):
    ce_check(ce_problem(B, T, F, D, dtype, seed=B + T + F + D))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_over_several_pieces_of_the_vocabulary(dtype):
    """Rows times classes beyond what a piece holds: several pieces, a last one that is not full, many ranges of rows."""
    ce_check(ce_problem(20, 1000, 5001, 72, dtype, seed=5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_rows_without_anything(dtype):
    """Sequences of no frames, frames without a target, and what stands there (NaN, infinities) is not looked at."""
    hidden, weight, bias, targets, lens, grad = ce_problem(6, 40, 77, 96, dtype, lens=[0, 40, 1, -3, 57, 17])
    targets[1, 3:9] = -1
    targets[4, ::2] = -100
    clean = hidden.clone()
    hidden[0] = float("nan")
    hidden[2, 1:] = float("inf")
    hidden[1, 3:9] = float("nan")
    hidden[4, ::2] = -float("inf")
    grad[0] = float("nan")
    grad[1, 3:9] = float("inf")
    clean_grad = torch.nan_to_num(grad, 0.0, 0.0, 0.0)
    targets_behind = targets.clone()
    targets_behind[0] = 10 ** 6          # behind the end: no target, whatever it says
    got = ce_run(hidden, weight, bias, targets_behind, lens, grad)
    want = ce_expected(clean, weight, bias, targets, lens, clean_grad)
    for k in got:
        close(got[k], *want[k], k)
    none = ce_run(hidden, weight, bias, targets, torch.zeros_like(lens), grad)
    assert all((x == 0).all() for x in none.values())


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_classes_that_are_ruled_out(dtype):
    """Biases of -inf and of the type's lowest value: no probability, no gradient, no NaN; whole tiles of them too."""
    hidden, weight, bias, targets, lens, grad = ce_problem(2, 30, 400, 64, dtype, lens=[30, 12])
    targets.fill_(350)
    bias[10:20] = torch.finfo(dtype).min
    bias[128:256] = -float("inf")
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    keep = torch.ones(400, dtype=torch.bool, device="cuda")
    keep[10:20] = keep[128:256] = False
    y = torch.full_like(targets, int(keep[:350].sum()))
    want = ce_expected(hidden, weight[keep].contiguous(), bias[keep].contiguous(), y, lens, grad)
    close(got["loss"], *want["loss"], "loss")
    close(got["hidden"], *want["hidden"], "hidden")
    close(got["weight"][keep], *want["weight"], "weight")
    close(got["bias"][keep], *want["bias"], "bias")
    assert (got["weight"][~keep] == 0).all() and (got["bias"][~keep] == 0).all()


def test_cross_entropy_large_and_small_values():
    """32-bit operands far from 1: the halves are scaled by the tensor's largest value; logits in the hundreds."""
    hidden, weight, bias, targets, lens, grad = ce_problem(2, 33, 90, 48, torch.float32, lens=[33, 20])
    ce_check((hidden * 1e12, weight * 1e-12, bias, targets, lens, grad * 1e-20))
    ce_check((hidden * 1e-25, weight * 1e27, bias * 50, targets, lens, grad * 1e8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_strides(dtype):
    hidden, weight, bias, targets, lens, grad = ce_problem(5, 21, 50, 64, dtype)
    plain = ce_run(hidden, weight, bias, targets, lens, grad)
    wide = torch.zeros((21, 5, 70), dtype=dtype, device="cuda")
    wide[:, :, 3:67] = hidden.transpose(0, 1)
    w_wide = torch.zeros((50, 67), dtype=dtype, device="cuda")
    w_wide[:, 1:65] = weight
    again = ce_run(wide.transpose(0, 1)[:, :, 3:67], w_wide[:, 1:65], bias, targets.T.contiguous().T, lens, grad.T.contiguous().T)
    columns = ce_run(hidden.transpose(1, 2).contiguous().transpose(1, 2), weight.T.contiguous().T, bias, targets, lens, grad)
    for k in plain:
        assert torch.equal(plain[k], again[k]) and torch.equal(plain[k], columns[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_without_bias_single_gradients_and_repeats(dtype):
    from i6_native_ops_amd.training import linear_cross_entropy
    hidden, weight, bias, targets, lens, grad = ce_problem(3, 100, 300, 40, dtype)
    want = ce_expected(hidden, weight, None, targets, lens, grad)
    got = ce_run(hidden, weight, None, targets, lens, grad)
    for k in got:
        close(got[k], *want[k], k)
    full = ce_run(hidden, weight, bias, targets, lens, grad)
    for i, k in enumerate(("hidden", "weight", "bias")):       # each gradient alone is the same, bit for bit, and so is a second run
        leaves = [x.detach().requires_grad_(i == j) for j, x in enumerate((hidden, weight, bias))]
        loss = linear_cross_entropy(leaves[0], leaves[1], targets, lens, bias=leaves[2])
        first, = torch.autograd.grad(loss, leaves[i], grad, retain_graph=True)
        second, = torch.autograd.grad(loss, leaves[i], grad)
        assert torch.equal(first, full[k]) and torch.equal(first, second), k
    # a gradient that is broadcast over the frames
    leaf = hidden.detach().requires_grad_()
    linear_cross_entropy(leaf, weight, targets, lens, bias=bias).sum().backward()
    close(leaf.grad, *ce_expected(hidden, weight, bias, targets, lens, torch.ones_like(grad))["hidden"], "ones")


def test_cross_entropy_gradient_against_differences():
    from i6_native_ops_amd.training import linear_cross_entropy
    hidden, weight, bias, targets, lens, grad = ce_problem(3, 40, 200, 64, torch.float32, lens=[40, 0, 25])
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    g, h = gen(9), 2.0 ** -6
    for i, k in enumerate(("hidden", "weight", "bias")):
        args = [hidden, weight, bias]
        v = torch.randn(args[i].shape, generator=g, device="cuda")
        v /= v.norm()
        sides = []
        for s in (h, -h):
            moved = list(args)
            moved[i] = args[i] + s * v
            sides.append((linear_cross_entropy(moved[0], moved[1], targets, lens, bias=moved[2]).double() * grad).sum())
        slope, want = float((sides[0] - sides[1]) / (2 * h)), float((got[k].double() * v).sum())
        # rounding of some hundred losses of size 10 over the step, and the third derivative's h^2 / 6
        assert abs(slope - want) < 1e-3 * max(1.0, abs(want)), (k, slope, want)


def test_cross_entropy_target_out_of_range():
    from i6_native_ops_amd import fbw
    from i6_native_ops_amd.training import check_status
    hidden, weight, bias, targets, lens, grad = ce_problem(4, 20, 30, 32, torch.float32, lens=[20, 20, 20, 20])
    fbw.set_status_mode("off")
    good = ce_run(hidden, weight, bias, torch.where(targets == targets[2, 5], targets, targets), lens, grad)
    bad_targets = targets.clone()
    bad_targets[2, 5] = 30
    bad = ce_run(hidden, weight, bias, bad_targets, lens, grad)
    torch.cuda.synchronize()
    fbw.set_status_mode("deferred")
    with pytest.raises(RuntimeError, match="sequence 2: target out of range"):
        check_status()
    check_status()
    mask = torch.ones((4, 20), dtype=torch.bool, device="cuda")
    mask[2, 5] = False
    assert torch.isnan(bad["loss"][2, 5]) and torch.isnan(bad["hidden"][2, 5]).all()
    assert torch.equal(bad["loss"][mask], good["loss"][mask])
    skipped = targets.clone()
    skipped[2, 5] = -1
    want = ce_expected(hidden, weight, bias, skipped, lens, grad)
    close(bad["weight"], *want["weight"], "weight")
    close(bad["bias"], *want["bias"], "bias")
    fbw.set_status_mode("sync")
    with pytest.raises(RuntimeError, match="sequence 2: target out of range"):
        ce_run(hidden, weight, bias, bad_targets, lens, grad)
    fbw.set_status_mode("deferred")


def test_cross_entropy_refusals():
    from i6_native_ops_amd.training import linear_cross_entropy
    hidden, weight, bias, targets, lens, _ = ce_problem(2, 5, 7, 8, torch.float32)
    for args, match in [
        ((hidden.cpu(), weight, targets, lens), "hidden must be a CUDA tensor"),
        ((hidden.half(), weight.half(), targets, lens), "Expected hidden"),
        ((hidden, weight.bfloat16(), targets, lens), "Expected weight"),
        ((hidden, weight[:, :7], targets, lens), "weight must have shape"),
        ((hidden, weight, targets.long(), lens), "Expected targets"),
        ((hidden, weight, targets[:, :4], lens), "targets must have shape"),
        ((hidden, weight, targets, lens.long()), "Expected seq_lens"),
        ((hidden, weight, targets, lens[:1]), "seq_lens must have shape"),
        ((hidden, weight, targets, lens, bias[:3]), "bias must be"),
        ((hidden, weight, targets, lens, bias.bfloat16()), "bias must be"),
        ((hidden[:, :0], weight, targets[:, :0], lens), "T > 0"),
        ((hidden[0], weight, targets, lens), "hidden must have shape"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            linear_cross_entropy(*args)


# --------------------------------------------------------------------------------------------------------- recurrence


def rec_problem(B, T, D, dtype, seed=1, lens=None, initial=True):
    g = gen(seed)
    x = torch.randn((B, T, D), generator=g, device="cuda").to(dtype)
    gate = (torch.randn((B, T, D), generator=g, device="cuda") * 2 + torch.linspace(-2, 6, D, device="cuda")).to(dtype)
    if lens is None:
        lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[B // 2] = T
    else:
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state = torch.randn((B, D), generator=g, device="cuda") if initial else None
    grads = torch.randn((B, T, D), generator=g, device="cuda").to(dtype), torch.randn((B, D), generator=g, device="cuda")
    return x, gate, lens, state, grads


def rec_expected(x, gate, lens, state, grads):
    """Frame by frame in 64 bits.  Errors of a few ulp per operation do not grow along the frames: every step is a mean of
    the state and the input, so they are summed with the weights the state itself has, at most 1 / (1 - f) of them."""
    B, T, D = x.shape
    xd, gd = x.double().cpu(), gate.double().cpu()
    n = (lens.long().clamp(0, T) if lens is not None else torch.full((B,), T, device="cuda")).cpu()[:, None]
    f, r = torch.sigmoid(gd), torch.sigmoid(-gd)
    s = state.double().cpu() if state is not None else torch.zeros(B, D, dtype=torch.float64)
    es = torch.zeros_like(s)
    unit = 8 * EPS32
    h, eh, before, eb = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    for t in range(T):
        live = t < n
        before[:, t], eb[:, t] = s, es
        es = torch.where(live, f[:, t] * es + unit * (f[:, t] * s.abs() + r[:, t] * xd[:, t].abs()), es)
        s = torch.where(live, f[:, t] * s + r[:, t] * xd[:, t], s)
        h[:, t], eh[:, t] = s * live, es * live
    out = EPS16 if x.dtype == torch.bfloat16 else 0.0
    want = {"h": (h, eh + out * h.abs()), "last": (s, es)}
    dh, d = grads[0].double().cpu(), grads[1].double().cpu()
    ed = torch.zeros_like(d)
    dx, ex, dg, eg = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    for t in reversed(range(T)):
        live = t < n
        ed = torch.where(live, ed + unit * (d.abs() + dh[:, t].abs()), ed)
        d = torch.where(live, d + dh[:, t], d)
        dx[:, t], ex[:, t] = d * r[:, t] * live, (ed + unit * d.abs()) * r[:, t]
        gap = before[:, t] - xd[:, t]
        dg[:, t] = d * gap * f[:, t] * r[:, t] * live
        eg[:, t] = (ed * gap.abs() + d.abs() * (eb[:, t] + unit * (before[:, t].abs() + xd[:, t].abs()))) * f[:, t] * r[:, t] + unit * dg[:, t].abs()
        ed = torch.where(live, f[:, t] * ed + unit * (f[:, t] * d).abs(), ed)
        d = torch.where(live, f[:, t] * d, d)
    want |= {"x": (dx, ex + out * dx.abs()), "gate": (dg, eg + out * dg.abs()), "initial": (d, ed)}
    return {k: (a.cuda(), 4 * b.cuda() + 1e-30) for k, (a, b) in want.items()}


def rec_run(x, gate, lens, state, grads):
    from i6_native_ops_amd.training import gated_recurrence
    leaves = [v.detach().requires_grad_() if v is not None else None for v in (x, gate, state)]
    h, last = gated_recurrence(leaves[0], leaves[1], lens, initial_state=leaves[2])
    inputs = [v for v in leaves if v is not None]
    got = torch.autograd.grad([h, last], inputs, list(grads))
    return dict(zip(("h", "last", "x", "gate", "initial"), (h.detach(), last.detach()) + got))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [
    (1, 1, 1), (3, 1, 130), (2, 2, 64), (5, 16, 33), (4, 17, 128), (3, 64, 65), (2, 65, 256), (7, 127, 129), (2, 129, 64), (3, 300, 70), (1, 700, 8), (300, 20, 64),
])
def test_recurrence_and_gradients(B, T, D, dtype):
    problem = rec_problem(B, T, D, dtype, seed=B + T + D)
    want, got = rec_expected(*problem), rec_run(*problem)
    for k in got:
        close(got[k], *want[k], k)
    from i6_native_ops_amd.training import gated_recurrence
    h, last = gated_recurrence(*problem[:3], initial_state=problem[3])       # without a gradient: the same bits
    assert torch.equal(h, got["h"]) and torch.equal(last, got["last"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,lens", [(1, 3000, None), (3, 2500, [2500, 0, 1300]), (2, 1025, [1, 1024])])
def test_recurrence_in_segments(B, T, lens, dtype):
    problem = rec_problem(B, T, 64, dtype, seed=T, lens=lens)
    want, got = rec_expected(*problem), rec_run(*problem)
    for k in got:
        close(got[k], *want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_frames_behind_the_end(dtype):
    """NaN and infinities there are not looked at; results are 0 there; sequences of no frames keep their state."""
    x, gate, lens, state, (dh, dl) = rec_problem(5, 150, 96, dtype, lens=[0, 150, 64, -1, 400])
    clean = rec_run(x, gate, lens, state, (dh, dl))
    behind = torch.arange(150, device="cuda") >= lens[:, None]
    for v, bad in ((x, float("nan")), (gate, float("inf")), (dh, float("nan"))):
        v[behind] = bad
    got = rec_run(x, gate, lens, state, (dh, dl))
    for k in got:
        assert torch.equal(got[k], clean[k]), k
    for k in ("h", "x", "gate"):
        assert (got[k][behind] == 0).all()
    assert torch.equal(got["last"][0], state[0]) and torch.equal(got["initial"][3], dl[3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_gates_that_are_shut_or_open(dtype):
    """Gates of the type's extremes and infinities: the state is kept or replaced exactly."""
    x, gate, lens, state, grads = rec_problem(2, 40, 64, dtype, lens=[40, 40])
    big = torch.finfo(dtype).max
    gate[0], gate[1] = big, -big
    gate[0, 7], gate[1, 7] = float("inf"), -float("inf")
    got = rec_run(x, gate, lens, state, grads)
    assert torch.equal(got["last"][0], state[0]) and torch.equal(got["h"][1], x[1])
    assert (got["gate"] == 0).all() and (got["x"][0] == 0).all() and torch.equal(got["x"][1][:-1], grads[0][1][:-1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_strides_and_missing_parts(dtype):
    from i6_native_ops_amd.training import gated_recurrence
    x, gate, lens, state, grads = rec_problem(4, 90, 66, dtype)
    want = rec_run(x, gate, lens, state, grads)
    both = torch.stack([x, gate], dim=2)                                       # interleaved, as one projection gives them
    odd = torch.zeros((90, 4, 67), dtype=dtype, device="cuda")                 # not aligned to pairs
    odd[:, :, 1:] = x.transpose(0, 1)
    for xs, gs in ((both[:, :, 0], both[:, :, 1]), (odd.transpose(0, 1)[:, :, 1:], gate), (x.transpose(1, 2).contiguous().transpose(1, 2), gate)):
        got = rec_run(xs, gs, lens, state, grads)
        for k in got:
            assert torch.equal(got[k], want[k]), k
    leaf = x.detach().requires_grad_()
    h, last = gated_recurrence(leaf, gate, lens)
    zero = rec_expected(x, gate, lens, None, (torch.ones_like(x), torch.zeros_like(state)))
    h.sum().backward()                                                          # no state, no gradient of the last state, a broadcast one of h
    close(leaf.grad, *zero["x"], "x")
    close(last.detach(), *zero["last"], "last")
    leaf.grad = None
    h, last = gated_recurrence(leaf, gate, initial_state=state)
    last.sum().backward()
    close(leaf.grad, *rec_expected(x, gate, None, state, (torch.zeros_like(x), torch.ones_like(state)))["x"], "last alone")


def test_recurrence_frame_by_frame():
    """Streams of single frames, and of a few, come to the same as the whole sequence."""
    from i6_native_ops_amd.training import gated_recurrence
    x, gate, _, state, _ = rec_problem(6, 33, 130, torch.float32)
    h, last = gated_recurrence(x, gate, initial_state=state)
    for step in (1, 5):
        s, parts = state, []
        for t in range(0, 33, step):
            part, s = gated_recurrence(x[:, t:t + step], gate[:, t:t + step], initial_state=s)
            parts.append(part)
        assert torch.allclose(torch.cat(parts, 1), h, rtol=1e-5, atol=1e-6) and torch.allclose(s, last, rtol=1e-5, atol=1e-6)


def test_recurrence_gradient_against_differences():
    from i6_native_ops_amd.training import gated_recurrence
    x, gate, lens, state, grads = rec_problem(2, 60, 64, torch.float32, lens=[60, 33])
    got = rec_run(x, gate, lens, state, grads)
    g, h = gen(4), 2.0 ** -5
    for i, k in enumerate(("x", "gate", "initial")):
        args = [x, gate, state]
        v = torch.randn(args[i].shape, generator=g, device="cuda")
        v /= v.norm()
        sides = []
        for s in (h, -h):
            moved = list(args)
            moved[i] = args[i] + s * v
            out, last = gated_recurrence(moved[0], moved[1], lens, initial_state=moved[2])
            sides.append((out.double() * grads[0]).sum() + (last.double() * grads[1]).sum())
        slope, want = float((sides[0] - sides[1]) / (2 * h)), float((got[k].double() * v).sum())
        assert abs(slope - want) < 1e-3 * max(1.0, abs(want)), (k, slope, want)


def test_recurrence_refusals():
    from i6_native_ops_amd.training import gated_recurrence
    x, gate, lens, state, _ = rec_problem(2, 5, 8, torch.float32)
    for args, match in [
        ((x.cpu(), gate), "x must be a CUDA tensor"),
        ((x.half(), gate.half()), "Expected x"),
        ((x, gate.bfloat16()), "Expected gate"),
        ((x, gate[:, :4]), "gate must have the shape"),
        ((x[0], gate[0]), "x must have shape"),
        ((x, gate, lens.long()), "seq_lens must be"),
        ((x, gate, lens[:1]), "seq_lens must be"),
        ((x, gate, lens, state[:, :3]), "initial_state must be"),
        ((x, gate, lens, state.bfloat16()), "initial_state must be"),
        ((x[:, :0], gate[:, :0]), "T > 0"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            gated_recurrence(*args)


# -------------------------------------------------------------------------------------------------------------- AdamW

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (255,), (256,), (257,), (17, 31), (4096,), (4097,), (3, 5001), (0,)]


def adamw_expected(p, g, m, v, step):
    (b1, b2), lr = HYPER["betas"], HYPER["lr"]
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    ahead = (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + HYPER["eps"])
    return p * (1 - lr * HYPER["weight_decay"]) - lr * ahead, m, v, ahead


def shifted(x, by):
    """The same values at an address that is off by some elements."""
    room = torch.empty(x.numel() + by, dtype=x.dtype, device="cuda")
    room[by:] = x.reshape(-1)
    return room[by:].view(x.shape)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_adamw_states_in_32_bits(dtype, off):
    from i6_native_ops_amd.training import adamw_step
    g = gen(3)
    p, gr, m, v = ([shifted(torch.randn(s, generator=g, device="cuda").to(t), off) for s in SIZES * 12] for t in (dtype, dtype, torch.float32, torch.float32))
    for x in v:
        x.abs_()
    want = [adamw_expected(*x, 7) for x in zip(p, gr, m, v)]
    adamw_step(p, gr, m, v, step=7, **HYPER)       # more tensors than one launch takes
    for i, (wp, wm, wv, ahead) in enumerate(want):
        # m cancels; p: a dozen roundings of the update and one of the result
        close(m[i], wm, 1e-6 * (wm.abs() + gr[i].double().abs() * 0.1) + 1e-30, i)
        close(v[i], wv, 1e-6 * wv + 1e-30, i)
        bound = 2e-6 * HYPER["lr"] * (ahead.abs() + 10) + 4 * EPS32 * wp.abs() + (EPS16 * wp.abs() if dtype == torch.bfloat16 else 0)
        close(p[i], wp, bound, i)


def grid(dev="cuda"):
    """All values of the 8-bit format that are not negative, and their order."""
    x = torch.arange(127, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).double()
    assert (x[1:] > x[:-1]).all() and x[-1] == 448
    return x


def neighbours(y):
    values = grid()
    i = (torch.searchsorted(values, y.contiguous(), right=True) - 1).clamp(0, 126)
    return values[i], values[(i + 1).clamp(max=126)]


@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_adamw_states_in_8_bits(dtype, off):
    from i6_native_ops_amd.training import BLOCK, adamw_step
    g = gen(5)
    sizes = SIZES[:-1] * 8 + [(0,)]
    p, gr = ([shifted(torch.randn(s, generator=g, device="cuda").to(dtype), off) for s in sizes] for _ in range(2))
    m, v, scales = [], [], []
    for s in sizes:
        n, blocks = math.prod(s), -(-math.prod(s) // BLOCK)
        m.append(shifted((torch.randn(s, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), off).view(torch.float8_e4m3fn))
        v.append(shifted((torch.randn(s, generator=g, device="cuda") * 100).abs().clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8), off).view(torch.float8_e4m3fn))
        scales.append((torch.rand(blocks, generator=g, device="cuda") / 100, torch.rand(blocks, generator=g, device="cuda") / 100))

    def held(x, s):
        return x.double() * s.double().repeat_interleave(BLOCK)[:x.numel()].view(x.shape)

    want = [adamw_expected(a, b, held(c, s[0]), held(d, s[1]).square(), 11) for a, b, c, d, s in zip(p, gr, m, v, scales)]
    adamw_step(p, gr, m, v, step=11, scales=scales, **HYPER)
    for i, (wp, wm, wv, ahead) in enumerate(want):
        bound = 2e-6 * HYPER["lr"] * (ahead.abs() + 10) + 4 * EPS32 * wp.abs() + (EPS16 * wp.abs() if dtype == torch.bfloat16 else 0)
        close(p[i], wp, bound, i)
        for x, s, exact in ((m[i], scales[i][0], wm), (v[i], scales[i][1], wv.sqrt())):
            if not x.numel():
                continue
            blocks = torch.nn.functional.pad(exact.reshape(-1), (0, -exact.numel() % BLOCK)).view(-1, BLOCK)
            close(s, blocks.abs().amax(1) / 448, 1e-6 * blocks.abs().amax(1) / 448 + 1e-30, i)
            y = exact.abs() / s.double().repeat_interleave(BLOCK)[:x.numel()].view(x.shape)
            low, high = neighbours(y)
            near = 1e-5 * (high - low) + 1e-5 * y
            got = x.double().abs()
            # one of the two neighbours, the sign kept, the smallest value instead of 0 for a root
            assert (((got == low) | (got == high)) | ((y - low).abs() < near) | ((high - y).abs() < near)).all(), i
            assert (x.double() * exact >= 0).all()
        assert (v[i].double()[wv > 0] > 0).all()


def test_adamw_8_bits_keep_their_means():
    """Rounding to 8 bits must not let a moment drift: over some hundred steps with gradients of one size, the second moment stays
    where it is, although a step moves it by less than half the distance of the 8-bit values."""
    from i6_native_ops_amd.training import adamw_step
    n, b2 = 256 * 64, 0.999
    g = gen(8)
    size = torch.exp(torch.randn(n, generator=g, device="cuda"))
    p = torch.zeros(n, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    scales = (torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))
    exact = torch.zeros(n, dtype=torch.float64, device="cuda")
    first = torch.zeros(n, dtype=torch.float64, device="cuda")
    for step in range(1, 601):
        grad = size * (1.0 + 0.5 * torch.randn(n, generator=g, device="cuda"))
        adamw_step([p], [grad], [m], [v], step=step, lr=1e-3, betas=(0.9, b2), scales=[scales])
        exact = b2 * exact + (1 - b2) * grad.double().square()
        first = 0.9 * first + 0.1 * grad.double()
    held_v = (v.double() * scales[1].double().repeat_interleave(256)).square()
    held_m = m.double() * scales[0].double().repeat_interleave(256)
    # single values carry the noise of their last roundings (an eighth of the value at most each), the mean over 16384 does not
    assert abs(float((held_v / exact).mean()) - 1) < 0.02, float((held_v / exact).mean())
    assert abs(float((held_m / size.double()).mean() / (first / size.double()).mean()) - 1) < 0.01


def test_adamw_infinities_and_zeros_in_8_bits():
    from i6_native_ops_amd.training import adamw_step
    for bits in (32, 8):
        p, g = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
        g[300] = float("nan")
        if bits == 8:
            m, v = (torch.zeros(1024, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
            scales = [(torch.ones(4, device="cuda"), torch.ones(4, device="cuda"))]
        else:
            m, v, scales = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda"), None
        adamw_step([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.5, scales=scales)
        bad = torch.isnan(p)
        assert bad.sum() == 1 and bad[300]                                  # the parameter of the bad gradient alone
        assert (p[~bad] == 0.75).all()
        assert torch.isnan(m.float()[300]) and (m.float()[:256] == 0).all() and (v.float()[512:] == 0).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_class(bits):
    """The optimiser trains, follows torch's with states in 32 bits, and goes on from a saved state."""
    from i6_native_ops_amd.training import AdamW
    torch.manual_seed(0)
    nets = [torch.nn.Sequential(torch.nn.Linear(40, 60), torch.nn.Tanh(), torch.nn.Linear(60, 3)).cuda() for _ in range(3)]
    for n in nets[1:]:
        n.load_state_dict(nets[0].state_dict())
    opts = [torch.optim.AdamW(nets[0].parameters(), lr=1e-3, weight_decay=0.02), AdamW(nets[1].parameters(), lr=1e-3, weight_decay=0.02, state_bits=bits),
            AdamW(nets[2].parameters(), lr=1e-3, weight_decay=0.02, state_bits=bits)]
    x = torch.randn(64, 40, device="cuda")
    y = torch.randn(64, 3, device="cuda")

    def train(net, opt, n):
        for _ in range(n):
            opt.zero_grad()
            loss = (net(x) - y).square().mean()
            loss.backward()
            opt.step()
        return float(loss.detach())

    losses = [train(nets[i], opts[i], 20) for i in (0, 1, 2)]
    start = float((nets[0](x) - y).square().mean().detach())
    assert abs(losses[1] - losses[0]) < (1e-4 if bits == 32 else 2e-2) * start
    saved = opts[1].state_dict()
    nets[2].load_state_dict(nets[1].state_dict())
    opts[2].load_state_dict(saved)
    first = opts[2].state[next(iter(nets[2].parameters()))]
    assert first["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32) and first["step"] == 20
    train(nets[1], opts[1], 3), train(nets[2], opts[2], 3)
    for a, b in zip(nets[1].parameters(), nets[2].parameters()):
        assert torch.equal(a, b)


def test_adamw_refusals():
    from i6_native_ops_amd.training import AdamW, adamw_step
    p, m8 = torch.ones(10, device="cuda"), torch.zeros(10, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.ones(1, device="cuda")
    for args, kw, match in [
        (([p.cpu()], [p], [p], [p]), {}, "params"),
        (([p], [p.half()], [p], [p]), {}, "grads"),
        (([p], [p[:4]], [p], [p]), {}, "grads"),
        (([p], [p], [p.bfloat16()], [p]), {}, "exp_avgs"),
        (([p], [p], [p], [p, p]), {}, "same length"),
        (([p], [p], [m8], [p]), {"scales": [(s, s)]}, "exp_avg_sqs"),
        (([p], [p], [m8], [m8]), {}, "scales"),
        (([p], [p], [p], [p]), {"scales": [(s, s)]}, "scales"),
        (([p], [p], [m8], [m8]), {"scales": [(s, torch.ones(2, device="cuda"))]}, "scales"),
        (([torch.ones(4, 6, device="cuda").T], [p], [p], [p]), {}, "contiguous"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            adamw_step(*args, step=1, lr=1e-3, **kw)
    with pytest.raises(RuntimeError, match="invalid argument"):
        adamw_step([p], [p], [p], [p], step=0, lr=1e-3)
    with pytest.raises(RuntimeError, match="invalid argument"):
        adamw_step([p], [p], [p], [p], step=1, lr=1e-3, betas=(1.0, 0.9))
    with pytest.raises(ValueError):
        AdamW([p], state_bits=16)


# ------------------------------------------------------------------------------------------------------------ streams


def test_operators_on_another_stream_and_in_a_graph():
    """The current stream is the one that is used; all three can be captured, and replays with new inputs in the same buffers give
    what an eager call gives."""
    from i6_native_ops_amd.training import adamw_step, gated_recurrence, linear_cross_entropy
    hidden, weight, bias, targets, lens, grad = ce_problem(4, 50, 70, 64, torch.float32, lens=[50, 40, 3, 0])
    x, gate, _, state, _ = rec_problem(4, 50, 64, torch.float32)
    p, m, v = torch.randn(70, 64, device="cuda"), torch.zeros(70, 64, device="cuda"), torch.zeros(70, 64, device="cuda")

    def work(params, mm, vv):
        h, last = gated_recurrence(x, gate, lens, initial_state=state)
        leaf, w = (h + hidden).detach().requires_grad_(), params.detach().requires_grad_()
        loss = linear_cross_entropy(leaf, w, targets, lens, bias=bias)
        dh, dw = torch.autograd.grad(loss, [leaf, w], grad)
        adamw_step([params], [dw], [mm], [vv], step=3, lr=1e-2)
        return [h, last, loss.detach(), dh, dw]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    start = (p.clone(), m.clone(), v.clone())
    with torch.cuda.stream(side):
        held = tuple(s.clone() for s in start)
        on_side = work(*held)
    torch.cuda.current_stream().wait_stream(side)
    here = tuple(s.clone() for s in start)
    eager = work(*here)
    for a, b in zip(on_side + list(held), eager + list(here)):
        assert torch.equal(a, b)

    buffers = tuple(s.clone() for s in start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work(*buffers)
    for turn in range(3):
        hidden.copy_(torch.randn(hidden.shape, generator=gen(turn), device="cuda"))
        gate.mul_(0.9)
        for b, s in zip(buffers, start):
            b.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        again = tuple(s.clone() for s in start)
        want = work(*again)
        for a, b in zip(captured + list(buffers), want + list(again)):
            assert torch.equal(a, b), turn


def test_gradients_of_gradients_are_refused():
    from i6_native_ops_amd.training import gated_recurrence, linear_cross_entropy
    hidden, weight, bias, targets, lens, grad = ce_problem(2, 5, 7, 8, torch.float32)
    leaf = hidden.detach().requires_grad_()
    got, = torch.autograd.grad(linear_cross_entropy(leaf, weight, targets, lens, bias=bias), leaf, grad.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="linear_cross_entropy can be differentiated once"):
        got.sum().backward()
    leaf = hidden.detach().requires_grad_()
    h, _ = gated_recurrence(leaf, hidden)
    got, = torch.autograd.grad(h, leaf, torch.ones_like(h).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="gated_recurrence can be differentiated once"):
        got.sum().backward()


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_large_steps(bits):
    """Steps that go past the caches come to the same as small ones, bit for bit: the large tensor repeats a small one."""
    from i6_native_ops_amd.training import adamw_step
    small, times = 1 << 16, 640
    g = gen(2)
    p, gr = torch.randn(small, generator=g, device="cuda"), torch.randn(small, generator=g, device="cuda")
    if bits == 8:
        m, v = (torch.zeros(small, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        scales = [(torch.ones(small // 256, device="cuda"), torch.ones(small // 256, device="cuda"))]
    else:
        m, v, scales = torch.zeros(small, device="cuda"), torch.zeros(small, device="cuda"), None

    def repeated(x):
        return x.view(torch.uint8).repeat(times).view(x.dtype)

    big = [repeated(x) for x in (p, gr, m, v)]
    big_scales = [tuple(repeated(s) for s in pair) for pair in scales] if scales else None
    adamw_step([p], [gr], [m], [v], step=1, lr=1e-2, scales=scales)
    adamw_step(*([x] for x in big), step=1, lr=1e-2, scales=big_scales)
    for a, b in zip([p, m, v] + (list(scales[0]) if scales else []), [big[0], big[2], big[3]] + (list(big_scales[0]) if scales else [])):
        assert torch.equal(repeated(a).view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,F,D", [(1, 1, 4099, 31), (2, 37, 2500, 64), (3, 300, 1030, 520)])
def test_cross_entropy_of_few_rows_over_many_classes(B, T, F, D, dtype):
    """The gradient of the features is summed over ranges of the classes."""
    problem = ce_problem(B, T, F, D, dtype, seed=F)
    problem[3][0, 0] = -1
    ce_check(problem)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_of_large_tiles(dtype):
    """Sizes whose products all take the large tiles, none of them full."""
    problem = ce_problem(3, 400, 7700, 450, dtype, lens=[400, 377, 330], seed=11)
    problem[3][1, 5:50] = -1
    ce_check(problem)


@pytest.mark.parametrize("B,T,F,D,dtype", [
    (9, 1000, 30001, 40, torch.bfloat16), (9, 1000, 15001, 40, torch.float32), (33, 1000, 9001, 24, torch.bfloat16), (33, 1000, 4501, 24, torch.float32),
])
def test_cross_entropy_of_pieces_with_ranges_of_classes_and_without(B, T, F, D, dtype):
    """More than one piece of the vocabulary; the gradient of the features is summed over ranges of each, or in one."""
    ce_check(ce_problem(B, T, F, D, dtype, seed=F, lens=[T] * (B - 1) + [3]))


def test_cross_entropy_wide_features():
    """As many features as are taken, in a batch of few frames; one more is refused."""
    from i6_native_ops_amd.training import linear_cross_entropy
    problem = ce_problem(1, 9, 300, 1 << 14, torch.bfloat16)
    ce_check(problem)
    with pytest.raises(RuntimeError, match="larger than"):
        linear_cross_entropy(torch.zeros(1, 9, (1 << 14) + 1, device="cuda"), torch.zeros(600, (1 << 14) + 1, device="cuda"), problem[3], problem[4])
