"""Log probabilities of targets, entropies and alternatives against 64 bits.  Bounds: an exponential is right to 2^-21 and the rounding of its argument,
sums add up to 64 terms one after another and then pairs; they are added up next to the expected values, from the terms that enter them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8
DTYPES = [torch.float32, torch.bfloat16]
INF = float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def problem(B, T, F, k, dtype, seed=1, lens=None, size=3.0):
    g = gen(seed)
    logits = (torch.randn((B, T, F), generator=g, device="cuda") * size)
    targets = torch.randint(0, F, (B, T), generator=g, device="cuda", dtype=torch.int32)
    # from frames that know nothing to frames whose others' shares are far below 2^-24
    logits.scatter_add_(2, targets.long()[:, :, None], torch.rand((B, T, 1), generator=g, device="cuda") * 30)
    if lens is None:
        lens = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[B // 2] = T
    else:
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    grads = [torch.randn(shape, generator=g, device="cuda") for shape in ((B, T), (B, T), (B, T, k))]
    return logits.to(dtype), targets, lens, k, grads


def expected(logits, targets, lens, k, grads):
    """{name: (values, bounds)}; whole numbers without a bound.  Frames of -inf alone as the documentation says."""
    B, T, F = logits.shape
    live = torch.arange(T, device="cuda") < lens[:, None]
    z = torch.where(live[:, :, None], logits.detach().double(), 0.0)
    m, first = z.max(2, keepdim=True)
    empty = (m == -INF)
    m = torch.where(empty, 0.0, m)
    d = z - m
    e = d.exp()
    others = e.scatter(2, first, 0.0)
    steps = 64 + 2 * math.ceil(F / (512 * 48)) * 48
    reach = torch.where(e > 0, d.abs(), 0.0)
    rest = others.sum(2, keepdim=True)
    total, log_total = 1 + rest, torch.log1p(rest)
    e1 = EPS32 * (others * (4 * reach + steps)).sum(2, keepdim=True) / total
    moment = (e * reach).sum(2, keepdim=True) / total
    e2 = EPS32 * (e * reach * (4 * reach + steps)).sum(2, keepdim=True) / total
    log_p = d - log_total
    bound_p = EPS32 * (2 * d.abs() + 4 * log_total + 2 * log_p.abs()) + e1
    entropy, bound_e = log_total + moment, EPS32 * 8 * (log_total + moment) + e1 * (1 + moment) + e2
    log_p, bound_p = torch.where(empty, -INF, log_p), torch.where(empty | (log_p == -INF), 0.0, bound_p)
    entropy, bound_e = torch.where(empty, 0.0, entropy), torch.where(empty, 0.0, bound_e)
    y = targets.long()
    has = live & (y >= 0)
    index = y.clamp(min=0)[:, :, None]
    classes = torch.sort(z, dim=2, descending=True, stable=True)[1][:, :, :k]
    tiny = 1e-37
    out = {"log_prob": (torch.where(has, log_p.gather(2, index)[:, :, 0], 0.0), bound_p.gather(2, index)[:, :, 0] + tiny),
           "entropy": (torch.where(live, entropy[:, :, 0], 0.0), bound_e[:, :, 0] + tiny),
           "top": (torch.where(live[:, :, None], log_p.gather(2, classes), 0.0), bound_p.gather(2, classes) + tiny),
           "classes": (torch.where(live[:, :, None], classes, -1), None)}
    gl, ge, gt = (torch.where(live.view(B, T, *[1] * (g.dim() - 2)), g.double(), 0.0) for g in grads)
    gl = torch.where(has, gl, 0.0)[:, :, None]
    p = torch.where(empty, 0.0, log_p.exp())
    finite = torch.where(p > 0, log_p, 0.0)
    by = gl + gt.sum(2, keepdim=True) + ge[:, :, None] * (finite + entropy)
    size = gl.abs() + gt.abs().sum(2, keepdim=True) + ge[:, :, None].abs() * (finite.abs() + entropy)
    grad = (-p * by).scatter_add_(2, index, gl).scatter_add_(2, classes, gt)
    relative = EPS32 * (4 * finite.abs() + 64) + bound_p
    bound = p * (size * (relative + 72 * EPS32) + ge[:, :, None].abs() * (bound_p + bound_e)) + EPS32 * 2 * grad.abs()
    grad, bound = torch.where(live[:, :, None] & ~empty, grad, 0.0), torch.where(empty, 0.0, bound)
    bound = bound + 2.0 ** -126 * (size + 1)       # 32-bit numbers end at 2^-126: a share below it may be 0, and it is multiplied by at most `size`
    if logits.dtype == torch.bfloat16:
        bound = bound + (EPS16 + EPS32) * (grad.abs() + bound)
    out["logits"] = (grad, bound + tiny)
    return out


def run(logits, targets, lens, k, grads):
    from i6_native_ops_amd.training import target_log_probs
    leaf = logits.detach().requires_grad_()
    got = target_log_probs(leaf, targets, lens, alternatives=k)
    grad, = torch.autograd.grad(got[:3] if k else got[:2], leaf, grads if k else grads[:2])
    plain = target_log_probs(logits, targets, lens, alternatives=k)
    assert all(torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b) for a, b in zip(got, plain))
    return dict(zip(("log_prob", "entropy", "top", "classes"), (x.detach() for x in got))) | {"logits": grad}


def check(got, want):
    for n, (w, bound) in want.items():
        x = got[n]
        assert x.shape == w.shape, n
        if bound is None:
            assert x.dtype == torch.int32 and torch.equal(x.long(), w.long()), (n, x[x != w][:5], w[x != w][:5])
            continue
        same = x.double() == w                      # infinities among them
        bad = ~same & ~((x.double() - w).abs() <= bound)
        assert not bad.any(), (n, int(bad.sum()), x[bad][:4], w[bad][:4], bound[bad][:4])


SIZES = [(1, 1, 1, 1), (1, 1, 2, 0), (3, 5, 10, 3), (2, 7, 63, 63), (2, 7, 264, 5), (3, 3, 511, 64), (2, 3, 513, 8), (2, 3, 1537, 33), (2, 2, 5001, 4), (2, 2, 6145, 7), (2, 3, 12001, 16),
         (1, 2, 12300, 64), (1, 3, 24577, 3), (1, 2, 70001, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,F,k", SIZES)
def test_values_and_gradients(B, T, F, k, dtype):
    p = problem(B, T, F, k, dtype, seed=B + T + F)
    check(run(*p), expected(*p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [9, 700, 5000, 13000, 30001])
def test_classes_that_are_ruled_out(F, dtype):
    """-inf, the type's lowest value, frames of nothing else, targets among them."""
    logits, targets, lens, k, grads = problem(2, 6, F, 4, dtype, lens=[6, 5])
    lowest = torch.finfo(dtype).min
    logits[0, 0, :] = -INF
    logits[0, 1, 3:] = -INF
    logits[0, 2, 1:] = lowest
    logits[0, 3, ::2] = -INF
    logits[0, 4, : F - 2] = -INF
    logits[0, 5, :] = lowest
    targets[0, 3] = 0
    targets[0, 1] = F - 1
    targets[1, 2] = -1
    logits[1, 5] = float("nan")             # behind the end
    check(run(logits, targets, lens, k, grads), expected(logits, targets, lens, k, grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F,k", [(50, 7), (700, 64), (2600, 64), (12001, 9), (30001, 64)])
def test_equal_scores_have_the_lowest_index_first(F, k, dtype):
    logits, targets, lens, _, grads = problem(1, 8, F, k, dtype, lens=[8])
    logits[0, 0] = 1.5
    logits[0, 1] = 0.0
    logits[0, 1, ::3] = -0.0
    logits[0, 2] = (torch.arange(F, device="cuda") % 5).to(dtype)
    logits[0, 3] = torch.arange(F, device="cuda").float().mul(1 / 64).to(dtype)            # rising: neighbouring classes have the best scores
    logits[0, 4] = -torch.arange(F, device="cuda").float().mul(1 / 64).to(dtype)
    logits[0, 5] = torch.where(torch.arange(F, device="cuda") % 256 < 4, 4.0, 0.0).to(dtype)
    logits[0, 6] = -INF
    logits[0, 6, F // 2:] = -7.25
    logits[0, 7] = torch.round(logits[0, 7])
    got = run(logits, targets, lens, k, grads)
    want = expected(logits, targets, lens, k, grads)
    # more than one largest score: the bound above is for one, and the others' part of it is exact here
    check(got, want)


def test_confident_frames_keep_their_small_losses():
    logits = torch.zeros((1, 3, 1000), device="cuda")
    logits[0, 0, 5], logits[0, 1, 5], logits[0, 2, 5] = 30.0, 60.0, 90.0
    from i6_native_ops_amd.training import target_log_probs
    log_prob, entropy, _, _ = target_log_probs(logits, torch.full((1, 3), 5, dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"))
    for t, x in enumerate((30.0, 60.0, 90.0)):
        want = math.log1p(999 * math.exp(-x))
        # 32-bit numbers end at 2^-126, 1.2e-38: each of 999 exponentials below it (exp(-90) is 8e-40) may be 0
        assert abs(float(log_prob[0, t]) + want) <= want * 200 * EPS32 + 999 * 2.0 ** -126
        want = want + 999 * x * math.exp(-x) / (1 + 999 * math.exp(-x))
        assert abs(float(entropy[0, t]) - want) <= want * 500 * EPS32 + 999 * (1 + x) * 2.0 ** -126


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [20, 3000, 40000])
def test_frames_that_are_no_distribution(F, dtype):
    logits, targets, lens, k, grads = problem(1, 5, F, 3, dtype, lens=[5])
    logits[0, 1, F // 2] = float("nan")
    logits[0, 3, F - 1] = INF
    logits[0, 4] = float("nan")
    got = run(logits, targets, lens, k, grads)
    for t in (1, 3, 4):
        assert all(torch.isnan(got[n][0, t]).all() for n in ("log_prob", "entropy", "top", "logits")) and (got["classes"][0, t] == -1).all()
    want = expected(logits.nan_to_num(0.0, 0.0), targets, lens, k, grads)
    keep = torch.tensor([0, 2], device="cuda")
    check({n: x[:, keep] for n, x in got.items()}, {n: (w[:, keep], b[:, keep] if b is not None else None) for n, (w, b) in want.items()})


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_repeats_and_single_gradients(dtype):
    from i6_native_ops_amd.training import target_log_probs
    logits, targets, lens, k, grads = problem(3, 9, 1000, 5, dtype)
    full = run(logits, targets, lens, k, grads)
    wide = torch.zeros((9, 3, 1011), dtype=dtype, device="cuda")
    wide[:, :, 3:1003] = logits.transpose(0, 1)
    again = run(wide.transpose(0, 1)[:, :, 3:1003], targets.T.contiguous().T, lens, k, grads)
    columns = run(logits.transpose(1, 2).contiguous().transpose(1, 2), targets, lens, k, grads)
    for n in full:
        # which thread has which score depends on where a row begins, and with it the order of its sums
        if n == "classes":
            assert torch.equal(full[n], again[n]) and torch.equal(full[n], columns[n])
    check(again, expected(logits, targets, lens, k, grads))
    check(columns, expected(logits, targets, lens, k, grads))
    repeat = run(logits, targets, lens, k, grads)
    assert all(torch.equal(full[n], repeat[n]) for n in full)
    leaf = logits.detach().requires_grad_()
    got = target_log_probs(leaf, targets, lens, alternatives=k)
    assert not got[3].requires_grad
    for i in range(3):
        one = [torch.zeros_like(g) for g in grads]
        one[i] = grads[i]
        grad, = torch.autograd.grad(got[i], leaf, grads[i], retain_graph=True)
        assert torch.equal(grad, run(logits, targets, lens, k, one)["logits"]), i
    # broadcast gradients, and targets that are among the alternatives
    best = got[3][:, :, 1].contiguous()
    log_prob, _, top, _ = target_log_probs(leaf, torch.where(best >= 0, best, 0), lens, alternatives=k)
    grad, = torch.autograd.grad(log_prob.sum() + 2 * top.sum(), leaf)
    ones = [torch.ones_like(grads[0]), torch.zeros_like(grads[1]), 2 * torch.ones_like(grads[2])]
    check({"logits": grad}, {"logits": expected(logits, torch.where(best >= 0, best, 0), lens, k, ones)["logits"]})


def test_gradient_against_differences():
    from i6_native_ops_amd.training import target_log_probs
    logits, targets, lens, k, grads = problem(2, 5, 40, 3, torch.float32, lens=[5, 3], size=1.0)
    got = run(logits, targets, lens, k, grads)["logits"]
    g, h = gen(3), 2.0 ** -8
    v = torch.randn(logits.shape, generator=g, device="cuda")
    v /= v.norm()
    sides = []
    for s in (h, -h):
        out = target_log_probs(logits + s * v, targets, lens, alternatives=k)
        sides.append(sum((x.double() * y).sum() for x, y in zip(out[:3], grads)))
    slope, want = float((sides[0] - sides[1]) / (2 * h)), float((got.double() * v).sum())
    # forty values of size 30 rounded to 2^-19, over 2^-7; third derivatives of size 1
    assert abs(slope - want) < 2e-3 * max(1.0, abs(want)), (slope, want)


@pytest.mark.parametrize("F", [40, 3000])
def test_target_out_of_range(F):
    from i6_native_ops_amd import fbw
    from i6_native_ops_amd.training import check_status
    logits, targets, lens, k, grads = problem(4, 20, F, 2, torch.float32, lens=[20, 20, 20, 20])
    good = run(logits, targets, lens, k, grads)
    bad_targets = targets.clone()
    bad_targets[2, 5] = F
    fbw.set_status_mode("off")
    bad = run(logits, bad_targets, lens, k, grads)
    torch.cuda.synchronize()
    fbw.set_status_mode("deferred")
    with pytest.raises(RuntimeError, match="sequence 2: target out of range"):
        check_status()
    check_status()
    mask = torch.ones((4, 20), dtype=torch.bool, device="cuda")
    mask[2, 5] = False
    assert torch.isnan(bad["log_prob"][2, 5]) and torch.isnan(bad["logits"][2, 5]).all() and torch.equal(bad["top"], good["top"]) and torch.equal(bad["entropy"], good["entropy"])
    assert torch.equal(bad["log_prob"][mask], good["log_prob"][mask]) and torch.equal(bad["logits"][mask], good["logits"][mask])
    fbw.set_status_mode("sync")
    with pytest.raises(RuntimeError, match="target_log_probs: sequence 2: target out of range"):
        run(logits, bad_targets, lens, k, grads)
    fbw.set_status_mode("deferred")


def test_captured_calls_and_another_stream():
    from i6_native_ops_amd.training import target_log_probs
    logits, targets, lens, k, grads = problem(2, 30, 5001, 6, torch.float32, lens=[30, 12])
    leaf = logits.detach().clone().requires_grad_()

    def step():
        got = target_log_probs(leaf, targets, lens, alternatives=k)
        return got + torch.autograd.grad(got[:3], leaf, grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = step()
    side.synchronize()
    want = run(logits, targets, lens, k, grads)
    for n, x in zip(want, aside):
        assert torch.equal(x, want[n]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        new = problem(2, 30, 5001, 6, torch.float32, seed=50 + seed, lens=[30, 12])[0]
        with torch.no_grad():
            leaf.copy_(new)
        want = run(new, targets, lens, k, grads)
        graph.replay()
        torch.cuda.synchronize()
        for n, x in zip(want, out):
            assert torch.equal(x, want[n]), (seed, n)


def test_of_the_losses_of_the_output_layer():
    """Beside linear_cross_entropy: the same losses from the logits of the same layer."""
    from i6_native_ops_amd.training import linear_cross_entropy, target_log_probs
    g = gen(4)
    hidden, weight = torch.randn((3, 50, 64), generator=g, device="cuda"), torch.randn((300, 64), generator=g, device="cuda") / 8
    targets = torch.randint(0, 300, (3, 50), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.tensor([50, 0, 31], dtype=torch.int32, device="cuda")
    loss = linear_cross_entropy(hidden, weight, targets, lens)
    log_prob = target_log_probs(hidden @ weight.T, targets, lens)[0]
    # two sums of 64 products of size 1 / 8 each, two logarithms of 300 classes
    assert float((loss + log_prob).abs().max()) < 64 * 64 * 2.0 ** -22 / 8 + 2.0 ** -18


def test_second_derivatives_tangents_and_refusals():
    from i6_native_ops_amd.training import target_log_probs
    logits, targets, lens, k, _ = problem(2, 5, 7, 2, torch.float32)
    leaf = logits.detach().requires_grad_()
    grad, = torch.autograd.grad(target_log_probs(leaf, targets, lens)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="target_log_probs can be differentiated once"):
        grad.square().sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        target_log_probs(fwd.make_dual(logits, torch.ones_like(logits)), targets, lens)
    for args, match in [
        ((logits.cpu(), targets, lens), "logits must be a CUDA tensor"),
        ((logits.half(), targets, lens), "Expected logits"),
        ((logits, targets.long(), lens), "Expected targets"),
        ((logits, targets[:, :4], lens), "targets must have shape"),
        ((logits, targets, lens.long()), "Expected seq_lens"),
        ((logits, targets, lens[:1]), "seq_lens must have shape"),
        ((logits, targets, lens, 8), "alternatives must be"),
        ((logits, targets, lens, -1), "alternatives must be"),
        ((torch.zeros((1, 1, 100), device="cuda"), targets[:1, :1], lens[:1], 65), "alternatives must be"),
        ((logits[0], targets, lens), "logits must have shape"),
        ((logits[:, :0], targets[:, :0], lens), "T > 0"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            target_log_probs(*args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [20, 700, 5000, 30001])
def test_large_incoming_gradients_leave_ruled_out_classes_alone(F, dtype):
    """-inf and scores far below the others have no share, whatever comes in: their gradients are 0 and not a product of 0 and infinity."""
    logits, targets, lens, k, grads = problem(1, 4, F, 2, dtype, lens=[4])
    logits[0, 0, ::3] = -INF
    logits[0, 1, ::3] = torch.finfo(dtype).min
    logits[0, 2, ::3] = -1e30
    targets[:] = 1
    grads = [g * 1e12 for g in grads]
    got = run(logits, targets, lens, k, grads)
    assert torch.isfinite(got["logits"]).all()
    for t in range(3):
        ruled_out = torch.zeros(F, dtype=torch.bool, device="cuda")
        ruled_out[::3] = True
        ruled_out[got["classes"][0, t].long()] = False
        assert (got["logits"][0, t, ruled_out] == 0).all()
    check(got, expected(logits, targets, lens, k, grads))


@pytest.mark.parametrize("F,k", [(100, 0), (1003, 1), (9001, 3)])
def test_confident_frames_keep_their_small_gradients(F, k):
    """1 - p is the others' sum, not the difference of two numbers next to 1.  An exponential's argument, at most 90 / ln 2, is rounded to 2^-24 of it: 130 * 0.7 EPS32 of the exponential;
    sums of them take (64 + 2 * 10) EPS32 more, log1p, expm1 and the products 20."""
    from i6_native_ops_amd.training import target_log_probs
    sizes = [10.0, 25.0, 45.0, 80.0]
    logits = torch.zeros((1, 4, F), device="cuda")
    logits[0, :, F - 3] = torch.tensor(sizes, device="cuda")
    logits.requires_grad_()
    targets, lens = torch.full((1, 4), F - 3, dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    log_prob, _, top, classes = target_log_probs(logits, targets, lens, alternatives=k)
    loss = log_prob.sum() + (0.5 * top[:, :, 0].sum() if k else 0.0)      # the best alternative is the target
    grad, = torch.autograd.grad(loss, logits)
    if k:
        assert (classes[0, :, 0] == F - 3).all()
    for t, x in enumerate(sizes):
        others = (F - 1) * math.exp(-x)
        want = (1.5 if k else 1.0) * others / (1.0 + others)
        assert abs(float(grad[0, t, F - 3]) - want) <= want * 200 * EPS32, (x, float(grad[0, t, F - 3]), want)
