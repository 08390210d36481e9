"""Cross entropy of frames, classes and incoming gradients of very different sizes: a large one changes nothing but what
it enters.  Bounds are those of tests/test_training_gpu.py, computed without the large one."""
import math

import pytest
import torch

from tests.test_training_gpu import DTYPES, EPS16, EPS32, EPS_HALVES, ce_check, ce_expected, ce_problem, ce_run, close, gen

pytestmark = pytest.mark.gpu

SIZES = [(2, 300, 400, 256), (5, 211, 1201, 72)]        # beyond the layers whose kernels work in 32 bits throughout


def without(targets, *places):
    targets = targets.clone()
    for at in places:
        targets[at] = -1
    return targets


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(2, 50, 10, 64), (2, 300, 400, 256)])
def test_confident_frames_have_no_negative_loss(sizes, dtype):
    """Features that are a multiple of their class's row, logits in the hundreds: the target is the largest logit, and the loss
    a logarithm of 1 or more."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=9, lens=[sizes[1]] * sizes[0])
    weight = weight * math.sqrt(sizes[3])
    hidden = (weight[targets.long()].float() * 3.7).to(dtype)
    from i6_native_ops_amd.training import linear_cross_entropy
    loss = linear_cross_entropy(hidden, weight, targets, lens, bias=bias)
    assert (loss >= -2.0 ** -20).all(), float(loss.min())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e12, 1e25])
@pytest.mark.parametrize("sizes", SIZES)
def test_gradients_of_a_large_frame_are_finite(sizes, size, dtype):
    """Its logits are as large; the sum over the classes and the target's logit have to agree on every bit of them."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=2, lens=[sizes[1]] * sizes[0])
    hidden[1, 7] *= size
    hidden[0, ::5] *= 1e7
    for target in range(5):
        targets[1, 7] = target
        got = ce_run(hidden, weight, bias, targets, lens, grad)
        assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(2, 50, 10, 64)] + SIZES)
def test_target_with_the_lowest_bias(sizes, dtype):
    """A class with the type's lowest value as bias costs, as a target, what the bias says; elsewhere it is not there."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=10, lens=[sizes[1]] * sizes[0])
    lowest = torch.finfo(dtype).min
    bias[3] = lowest
    targets[0, 5] = 3
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    assert all(torch.isfinite(x).all() for x in got.values())
    assert abs(float(got["loss"][0, 5]) / -lowest - 1) < 1e-5
    others, keep = targets != 3, torch.arange(sizes[2], device="cuda") != 3
    renumbered = torch.where(targets > 3, targets - 1, torch.where(others, targets, -1))
    want = ce_expected(hidden, weight[keep].contiguous(), bias[keep].contiguous(), renumbered, lens, grad)
    for k in ("loss", "hidden"):
        close(got[k][others], want[k][0][others], want[k][1][others], k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_layers_whose_classes_all_have_the_lowest_bias(dtype):
    """Sums of the lowest value and a logit round to the lowest value: the classes are equal."""
    hidden, weight, _, targets, lens, grad = ce_problem(2, 50, 10, 64, dtype, seed=10, lens=[50, 50])
    got = ce_run(hidden, weight, torch.full((10,), torch.finfo(dtype).min, dtype=dtype, device="cuda"), targets, lens, grad)
    assert (got["loss"] - math.log(10)).abs().max() < 1e-5
    G = (torch.full((2, 50, 10), 0.1, dtype=torch.float64, device="cuda") - torch.nn.functional.one_hot(targets.long(), 10)) * grad.double()[:, :, None]
    close(got["hidden"], G @ weight.double(), (G.abs() @ weight.double().abs()) * (2.0 ** -20 + (EPS16 if dtype == torch.bfloat16 else 0)), "hidden")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e9, 1e12, 1e15, 1e25])
@pytest.mark.parametrize("elements", [1, 64])
@pytest.mark.parametrize("sizes", SIZES)
def test_loss_beside_a_large_frame(sizes, elements, size, dtype):
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=3, lens=[sizes[1]] * sizes[0])
    from i6_native_ops_amd.training import linear_cross_entropy
    ordinary = linear_cross_entropy(hidden, weight, targets, lens, bias=bias)
    hidden[1, 7, :elements] *= size
    loss = linear_cross_entropy(hidden, weight, targets, lens, bias=bias)
    want, bound = ce_expected(hidden, weight, bias, without(targets, (1, 7)), lens, grad)["loss"]
    others = torch.ones_like(targets, dtype=torch.bool)
    others[1, 7] = False
    close(loss[others], want[others], bound[others], "loss")
    if dtype == torch.bfloat16:
        assert torch.equal(loss[others], ordinary[others])
    # the frame itself: between 0 and what its logits can differ by
    z = hidden[1, 7].double() @ weight.double().T + bias.double()
    exact = torch.logsumexp(z, 0) - z[targets[1, 7].long()]
    reach = (hidden[1, 7].double().abs() @ weight.double().abs().T).max()
    assert loss[1, 7] >= -2.0 ** -20 and abs(float(loss[1, 7]) - float(exact)) <= 2 * float(reach) * (sizes[3] + 4) * EPS_HALVES + 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e9, 1e12, 1e15, 1e25])
@pytest.mark.parametrize("elements", [1, 64])
@pytest.mark.parametrize("sizes", SIZES)
def test_gradients_beside_a_large_frame(sizes, elements, size, dtype):
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=4, lens=[sizes[1]] * sizes[0])
    at = (1, 7)
    hidden[1, 7, :elements] *= size
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    assert all(torch.isfinite(x).all() for x in got.values())
    want = ce_expected(hidden, weight, bias, without(targets, at), lens, grad)
    others = torch.ones_like(targets, dtype=torch.bool)
    others[at] = False
    close(got["hidden"][others], want["hidden"][0][others], want["hidden"][1][others], "hidden")
    # classes that the large frame says nothing about: neither its target nor of any probability there
    z = hidden[at].double() @ weight.double().T + bias.double()
    free = z < z.max() - 1000 - (hidden[at].double().abs() @ weight.double().abs().T).max() * sizes[3] * EPS_HALVES
    free[targets[at].long()] = False
    assert free.sum() > sizes[2] // 2
    for k in ("weight", "bias"):
        close(got[k][free], want[k][0][free], want[k][1][free], k)
    # all of its gradient is in the two classes that it does say something about
    if float(z.max() - z[targets[at].long()]) > float(z.max() - z[free].max()) / 2:
        y = int(targets[at])
        share = -grad[at].double() * hidden[at].double()
        error = (got["weight"][y].double() - share - want["weight"][0][y]).abs()
        assert (error <= want["weight"][1][y] + share.abs() * 4 * (EPS16 if dtype == torch.bfloat16 else EPS_HALVES) + (EPS16 if dtype == torch.bfloat16 else 4 * EPS32) * share.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e9, 1e12, 1e25])
@pytest.mark.parametrize("sizes", SIZES)
def test_loss_and_gradients_beside_a_large_class(sizes, size, dtype):
    """A class whose weights are far larger than the others': frames that it is improbable for are as they would be without it."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=5, lens=[sizes[1]] * sizes[0])
    c = 130
    targets[targets == c] = 0
    weight[c] = (weight[c].float() * size).to(dtype)
    z = hidden.double() @ weight[c].double()
    margin = (hidden.double().abs() @ weight[c].double().abs()) * (sizes[3] + 4) * EPS_HALVES + 1000
    targets[z > -margin] = -1
    assert (targets >= 0).float().mean() > 0.3
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    keep = torch.arange(sizes[2], device="cuda") != c
    renumbered = torch.where(targets > c, targets - 1, targets)
    want = ce_expected(hidden, weight[keep].contiguous(), bias[keep].contiguous(), renumbered, lens, grad)
    close(got["loss"], *want["loss"], "loss")
    close(got["hidden"], *want["hidden"], "hidden")
    for k in ("weight", "bias"):
        close(got[k][keep], *want[k], k)
        assert (got[k][c] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_gradients_of_very_small_and_very_large_shares(sizes, dtype):
    """Incoming gradients over thirty powers of ten: every frame's gradient is as precise as it would be alone."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=6)
    share = torch.exp((torch.rand(targets.shape, generator=gen(7), device="cuda") - 0.5) * 30 * math.log(10.0))
    got = ce_run(hidden, weight, bias, targets, lens, share * grad.sign())
    alone, bound = ce_expected(hidden, weight, bias, targets, lens, grad.sign())["hidden"]
    by = share.double()[:, :, None]
    close(got["hidden"], alone * by, bound * by, "hidden")
    want = ce_expected(hidden, weight, bias, targets, lens, share * grad.sign())
    for k in ("weight", "bias"):
        close(got[k], *want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_frames_of_many_sizes(dtype):
    """Frames over twenty powers of ten."""
    hidden, weight, bias, targets, lens, grad = ce_problem(3, 250, 300, 128, dtype, seed=8, lens=[250, 250, 99])
    size = torch.exp(-torch.rand((3, 250, 1), generator=gen(9), device="cuda") * 20 * math.log(10.0))
    hidden = (hidden.float() * size).to(dtype)
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    want = ce_expected(hidden, weight, bias, targets, lens, grad)
    for k in got:
        close(got[k], *want[k], k)


@pytest.mark.parametrize("B,T,F,D,dtype", [
    (3, 400, 7700, 450, torch.float32), (3, 400, 7700, 450, torch.bfloat16), (9, 1000, 15001, 40, torch.float32), (33, 1000, 9001, 24, torch.bfloat16),
    (1, 700, 4099, 31, torch.float32), (20, 300, 130, 500, torch.float32), (8, 2000, 3001, 260, torch.float32),
])
def test_frames_and_shares_of_many_sizes_in_large_layers(B, T, F, D, dtype):
    """Large and small tiles, several pieces of the vocabulary, ranges of frames and of classes."""
    hidden, weight, bias, targets, lens, grad = ce_problem(B, T, F, D, dtype, seed=F, lens=[T] * (B - 1) + [T - 5])
    targets[0, 3:9] = -1
    hidden[0, 3:9] = float("nan")
    size = torch.exp(-torch.rand((B, T, 1), generator=gen(9), device="cuda") * 12 * math.log(10.0))
    clean = torch.nan_to_num(hidden.float() * size).to(dtype)
    got = ce_run((hidden.float() * size).to(dtype), weight, bias, targets, lens, grad * size[:, :, 0].flip(1))
    want = ce_expected(clean, weight, bias, targets, lens, grad * size[:, :, 0].flip(1))
    for k in got:
        close(got[k], *want[k], k)
    again = ce_run((hidden.float() * size).to(dtype), weight, bias, targets, lens, grad * size[:, :, 0].flip(1))
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e6, 1e12, 1e20])
@pytest.mark.parametrize("of", ["hidden", "weight"])
@pytest.mark.parametrize("sizes", SIZES + [(3, 300, 100, 9)])
def test_a_large_feature(sizes, of, size, dtype):
    """One feature of all frames, or of all classes, far larger than the others, where the other operand has zeros: nothing of it is in the logits."""
    hidden, weight, bias, targets, lens, grad = ce_problem(*sizes, dtype, seed=12, lens=[sizes[1]] * sizes[0])
    large, zero = (hidden, weight) if of == "hidden" else (weight, hidden)
    large[..., 5] *= size
    zero[..., 5] = 0
    ce_check((hidden, weight, bias, targets, lens, grad))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e4, 1e6, 1e12])
def test_a_large_frame_in_a_large_layer(size, dtype):
    """The statistics have other tiles here than the gradient of the logits, whose exponentials have to fit them bit for bit."""
    hidden, weight, bias, targets, lens, grad = ce_problem(3, 400, 7700, 450, dtype, seed=13, lens=[400, 400, 390])
    hidden[1, 5:80:7] *= size
    got = ce_run(hidden, weight, bias, targets, lens, grad)
    assert all(torch.isfinite(x).all() for x in got.values()) and (got["loss"] >= -2.0 ** -20).all()
    others = torch.ones_like(targets, dtype=torch.bool)
    others[1, 5:80:7] = False
    want = ce_expected(hidden, weight, bias, torch.where(others, targets, -1), lens, grad)
    for k in ("loss", "hidden"):
        close(got[k][others], want[k][0][others], want[k][1][others], k)
    # a large frame's probabilities are 0 and 1: its gradient is the difference of two rows of the weights, or nothing
    z = hidden[1, 5:80:7].double() @ weight.double().T + bias.double()
    two = z.topk(2).values
    sure = two[:, 0] - two[:, 1] > (hidden[1, 5:80:7].double().abs() @ weight.double().abs().T).amax(1) * 460 * EPS_HALVES + 100
    rows = weight.double()[z.argmax(1)] - weight.double()[targets[1, 5:80:7].long()]
    exact = rows * grad[1, 5:80:7].double()[:, None]
    error = (got["hidden"][1, 5:80:7].double() - exact).abs()
    allowed = (rows.abs() + 2 * weight.double().abs().max()) * grad[1, 5:80:7].double().abs()[:, None] * (4 * EPS16 if dtype == torch.bfloat16 else 8 * EPS_HALVES) + 1e-30
    assert (error <= allowed)[sure].all()
    assert sure.any() or size < 1e5
