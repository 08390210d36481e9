"""Cross entropy of frames, classes and incoming gradients of very different sizes."""
import math

import pytest
import torch

from tests.test_training_gpu import DTYPES, ce_expected, ce_problem, ce_run, close

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
@pytest.mark.parametrize("sizes", SIZES)
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
