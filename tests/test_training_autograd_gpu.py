"""What the operators around the losses owe to torch's bookkeeping."""
import pytest
import torch

from tests.test_training_gpu import ce_problem, rec_problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["hidden", "weight", "bias"])
@pytest.mark.parametrize("sizes", [(2, 5, 7, 8), (2, 300, 400, 64)])
def test_gradient_penalty_of_the_cross_entropy_is_refused(sizes, which):
    """An incoming gradient that is constant: the gradient depends on the inputs all the same."""
    from i6_native_ops_amd.training import linear_cross_entropy
    hidden, weight, bias, targets, lens, _ = ce_problem(*sizes, torch.float32)
    args = dict(hidden=hidden, weight=weight, bias=bias)
    leaf = args[which].requires_grad_()
    loss = linear_cross_entropy(args["hidden"], args["weight"], targets, lens, bias=args["bias"]).sum()
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="linear_cross_entropy can be differentiated once"):
        (loss + grad.square().sum()).backward()


@pytest.mark.parametrize("which", ["x", "gate", "initial"])
def test_gradient_penalty_of_the_recurrence_is_refused(which):
    from i6_native_ops_amd.training import gated_recurrence
    x, gate, lens, state, _ = rec_problem(2, 40, 64, torch.float32)
    args = dict(x=x, gate=gate, initial=state)
    leaf = args[which].requires_grad_()
    h, _ = gated_recurrence(args["x"], args["gate"], lens, initial_state=args["initial"])
    grad, = torch.autograd.grad(h.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="gated_recurrence can be differentiated once"):
        grad.square().sum().backward()


def test_a_graph_of_the_gradients_that_is_not_used():
    """create_graph alone is no second derivative: the first one is what it is without."""
    from i6_native_ops_amd.training import linear_cross_entropy
    hidden, weight, bias, targets, lens, _ = ce_problem(2, 50, 70, 64, torch.float32)
    leaves = [v.requires_grad_() for v in (hidden, weight, bias)]
    loss = linear_cross_entropy(hidden, weight, targets, lens, bias=bias)
    plain = torch.autograd.grad(loss.sum(), leaves, retain_graph=True)
    again = torch.autograd.grad(loss.sum(), leaves, create_graph=True)
    for a, b in zip(plain, again):
        assert torch.equal(a, b.detach())
