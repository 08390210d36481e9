"""What the operators around the losses owe to torch's bookkeeping."""
import pytest
import torch

from tests.test_training_gpu import DTYPES, ce_problem, rec_problem

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


@pytest.mark.parametrize("bits", [8, 32])
def test_optimiser_steps_are_seen_by_autograd(bits):
    """A second backward pass over a graph whose weights a step has changed raises, as after torch's own optimisers."""
    from i6_native_ops_amd.training import AdamW, linear_cross_entropy
    for sizes in [(2, 5, 7, 8), (2, 300, 400, 64)]:
        hidden, weight, bias, targets, lens, _ = ce_problem(*sizes, torch.float32)
        hidden.requires_grad_()
        weight = torch.nn.Parameter(weight)
        opt = AdamW([weight], lr=1e-2, state_bits=bits)
        loss = linear_cross_entropy(hidden, weight, targets, lens, bias=bias).sum()
        loss.backward(retain_graph=True)
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_steps_count_as_changes_of_all_they_write():
    from i6_native_ops_amd.training import adamw_step
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    m, v = (torch.zeros(300, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    scales = (torch.ones(2, device="cuda"), torch.ones(2, device="cuda"))
    before = [x._version for x in (p, m, v, *scales)]
    adamw_step([p], [g], [m], [v], step=1, lr=1e-2, scales=[scales])
    assert all(x._version > b for x, b in zip((p, m, v, *scales), before)) and g._version == 0
    with torch.inference_mode():                         # tensors without a version
        p, m, v = (torch.ones(300, device="cuda") for _ in range(3))
        adamw_step([p], [p.clone()], [m], [v], step=1, lr=1e-2)
    adamw_step([p], [p.clone()], [m], [v], step=2, lr=1e-2)
    assert torch.isfinite(p).all()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tangents_are_refused(which):
    import torch.autograd.forward_ad as fwad
    from i6_native_ops_amd.training import gated_recurrence, linear_cross_entropy
    hidden, weight, bias, targets, lens, _ = ce_problem(2, 5, 7, 8, torch.float32)
    x, gate, rec_lens, state, _ = rec_problem(2, 5, 8, torch.float32)
    with fwad.dual_level():
        args = [hidden, weight, bias]
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="linear_cross_entropy has no forward-mode derivative"):
            linear_cross_entropy(args[0], args[1], targets, lens, bias=args[2])
        args = [x, gate, state]
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="gated_recurrence has no forward-mode derivative"):
            gated_recurrence(args[0], args[1], rec_lens, initial_state=args[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_single_channels_of_any_stride(dtype):
    """Where the last dimension has one value its stride says nothing, and torch leaves it as it is."""
    from i6_native_ops_amd.training import gated_recurrence, linear_cross_entropy
    x, gate, lens, state, _ = rec_problem(2, 30, 1, dtype)
    want, last = gated_recurrence(x, gate, lens, initial_state=state)
    odd = [torch.as_strided(v, v.shape, (30, 1, 30)) for v in (x, gate)]
    leaf = odd[0].detach().requires_grad_()
    h, again = gated_recurrence(leaf, odd[1], lens, initial_state=state)
    assert torch.equal(h, want) and torch.equal(again, last)
    h.sum().backward()
    assert leaf.grad.shape == x.shape
    one = torch.ones((1, 1, 1), dtype=dtype, device="cuda").requires_grad_()
    h, _ = gated_recurrence(one, one.detach())
    h.sum().backward()                                   # an incoming gradient whose strides are all 0
    assert abs(float(one.grad) - float(torch.sigmoid(torch.tensor(-1.0)))) < 2.0 ** -8
    hidden, weight, bias, targets, lens, _ = ce_problem(2, 300, 40, 1, dtype)
    want = linear_cross_entropy(hidden, weight, targets, lens, bias=bias)
    got = linear_cross_entropy(torch.as_strided(hidden, hidden.shape, (300, 1, 300)), torch.as_strided(weight, weight.shape, (1, 40)), targets, lens, bias=bias)
    assert torch.equal(want, got)
