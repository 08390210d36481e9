"""The second set of training operators at the largest sizes: tensors of more than 2^31 values, matrices of 32 768 rows and columns."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8


def normal(*shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=torch.bfloat16)


def test_delta_rule_with_more_than_2_31_values():
    """The last frames of a long call, outputs and gradients, are those of a call that begins with their state.  Both are a rounding of 2^-8 off what is right, and so 2 * 2^-8 off each
    other; states are right to the 128 + 128 + 4 * 32 + 1000 terms (they last for a thousand frames at most) that the other tests derive, four times for what cancels, twice."""
    from i6_native_ops_amd.training import gated_delta_rule
    T, H, D, tail = 263000, 64, 128, 700
    assert T * H * D > 2 ** 31
    x = {n: normal(1, T, H, D, seed=i) for i, n in enumerate(("q", "k", "v"))}
    x["gate"], x["beta"] = normal(1, T, H, seed=4) + 3, normal(1, T, H, seed=5)
    x = {n: t.requires_grad_() for n, t in x.items()}
    o, last = gated_delta_rule(*x.values())
    grad_o = normal(1, T, H, D, seed=6)
    grads = torch.autograd.grad([o], list(x.values()), [grad_o])
    got = [o[:, -tail:].detach().clone(), *(g[:, -tail:].clone() for g in grads)]
    with torch.no_grad():
        _, state = gated_delta_rule(*(t[:, :T - tail] for t in x.values()))
    del o, grads
    y = [t[:, T - tail:].detach().requires_grad_() for t in x.values()]
    o, end = gated_delta_rule(*y, initial_state=state)
    want = [o.detach(), *torch.autograd.grad([o], y, [grad_o[:, -tail:]])]
    bound = 2 * 16 * (128 + 128 + 4 * 32 + 1000) * EPS32
    for n, g, w in zip(("o", *x), got, want):
        assert float((g.double() - w.double()).norm()) <= (2 * EPS16 + bound) * float(w.double().norm()), n
    assert float((end.double() - last.double()).norm()) <= bound * float(end.double().norm())


def test_log_probs_with_more_than_2_31_values():
    """The last frames of a call are those of a call on them alone.  Sums have F terms, 2^-24 each of a sum that is 1 at least; gradients are rounded once more."""
    from i6_native_ops_amd.training import target_log_probs
    B, T, F, tail = 8, 22500, 12001, 40
    assert B * T * F > 2 ** 31
    z = normal(B, T, F, seed=1).requires_grad_()
    y = torch.randint(0, F, (B, T), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda", dtype=torch.int32)
    lens = torch.full((B,), T, dtype=torch.int32, device="cuda")
    out = target_log_probs(z, y, lens, alternatives=3)
    loss_grads = [torch.ones_like(out[0]), torch.full_like(out[1], 0.5)]
    grad, = torch.autograd.grad(out[:2], z, loss_grads)
    part = z[-1:, -tail:].detach().clone().requires_grad_()
    want = target_log_probs(part, y[-1:, -tail:].contiguous(), torch.full((1,), tail, dtype=torch.int32, device="cuda"), alternatives=3)
    want_grad, = torch.autograd.grad(want[:2], part, [g[-1:, -tail:].contiguous() for g in loss_grads])
    bound = 2 * F * EPS32
    for g, w in zip(out[:3], want[:3]):
        assert float((g[-1:, -tail:] - w).abs().max()) <= bound * 12         # log p and entropies are 12 at most
    assert torch.equal(out[3][-1:, -tail:], want[3])
    d = (grad[-1:, -tail:].double() - want_grad.double()).abs()
    assert (d <= (2 * EPS16 + 24 * bound) * want_grad.double().abs() + 2.0 ** -133).all()


def test_the_largest_matrix():
    """One iteration on 32 768 x 32 768; columns of the result by products with vectors in 64 bits.  Two products of 11-bit halves and one of rounded operands, as in the other tests."""
    from i6_native_ops_amd.training import orthogonalize
    n = 32768
    u = normal(n, n, seed=3)
    got, = orthogonalize([u], steps=1)
    columns = torch.tensor([0, 1, 777, 16384, 32767], device="cuda")
    x = u.double()
    x /= x.norm()
    e = torch.zeros((n, len(columns)), dtype=torch.float64, device="cuda")
    e[columns, torch.arange(len(columns))] = 1.0
    y = x @ e
    ay = x @ (x.T @ y)
    want = 3.4445 * y - 4.7750 * ay + 2.0315 * (x @ (x.T @ ay))
    d = got[:, columns].double() - want
    assert float(d.norm()) <= (7 * 2 * (2.0 ** -23 + EPS32 * n ** 0.5) + EPS16 + 3.45 * 2 * 2.0 ** -11) * float(want.norm())
