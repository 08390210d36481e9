"""The gated delta rule with values of very different sizes, and with values that are no numbers."""
import pytest
import torch

from tests.test_delta_gpu import DTYPES, NAMES, check, expected, problem, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V,at", [(70, 16, 16, (0, 21)), (70, 64, 40, (15, 16, 31, 63, 64)), (130, 128, 128, (33, 127)), (1300, 64, 64, (700,))])
def test_what_is_no_number_stays_out_of_the_frames_in_front_of_it(T, K, V, at, dtype):
    """A value that is NaN or infinite spoils its column from its frame on, a key or share all columns: never a frame in front of it, another column or another sequence."""
    from i6_native_ops_amd.training import gated_delta_rule

    def outputs(p):
        with torch.no_grad():
            plain = gated_delta_rule(*(p[n] for n in NAMES[:5]), initial_state=p["initial"])
        trained = gated_delta_rule(*(p[n].requires_grad_(n == "v") for n in NAMES[:5]), initial_state=p["initial"])
        assert all(torch.equal(a.nan_to_num(7.0), b.detach().nan_to_num(7.0)) for a, b in zip(plain, trained))
        return plain

    p = problem(2, T, 2, 2, K, V, dtype, lens="all")
    want = outputs({n: x.clone() if torch.is_tensor(x) else x for n, x in p.items()})
    for t in at:
        for name, bad in (("v", float("nan")), ("v", float("inf")), ("k", float("nan")), ("beta", float("nan"))):
            q = {n: x.clone() if torch.is_tensor(x) else x for n, x in p.items()}
            q[name][(0, t, 1, 3) if name == "v" else (0, t, 1)] = bad
            o, last = outputs(q)
            columns = [3] if name == "v" else list(range(V))
            spoilt = torch.zeros(o.shape, dtype=torch.bool, device="cuda")
            spoilt[0, t:, 1, columns] = True
            assert not torch.isfinite(o[spoilt]).any(), (name, t)
            assert torch.equal(o[~spoilt], want[0][~spoilt]), (name, t)
            of_state = torch.zeros(last.shape, dtype=torch.bool, device="cuda")
            of_state[0, 1, :, columns] = True
            assert not torch.isfinite(last[of_state]).any() and torch.equal(last[~of_state], want[1][~of_state]), (name, t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V,t", [(10, 16, 16, 4), (40, 16, 16, 5), (70, 64, 40, 63), (130, 128, 128, 64), (1300, 64, 64, 700)])
def test_a_gate_that_is_no_number(T, K, V, t, dtype):
    """It is none of the gates that forget: all of the head is spoilt from its frame on, and not replaced by what looks like results.  In chunks as frame by frame."""
    from i6_native_ops_amd.training import gated_delta_rule
    p = problem(2, T, 2, 2, K, V, dtype, lens="all")
    with torch.no_grad():
        want = gated_delta_rule(*(p[n] for n in NAMES[:5]), initial_state=p["initial"])
        p["gate"][1, t, 0] = float("nan")
        o, last = gated_delta_rule(*(p[n] for n in NAMES[:5]), initial_state=p["initial"])
    trained = gated_delta_rule(*(p[n].requires_grad_(n == "v") for n in NAMES[:5]), initial_state=p["initial"])[0].detach()
    assert torch.isnan(o[1, t:, 0]).all() and torch.isnan(trained[1, t:, 0]).all() and torch.isnan(last[1, 0]).all()
    o[1, t:, 0] = want[0][1, t:, 0]
    last[1, 0] = want[1][1, 0]
    assert torch.equal(o, want[0]) and torch.equal(last, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V", [(40, 16, 16), (64, 64, 40), (130, 128, 128), (150, 32, 100)])
def test_gates_of_frames_in_front_of_a_far_larger_one(T, K, V, dtype):
    """Their gradients are sums of what decays over them, none of which a later frame's value enters: as right as without it.  (The incoming gradients do not depend on it.)"""
    p = problem(2, T, 2, 1, K, V, dtype, lens="all")
    t = T - 11
    p["v"][:, t] *= 2.0 ** 20
    want, got = expected(p), run(p)
    n = slice(0, t + 1)
    check(p, {"gate": got["gate"][:, n]}, {"gate": want["gate"][:, n]})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [-3.0, -10.0, -20.0, -60.0])
@pytest.mark.parametrize("K,V", [(16, 16), (128, 128)])
def test_gates_that_leave_little(gate, K, V, dtype):
    """The gradients of gates are in proportion to what is left, e^gate of the other sums, and right in that proportion."""
    p = problem(2, 100, 2, 1, K, V, dtype, lens="all")
    p["gate"][:] = gate
    p["gate"][:, ::7] += 2.0
    check(p, run(p), expected(p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V", [(40, 16, 16), (100, 64, 64), (130, 128, 128), (70, 32, 100), (1300, 64, 40)])
def test_columns_of_very_different_sizes(T, K, V, dtype):
    """Values times powers of two, incoming gradients divided by them: every product of the one with the other is what it was, and so is every result, to the last bit."""
    p = problem(2, T, 2, 1, K, V, dtype, lens="all")
    plain = run(p)
    if T < 1000:
        check(p, plain, expected(p))
    sizes = torch.tensor([2.0 ** i for i in torch.randint(-20, 41, (V,), generator=torch.Generator().manual_seed(5)).tolist()], device="cuda")    # (the card's powers are not exact)
    moved = dict(p, v=(p["v"].float() * sizes).to(dtype), initial=p["initial"] * sizes, grad_o=(p["grad_o"].float() / sizes).to(dtype), grad_last=p["grad_last"] / sizes)
    got = run(moved)
    for n in ("q", "k", "gate", "beta"):
        assert torch.equal(got[n], plain[n]), n
    for n, by in (("o", 1 / sizes), ("last", 1 / sizes), ("v", sizes), ("initial", sizes)):
        assert torch.equal((got[n].float() * by).to(got[n].dtype), plain[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,V", [(40, 16, 16), (100, 64, 64), (130, 128, 128), (70, 32, 100)])
def test_frames_of_very_different_sizes(T, K, V, dtype):
    """What a far larger value or incoming gradient does not enter is as right as without it: results of frames in front of the value, gradients of frames behind the incoming one."""
    t = T - 21
    p = problem(2, T, 2, 1, K, V, dtype, lens="all")
    p["v"][:, t] *= 2.0 ** 40
    want, got = expected(p), run(p)
    for n in ("o", "q", "k", "beta", "gate"):
        check(p, {n: got[n][:, :t]}, {n: want[n][:, :t]})
    check(p, {"v": got["v"]}, {"v": want["v"]})
    p = problem(2, T, 2, 1, K, V, dtype, lens="all")
    p["grad_o"][:, t] *= 2.0 ** 40
    want, got = expected(p), run(p)
    for n in ("q", "k", "v", "beta", "gate"):
        check(p, {n: got[n][:, t + 1:]}, {n: want[n][:, t + 1:]})
