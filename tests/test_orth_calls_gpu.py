"""Muon and orthogonalised updates as calls go: matrices without values, many at once, captured."""
import pytest
import torch

from tests.test_orth_gpu import DTYPES, check, expected, matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [0, 1, 2])
def test_matrices_without_values_among_others(at, dtype):
    """As if they were not there, first, in the middle or last; a call that is refused raises no version."""
    from i6_native_ops_amd.training import Muon, muon_step
    shapes = [(64, 40), (30, 90)]
    shapes.insert(at, (0, 8))
    params = [matrix(r, c, dtype, seed=i, size=0.05) if r else torch.zeros((r, c), dtype=dtype, device="cuda") for i, (r, c) in enumerate(shapes)]
    grads = [matrix(r, c, dtype, seed=10 + i) if r else torch.zeros_like(p) for i, ((r, c), p) in enumerate(zip(shapes, params))]
    others = [i for i in range(3) if i != at]
    alone = [p.clone() for p in params]
    moved = [torch.zeros(s, device="cuda") for s in shapes]
    muon_step([alone[i] for i in others], [grads[i] for i in others], [moved[i] for i in others], lr=0.02)
    momenta = [torch.zeros(s, device="cuda") for s in shapes]
    muon_step(params, grads, momenta, lr=0.02)
    for p, q, m, n in zip(params, alone, momenta, moved):
        assert torch.equal(p, q) and torch.equal(m, n)
    weights = [torch.nn.Parameter(p.clone()) for p in params]
    for w, g in zip(weights, grads):
        w.grad = g
    Muon(weights, lr=0.02).step()
    versions = [p._version for p in params]
    with pytest.raises(RuntimeError, match="momentum must be"):
        muon_step(params, grads, momenta, lr=0.02, momentum=1.0)
    with pytest.raises(RuntimeError, match="steps must be"):
        muon_step(params, grads, momenta, lr=0.02, steps=-1)
    assert versions == [p._version for p in params]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,rows,cols", [(36, 130, 300), (70, 140, 136), (34, 200, 129), (35, 129, 200), (5, 257, 513), (3, 513, 511)])
def test_every_matrix_of_calls_that_take_several_launches(count, rows, cols, dtype):
    """Matrices of one launch follow those of another in the same memory.  All of them, and again."""
    from i6_native_ops_amd.training import orthogonalize
    updates = [matrix(rows + i % 3, cols, dtype, seed=i) for i in range(count)]
    got, again = orthogonalize(updates), orthogonalize(updates)
    for u, x, y in zip(updates, got, again):
        assert torch.equal(x, y)
        check(x, expected(u), max(u.shape))


@pytest.mark.parametrize("steps", [0, 1, 5])
def test_many_small_matrices_with_and_without_iterations(steps):
    from i6_native_ops_amd.training import orthogonalize
    sizes = [(20 + i % 9, 30 + i % 7) for i in range(80)] + [(150, 170), (0, 3)]
    updates = [matrix(r, c, torch.float32, seed=i) if r else torch.zeros((r, c), device="cuda") for i, (r, c) in enumerate(sizes)]
    for u, x in zip(updates, orthogonalize(updates, steps=steps)):
        assert x.shape == u.shape
        if u.numel():
            check(x, expected(u, steps), max(u.shape))


def test_a_captured_optimiser_goes_on_with_its_averages():
    """The step that makes them is refused under capture (each replay would begin them anew); behind it replays are the steps that eager calls are."""
    from i6_native_ops_amd.training import Muon
    weights = [torch.nn.Parameter(matrix(60, 40, torch.float32, seed=1, size=0.05)) for _ in range(2)]
    for w in weights:
        w.grad = matrix(60, 40, torch.float32, seed=2)
    captured, eager = Muon(weights[:1], lr=0.02), Muon(weights[1:], lr=0.02)
    graph = torch.cuda.CUDAGraph()
    before = weights[0].detach().clone()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(graph):
            captured.step()
    assert torch.equal(weights[0], before)
    captured.step(), eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for step in range(3):
        for w in weights:
            w.grad.copy_(matrix(60, 40, torch.float32, seed=3 + step))
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(weights[0], weights[1]) and torch.equal(captured.state[weights[0]]["momentum"], eager.state[weights[1]]["momentum"]), step
