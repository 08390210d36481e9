"""Orthogonalised updates and Muon against 64 bits.

Tolerances.  Operands are held to 2^-23 of each value, products add up n terms of both signs (2^-24 sqrt(n) of the sum's size).  What an iteration adds in left
singular directions of small singular values grows 3.45 times in each of those that follow, 3.45^4 = 142 times in four; the errors of one iteration, 4.775 and 2.0315 times those of A and A A
with singular values of 1 at most, are 7 times those of a product.  So the 2-norm of the error is at most 7 * 142 * 2 * (2^-23 + 2^-24 sqrt(n)) of that of X of an
update whose singular values are all near the largest.  For 16-bit results the last product has operands of 11 bits: each is off by 2^-11 of its size at most, the
first one's singular values are 3.45 at most, and so the 2-norm is off by 3.45 * 2 * 2^-11 more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8
DTYPES = [torch.float32, torch.bfloat16]
A, B, C = 3.4445, -4.7750, 2.0315


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(rows, cols, dtype, seed=1, size=1e-3):
    return (torch.randn((rows, cols), generator=gen(seed), device="cuda") * size).to(dtype)


def expected(u, steps=5):
    x = u.double().cpu()
    turned = x.shape[0] > x.shape[1]
    x = x.T if turned else x
    x = x / x.norm().clamp(min=1e-7)
    for _ in range(steps):
        g = x @ x.T
        x = A * x + (B * g + C * g @ g) @ x
    return (x.T if turned else x).cuda()


def check(got, want, terms):
    out = EPS16 if got.dtype == torch.bfloat16 else 0.0
    bound = 7 * 142 * 2 * (2.0 ** -23 + EPS32 * terms ** 0.5) + out + (3.45 * 2 * 2.0 ** -11 if out else 0.0)
    d = got.double() - want
    least = 485 * 2.0 ** -39                 # an update whose norm is below 1e-7 is not scaled up to 1, and what X holds ends at 2^-39
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert float(d.norm()) <= bound * float(want.norm()) + least * want.numel() ** 0.5, (float(d.norm() / want.norm()), bound)
    rms = float(want.square().mean().sqrt())
    assert (d.abs() <= 8 * bound * rms + out * want.abs() + 8 * least).all(), (float(d.abs().max()), rms)


SIZES = [(1, 1), (1, 9), (7, 1), (5, 5), (32, 32), (33, 31), (64, 128), (128, 64), (65, 257), (130, 129), (128, 128), (300, 40), (17, 1000), (512, 300), (1000, 12)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_one_matrix(rows, cols, dtype):
    from i6_native_ops_amd.training import orthogonalize
    u = matrix(rows, cols, dtype, seed=rows + cols)
    kept = u.clone()
    got, = orthogonalize([u])
    check(got, expected(u), max(rows, cols))
    assert torch.equal(u, kept) and got.dtype == dtype


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_matrices_of_all_sizes(dtype):
    """More than one launch's table holds; each as if it were alone, and the same in every run."""
    from i6_native_ops_amd.training import orthogonalize
    g = torch.Generator().manual_seed(2)
    sizes = [tuple(torch.randint(1, 200, (2,), generator=g).tolist()) for _ in range(90)] + [(0, 5), (4, 0), (260, 140)]
    updates = [matrix(r, c, dtype, seed=i) for i, (r, c) in enumerate(sizes)]
    got, again = orthogonalize(updates), orthogonalize(updates)
    for u, x, y in zip(updates, got, again):
        assert torch.equal(x, y) and x.shape == u.shape
        if u.numel():
            check(x, expected(u), max(u.shape))
            assert torch.equal(x, orthogonalize([u])[0])
    assert orthogonalize([]) == []


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,cols", [(20, 1000, 1100), (16, 1024, 1300), (3, 2100, 1500), (5, 257, 513), (70, 130, 600), (1, 200, 4096), (2, 3000, 70), (1, 8, 30000), (1, 700, 520), (3, 513, 511)])
def test_many_large_matrices(n, rows, cols, dtype):
    """Large tiles, large ones and their quarters, quarters alone, small ones; more than a launch's table; few tiles, whose sums are formed in parts."""
    from i6_native_ops_amd.training import orthogonalize
    updates = [matrix(rows, cols, dtype, seed=i) for i in range(n)]
    got, again = orthogonalize(updates), orthogonalize(updates)
    for i, (u, x, y) in enumerate(zip(updates, got, again)):
        assert torch.equal(x, y)
        if i in (0, n // 2, n - 1):
            check(x, expected(u), max(rows, cols))
        else:                            # singular values near one, and those of the update's own singular vectors
            assert float((x.double() @ x.double().T if rows <= cols else x.double().T @ x.double()).diagonal().max()) < 1.5


def test_the_limits_of_matrices_that_a_workgroup_does_alone():
    from i6_native_ops_amd.training import orthogonalize
    for rows, cols in [(16, 1024), (16, 1025), (1, 1024), (17, 512), (32, 513), (512, 32), (33, 256), (64, 257), (65, 128), (128, 129), (129, 128), (15, 15), (2, 2000)]:
        u = matrix(rows, cols, torch.float32, seed=rows)
        check(orthogonalize([u])[0], expected(u), max(rows, cols))


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 5, 9])
def test_numbers_of_iterations(steps):
    from i6_native_ops_amd.training import orthogonalize
    u = matrix(90, 140, torch.float32)
    check(orthogonalize([u], steps=steps)[0], expected(u, steps), 140)
    check(orthogonalize([u.T.contiguous()], steps=steps)[0], expected(u, steps).T, 140)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e15])
def test_sizes_of_values(size, dtype):
    """The result does not depend on an update's size, down to a norm of 1e-7, below which it does not grow."""
    from i6_native_ops_amd.training import orthogonalize
    u = matrix(60, 100, dtype, size=size)
    check(orthogonalize([u])[0], expected(u), 100)


def test_single_values_and_zeros_and_what_is_no_number():
    from i6_native_ops_amd.training import orthogonalize
    one = torch.zeros((40, 50), device="cuda")
    one[3, 7] = -2.0
    zero = torch.zeros((40, 50), device="cuda")
    bad = matrix(40, 50, torch.float32)
    bad[1, 1] = float("nan")
    endless = matrix(40, 50, torch.float32)
    endless[1, 1] = float("inf")
    good = matrix(40, 50, torch.float32)
    got = orthogonalize([one, zero, bad, endless, good])
    check(got[0], expected(one), 50)
    assert (got[1] == 0).all() and torch.isnan(got[2]).any() and torch.isnan(got[3]).any()
    check(got[4], expected(good), 50)


def test_singular_values_end_near_one():
    from i6_native_ops_amd.training import orthogonalize
    g = gen(3)
    u = torch.linalg.qr(torch.randn((200, 200), generator=g, device="cuda").double().cpu())[0]
    v = torch.linalg.qr(torch.randn((300, 200), generator=g, device="cuda").double().cpu())[0]
    s = torch.logspace(0, -1.5, 200, dtype=torch.float64)
    x = orthogonalize([((u * s) @ v.T).float().cuda()])[0]
    values = torch.linalg.svdvals(x.double().cpu())
    # the map of the singular values, whose largest is 1.2 and which five iterations bring from 0.0022 (a norm of 4.7 here, 0.032 / 4.7 = 0.0067) over 0.68
    assert float(values.max()) < 1.21 and float(values.min()) > 0.68


def muon_expected(p, g, m, lr, mu, nesterov, decay, scale):
    p, g, m = p.double(), g.double(), m.double()
    m = mu * m + (1 - mu) * g
    u = mu * m + (1 - mu) * g if nesterov else m
    return p * (1 - lr * decay) - lr * scale * expected(u), m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw"])
def test_steps_of_muon(adjust, nesterov, dtype):
    from i6_native_ops_amd.training import muon_step
    sizes = [(64, 64), (128, 40), (40, 128), (1, 30)]
    params = [matrix(r, c, dtype, seed=i, size=0.05) for i, (r, c) in enumerate(sizes)]
    momenta = [matrix(r, c, torch.float32, seed=20 + i) for i, (r, c) in enumerate(sizes)]
    for step in range(2):
        grads = [matrix(r, c, dtype, seed=40 + i + 10 * step) for i, (r, c) in enumerate(sizes)]
        want = []
        for p, g, m, (r, c) in zip(params, grads, momenta, sizes):
            scale = max(1.0, r / c) ** 0.5 if adjust == "original" else 0.2 * max(r, c) ** 0.5
            want.append(muon_expected(p, g, m, 0.02, 0.9, nesterov, 0.1, scale) + (0.02 * scale,))
        versions = [p._version for p in params]
        muon_step(params, grads, momenta, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust)
        assert all(p._version > v for p, v in zip(params, versions))
        for p, m, (wp, wm, rate) in zip(params, momenta, want):
            assert (m.double() - wm).abs().max() <= 4 * EPS32 * wm.abs().max()
            out = EPS16 if dtype == torch.bfloat16 else 2 * EPS32
            bound = rate * 7 * 142 * 2 * (2.0 ** -23 + EPS32 * 128 ** 0.5) * 8 / min(p.shape) ** 0.5 + out * wp.abs()
            assert ((p.double() - wp).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_optimiser(dtype):
    """As torch's own, whose products are bfloat16's (2^-8 of each value, grown like the errors above in directions of small singular values: a fifth of the step)."""
    from i6_native_ops_amd.training import Muon
    start = [matrix(r, c, dtype, seed=i, size=0.005) for i, (r, c) in enumerate([(96, 64), (64, 96)])]
    ours, theirs = [torch.nn.Parameter(x.clone()) for x in start], [torch.nn.Parameter(x.clone()) for x in start]
    opt = Muon(ours, lr=0.02, weight_decay=0.1)
    ref = torch.optim.Muon(theirs, lr=0.02, weight_decay=0.1)
    for step in range(3):
        for i, (p, q) in enumerate(zip(ours, theirs)):
            p.grad = matrix(*p.shape, dtype, seed=9 * step + i)
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
    for p, q, s in zip(ours, theirs, start):
        moved = (q.double() - s.double()).norm()
        assert float((p.double() - q.double()).norm() / moved) < 0.2
    saved = opt.state_dict()
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    other = Muon(twin, lr=0.02, weight_decay=0.1)
    other.load_state_dict(saved)
    for p, q in zip(ours, twin):
        p.grad = matrix(*p.shape, dtype, seed=77)
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    for p, q in zip(ours, twin):
        assert torch.equal(p, q) and other.state[q]["momentum"].dtype == torch.float32


def test_captured_steps_and_another_stream():
    """A captured step is the same for every replay but for what the tensors hold: momenta and parameters move on."""
    from i6_native_ops_amd.training import muon_step, orthogonalize
    params, momenta = [matrix(96, 64, torch.float32, size=0.05)], [torch.zeros((96, 64), device="cuda")]
    grads = [matrix(96, 64, torch.float32, seed=5)]
    other = [x.clone() for x in params], [x.clone() for x in momenta]
    muon_step(*other[:1], grads, other[1], lr=0.02)
    other = [x.clone() for x in params], [x.clone() for x in momenta]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(params, grads, momenta, lr=0.02)
    for step in range(4):
        grads[0].copy_(matrix(96, 64, torch.float32, seed=5 + step))
        graph.replay()
        muon_step(other[0], grads, other[1], lr=0.02)
        torch.cuda.synchronize()
        assert torch.equal(params[0], other[0][0]) and torch.equal(momenta[0], other[1][0]), step
    u = matrix(200, 100, torch.float32)
    want = orthogonalize([u])[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize([u])[0]
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    from i6_native_ops_amd.training import Muon, muon_step, orthogonalize
    u = matrix(8, 6, torch.float32)
    for updates, match in [([u.cpu()], "contiguous CUDA matrix"), ([u.half()], "Expected updates"), ([u, u.bfloat16()], "of the type and on the device"), ([u[0]], "matrix"),
                           ([u.T], "contiguous"), ([torch.zeros((32769, 1), device="cuda")], "larger than")]:
        with pytest.raises(RuntimeError, match=match):
            orthogonalize(updates)
    with pytest.raises(RuntimeError, match="steps must be"):
        orthogonalize([u], steps=-1)
    with pytest.raises(RuntimeError, match="no gradient"):
        orthogonalize([u.clone().requires_grad_()])
    m = torch.zeros_like(u)
    with pytest.raises(RuntimeError, match="same length"):
        muon_step([u], [], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="grads"):
        muon_step([u], [u[:4]], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="momenta"):
        muon_step([u], [u.clone()], [m.bfloat16()], lr=0.1)
    with pytest.raises(RuntimeError, match="momentum must be"):
        muon_step([u], [u.clone()], [m], lr=0.1, momentum=1.0)
    with pytest.raises(ValueError):
        muon_step([u], [u.clone()], [m], lr=0.1, adjust_lr="other")
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(5, device="cuda"))])
    # memory that would be written twice, or read after it has been written
    g, buffer = u.clone(), torch.zeros(2, 8, 6, device="cuda")
    for params, grads, momenta in [([u, u], [g, g], [m, m.clone()]), ([u, u.clone()], [g, g], [m, m]), ([u], [m], [m]), ([u], [g], [u]), ([u], [u], [m]),
                                   ([buffer.view(-1)[:48].view(8, 6), buffer.view(-1)[24:72].view(8, 6)], [g, g], [m, m.clone()])]:
        with pytest.raises(RuntimeError, match="memory"):
            muon_step(params, grads, momenta, lr=0.1)
    muon_step([buffer[0], buffer[1]], [g, g], [m, m.clone()], lr=0.1)       # one gradient for two, side by side
    assert torch.equal(buffer[0], buffer[1]) and float(buffer.abs().max()) > 0
    muon_step([], [], [], lr=0.1)
