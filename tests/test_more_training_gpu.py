"""The second set of training operators as they are used together: a recurrent layer with a matrix as its state, log probabilities of an alignment with an entropy term,
Muon for the layers between and AdamW for the rest.

Tolerances.  Gradients: the layers' products are torch's in float32, sums of at most D = 64 or B T = 120 terms, and the operators' have theirs of K + V + 4 * 32 terms and of F; an
error of each is 2^-24 times the number of its terms of the size of what is added up, four layers after one another, with a factor of 16 for what cancels.  In float32
that is 16 * 4 * 2^-24 * 400 = 1.5e-3 of a tensor's 2-norm at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H, K, V, D, F = 2, 16, 16, 64, 37
BOUND = 16 * 4 * 2.0 ** -24 * 400


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.project = torch.nn.Linear(D, 2 * H * K + H * V + 2 * H)
        self.back = torch.nn.Linear(H * V, D)
        self.output = torch.nn.Linear(D, F)

    def split(self, x):
        y = self.project(x)
        B, T = x.shape[:2]
        q, k, v, gate, beta = y.split([H * K, H * K, H * V, H, H], dim=-1)
        return q.reshape(B, T, H, K), k.reshape(B, T, H, K), v.reshape(B, T, H, V), gate + 2, beta

    def forward(self, x, lens=None, state=None):
        from i6_native_ops_amd.training import gated_delta_rule
        o, state = gated_delta_rule(*self.split(x), lens, state)
        return self.output(x + self.back(o.flatten(2))), state


def reference(model, x, lens, targets):
    """Scores, and the loss, in the model's own type by the definitions."""
    q, k, v, gate, beta = model.split(x)
    unit = lambda z: z / (z.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q, k, f, w = unit(q), unit(k), torch.sigmoid(gate), torch.sigmoid(beta)
    S, o = torch.zeros(x.shape[0], H, K, V, dtype=x.dtype), []
    for t in range(x.shape[1]):
        S = f[:, t, :, None, None] * S
        u = w[:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None]
        o.append((S * q[:, t, :, :, None]).sum(2))
    log_p = torch.log_softmax(model.output(x + model.back(torch.stack(o, 1).flatten(2))), -1)
    live = (torch.arange(x.shape[1])[None] < lens[:, None]).to(x.dtype)
    entropy = -(log_p.exp() * log_p).sum(-1)
    return -(live * (log_p.gather(-1, targets[..., None])[..., 0] + 0.1 * entropy)).sum()


def data(seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((4, 30, D), generator=g), torch.tensor([30, 17, 1, 25], dtype=torch.int32), torch.randint(0, F, (4, 30), generator=g)


def loss_of(model, x, lens, targets):
    from i6_native_ops_amd.training import target_log_probs
    scores, _ = model(x, lens)
    log_prob, entropy, _, _ = target_log_probs(scores, targets.int(), lens)
    return -(log_prob + 0.1 * entropy).sum()


def test_gradients_of_a_layer_with_its_loss():
    torch.manual_seed(1)
    model = Layer()
    exact = Layer().double()
    exact.load_state_dict(model.state_dict())
    x, lens, targets = data()
    want = reference(exact, x.double(), lens, targets)
    want.backward()
    model.cuda()
    loss = loss_of(model, x.cuda(), lens.cuda(), targets.cuda())
    loss.backward()
    assert abs(float(loss) - float(want)) <= BOUND * abs(float(want))
    for (name, p), q in zip(model.named_parameters(), exact.parameters()):
        d = (p.grad.double().cpu() - q.grad).norm() / q.grad.norm()
        assert float(d) <= BOUND, (name, float(d))


def test_steps_of_both_optimisers_and_single_frames():
    """What a step changes is what the optimisers' own functions make of the gradients, and frames one by one give the scores of whole sequences."""
    from i6_native_ops_amd.training import AdamW, Muon, orthogonalize
    torch.manual_seed(2)
    model = Layer().cuda()
    x, lens, targets = (y.cuda() for y in data(5))
    between = [model.project.weight, model.back.weight]
    rest = [p for p in model.parameters() if all(p is not q for q in between)]
    muon, adamw = Muon(between, lr=0.02, weight_decay=0.0), AdamW(rest, lr=1e-3)
    for _ in range(3):
        before = [p.detach().clone() for p in between]
        muon.zero_grad(), adamw.zero_grad()
        loss = loss_of(model, x, lens, targets)
        loss.backward()
        muon.step(), adamw.step()
        assert torch.isfinite(loss) and all(torch.isfinite(p).all() for p in model.parameters())
        # nesterov's average of what the step has left in its state, and the gradient
        updates = [0.95 * muon.state[p]["momentum"] + 0.05 * p.grad for p in between]
        for p, b, o in zip(between, before, orthogonalize(updates)):
            rate = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            # two roundings of the update, 142 * 14 times larger in the result, and one of each value
            assert float((p - (b - rate * o)).norm()) <= rate * float(o.norm()) * 142 * 14 * 2.0 ** -23 + 2.0 ** -23 * float(b.norm())
    with torch.no_grad():
        whole, last = model(x)
        state, scores = None, []
        for t in range(x.shape[1]):
            s, state = model(x[:, t:t + 1], state=state)
            scores.append(s)
        assert float((torch.cat(scores, 1) - whole).norm()) <= BOUND * float(whole.norm())
        assert float((state - last).norm()) <= BOUND * float(last.norm())


def test_a_captured_step():
    """Forward, backward and Muon's step in a graph: replays are steps, like eager ones.  A gradient's sums have 120 terms, 2^-24 each if the products of a replay are added up in
    another order; orthogonalised, that is 142 * 14 times as much of matrices of at most 64 singular values up to 1.21, three times at rates of 0.02 sqrt(2.1)."""
    import copy

    from i6_native_ops_amd.training import muon_step
    torch.manual_seed(4)
    model = Layer().cuda()
    x, lens, targets = (y.cuda() for y in data(7))
    targets = targets.int()
    matrices = [model.project.weight, model.back.weight, model.output.weight]
    momenta = [torch.zeros_like(p) for p in matrices]
    start, stream = copy.deepcopy(model.state_dict()), torch.cuda.Stream()

    def step():
        grads = torch.autograd.grad(loss_of(model, x, lens, targets), matrices)
        with torch.no_grad():
            muon_step(matrices, [g.contiguous() for g in grads], momenta, lr=0.02)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    eager = [p.detach().clone() for p in matrices]

    def reset():
        model.load_state_dict(start)
        for m in momenta:
            m.zero_()

    reset()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(2):
        reset()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            x.square().mean().item()
        for p, e in zip(matrices, eager):
            assert float((p - e).norm()) <= 3 * 0.02 * 2.1 ** 0.5 * 142 * 14 * 120 * 2.0 ** -24 * 1.21 * 8, float((p - e).norm())
