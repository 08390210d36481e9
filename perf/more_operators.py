"""The second set of operators whose speed this repository looks after: each stands beside one of the first set
(``perf/operators.py``), through the public functions of ``i6_native_ops_amd.training``.

* ``target_log_probs``: from the scores of all classes the log probability of given ones, the entropy and the best
  alternatives of every frame, with gradients: confidences, rescoring, the classes a search goes on with; beside
  ``linear_cross_entropy``;
* ``gated_delta_rule``: a recurrence over the frames whose state is a matrix per head, written to by keys and read by
  queries, its gradient, and its form for single frames; beside ``gated_recurrence``;
* ``orthogonalize``: the orthogonal factor of updates by Newton-Schulz products, the work of a ``Muon`` step; beside
  ``adamw_step``.

With ``own`` false, ``run`` computes the same from elementary operations in 32 bits.
"""
import math

import torch

own = False

NORM_EPS = 1e-6                              # under the root of the length of keys and queries
QUINTIC = (3.4445, -4.7750, 2.0315)          # x -> a x + b x^3 + c x^5 on the singular values
CHUNK = 64                                   # frames of a chunk in the plain form


def listed():
    return [
        # recognition, the next frame of 64 streams: tied triphone states, the classes a search goes on with
        dict(name="logp_step", op="logp", B=64, T=1, F=12001, k=16, dtype="float32", train=False, shortest=1.0, masked=0.0),
        # confidences of an alignment on the headline batch
        dict(name="logp_cart", op="logp", B=32, T=1000, F=12001, k=8, dtype="float32", train=False, shortest=0.8, masked=0.0),
        # subword units in bfloat16: a loss on log probability, entropy and alternatives; units that a mask excludes
        dict(name="logp_units_train", op="logp", B=256, T=200, F=5001, k=4, dtype="bfloat16", train=True, shortest=0.75, masked=0.1),
        # monophone states: short rows
        dict(name="logp_monophone_train", op="logp", B=32, T=500, F=264, k=5, dtype="float32", train=True, shortest=0.8, masked=0.0),
        # the recurrence while recognising: the next frame of 64 streams
        dict(name="delta_step", op="delta", B=64, T=1, H=8, G=8, K=128, V=128, dtype="bfloat16", train=False, shortest=1.0),
        # ragged odd batch in 32 bits, two value heads to a key head
        dict(name="delta_ragged_fp32", op="delta", B=19, T=437, H=6, G=3, K=40, V=72, dtype="float32", train=True, shortest=0.0),
        # the layer in training on the headline batch, 1024 channels
        dict(name="delta_cart", op="delta", B=32, T=1000, H=8, G=8, K=128, V=128, dtype="bfloat16", train=True, shortest=0.8),
        # one recording of five minutes
        dict(name="delta_recording", op="delta", B=1, T=30000, H=8, G=8, K=64, V=64, dtype="bfloat16", train=False, shortest=1.0),
        # the layers of the smallest model
        dict(name="orth_tiny", op="orth", layers=2, rows=128, cols=64, dtype="float32"),
        # an encoder of 1024 channels
        dict(name="orth_cart", op="orth", layers=12, rows=2048, cols=1024, dtype="float32"),
        # a large one in bfloat16
        dict(name="orth_large", op="orth", layers=24, rows=4096, cols=2048, dtype="bfloat16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("logp", "delta", "orth"))
    dtype = rng.choice(("float32", "bfloat16"))
    if op == "orth":
        rows, cols = _log_uniform(rng, 8, 4096), _log_uniform(rng, 8, 4096)
        small, large = min(rows, cols), max(rows, cols)
        most = 24 * (2 * 2048 ** 2 * 4096 + 2048 ** 3) // (2 * small ** 2 * large + small ** 3)
        return dict(op=op, layers=_log_uniform(rng, 1, max(1, min(24, most))), rows=rows, cols=cols, dtype=dtype)
    shortest = round(rng.uniform(0.0, 1.0), 2)
    train = rng.random() < 0.6
    T = 1 if rng.random() < 0.2 else _log_uniform(rng, 2, 4000 if op == "logp" else 12000)
    if op == "logp":
        F = _log_uniform(rng, 2, 30000)
        B = _log_uniform(rng, 1, max(1, min(256, 380_000_000 // (T * F))))
        T = min(T, 380_000_000 // (B * F))
        k = min(F, rng.choice((0, 1, rng.randint(2, 16), rng.randint(17, 64))))
        return dict(op=op, B=B, T=T, F=F, k=k, dtype=dtype, train=train, shortest=shortest, masked=rng.choice((0.0, 0.0, 0.3)))
    G = rng.randint(1, 8)
    H = G * rng.choice((1, 1, 2, 4))
    K, V = _log_uniform(rng, 8, 128), _log_uniform(rng, 8, 128)
    if rng.random() < 0.5:
        K, V = rng.choice((32, 64, 128)), rng.choice((32, 64, 128))
    most = 250_000_000 if not train else 32_000_000
    B = _log_uniform(rng, 1, max(1, min(128, most // (T * H * max(K, V)))))
    return dict(op=op, B=B, T=T, H=H, G=G, K=K, V=V, dtype=dtype, train=train, shortest=shortest)


# ------------------------------------------------------------------------------------------------------------- inputs


def _lens(case, gen, dev):
    B, T = case["B"], case["T"]
    lens = torch.randint(int(case["shortest"] * T), T + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
    lens[B // 2] = T
    return lens


def _prepare_logp(case, gen, dev):
    B, T, F, k = (case[n] for n in ("B", "T", "F", "k"))
    dtype = getattr(torch, case["dtype"])
    targets = torch.randint(0, F, (B, T), generator=gen, device=dev, dtype=torch.int32)
    # scores of a model that has learned something: the target's are raised, in some frames far above all others
    logits = torch.randn((B, T, F), generator=gen, device=dev).mul_(3.0)
    sure = torch.rand((B, T), generator=gen, device=dev).mul_(24.0)
    logits.scatter_add_(2, targets.long()[:, :, None], sure[:, :, None])
    if case["masked"]:
        excluded = torch.rand((F,), generator=gen, device=dev) < case["masked"]
        excluded[0] = False
        keep = torch.zeros((B, T, F), dtype=torch.bool, device=dev).scatter_(2, targets.long()[:, :, None], True)
        logits.masked_fill_(excluded & ~keep, -math.inf)
        del keep
    state = dict(logits=logits.to(dtype).requires_grad_(case["train"]), targets=targets, lens=_lens(case, gen, dev), k=k, train=case["train"])
    if case["train"]:
        share = 1.0 / max(1, B * T)
        for name, shape in (("grad_log_prob", (B, T)), ("grad_entropy", (B, T)), ("grad_top", (B, T, k))):
            state[name] = torch.randn(shape, generator=gen, device=dev) * share
    return state


def _prepare_delta(case, gen, dev):
    B, T, H, G, K, V = (case[n] for n in ("B", "T", "H", "G", "K", "V"))
    dtype = getattr(torch, case["dtype"])
    state = dict(lens=_lens(case, gen, dev), train=case["train"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    # keys that neighbouring frames share in part, as those of speech do
    near = normal(B, (T + 7) // 8, G, K).repeat_interleave(8, dim=1)[:, :T]
    values = dict(q=normal(B, T, G, K) + 0.5 * near, k=normal(B, T, G, K) + near, v=normal(B, T, H, V))
    # heads that keep their state for between three and some hundred frames; half of what a key holds is replaced on the average
    values["gate"] = normal(B, T, H) + torch.linspace(1.0, 6.0, H, device=dev)
    values["beta"] = normal(B, T, H)
    for name, x in values.items():
        state[name] = x.to(dtype).requires_grad_(case["train"])
    state["initial"] = normal(B, H, K, V).requires_grad_(case["train"])
    if case["train"]:
        state["grad_o"] = normal(B, T, H, V).to(dtype)
        state["grad_last"] = normal(B, H, K, V)
    return state


def _prepare_orth(case, gen, dev):
    rows, cols = case["rows"], case["cols"]
    dtype = getattr(torch, case["dtype"])
    updates = []
    for _ in range(case["layers"]):
        # a few directions that many examples agree on, and noise
        rank = max(1, min(rows, cols) // 16)
        size = torch.exp(-4.0 * torch.rand(rank, generator=gen, device=dev))
        part = (torch.randn((rows, rank), generator=gen, device=dev) * size) @ torch.randn((rank, cols), generator=gen, device=dev)
        noise = torch.randn((rows, cols), generator=gen, device=dev)
        updates.append(((part / math.sqrt(rank) + 0.2 * noise) * 1e-3).to(dtype))
    return dict(updates=updates)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    state = {"logp": _prepare_logp, "delta": _prepare_delta, "orth": _prepare_orth}[case["op"]](case, gen, dev)
    state["op"] = case["op"]
    return state


# -------------------------------------------------------------------------------------------------------- plain forms


def _best(z, k):
    """The k largest of the last dimension, each with the lowest index of those that equal it."""
    bits = (z + 0.0).view(torch.int32)
    key = bits ^ ((bits >> 31) & 0x7FFFFFFF)                     # whole numbers in the order of the values
    number = torch.arange(z.shape[-1], device=z.device, dtype=torch.int32)
    found = []
    for _ in range(k):
        largest = key.amax(dim=-1, keepdim=True)
        found.append(torch.where(key == largest, number, z.shape[-1]).amin(dim=-1, keepdim=True))
        key.scatter_(-1, found[-1].long(), -2 ** 31)             # below minus infinity's
    return torch.cat(found, dim=-1) if k else number.new_zeros(z.shape[:-1] + (0,))


def _plain_logp(s):
    B, T, F = s["logits"].shape
    live = torch.arange(T, device=s["lens"].device) < s["lens"][:, None]
    z = s["logits"].detach().float()
    classes = _best(z, s["k"])
    index = s["targets"].long()[:, :, None]
    z = z - z.amax(dim=2, keepdim=True)
    e = torch.exp(z)
    # the largest apart from the others, so that their small shares are not lost beside its 1
    largest = z == 0
    n = largest.sum(dim=2, keepdim=True).float()
    rest = torch.where(largest, 0.0, e).sum(dim=2, keepdim=True)
    total, log_total = n + rest, n.log() + torch.log1p(rest / n)
    entropy = log_total - torch.where(e > 0, e * z, 0.0).sum(dim=2, keepdim=True) / total
    out = {
        "log_prob": torch.where(live, (z.gather(2, index) - log_total)[:, :, 0], 0.0),
        "entropy": torch.where(live, entropy[:, :, 0], 0.0),
        "top_log_probs": torch.where(live[:, :, None], z.gather(2, classes.long()) - log_total, 0.0),
        "top_classes": torch.where(live[:, :, None], classes, -1),
    }
    if not s["train"]:
        return out
    gl, ge, gt = s["grad_log_prob"][:, :, None], s["grad_entropy"][:, :, None], s["grad_top"]
    p = e.div_(total)
    grad = torch.where(p > 0, p * (ge * (log_total - entropy - z) - gl - gt.sum(dim=2, keepdim=True)), 0.0)
    grad.scatter_add_(2, index, gl).scatter_add_(2, classes.long(), gt)
    out["logits"] = torch.where(live[:, :, None], grad, 0.0).to(s["logits"].dtype)
    return out


def _length(x):
    """1 / length of the rows; of no row is it infinite"""
    return 1.0 / (x.square().sum(dim=-1, keepdim=True) + NORM_EPS).sqrt()


def _plain_delta(s):
    """Chunks of C frames.  With c the sums of log f within a chunk and S the state in front of it, the rows u that are
    written solve (1 + A) u = beta (v - exp(c) k S), A_ij = beta_i exp(c_i - c_j) k_i k_j for j < i; then
    o = exp(c) q S + P u, P_ij = exp(c_i - c_j) q_i k_j for j <= i, and S' = exp(c_C) S + (exp(c_C - c) k)' u."""
    B, T, H, V = s["v"].shape
    G, K = s["k"].shape[2:]
    C = min(CHUNK, T)
    N = -(-T // C)
    live = torch.arange(N * C, device=s["lens"].device) < s["lens"][:, None]

    def chunks(x, heads):
        """[B, T, heads, n] -> [B, H, N, C, n] in 32 bits, 0 behind the end"""
        x = x.detach().float()
        x = torch.where(live[:, :T, None, None], x, 0.0)
        x = torch.cat([x, x.new_zeros((B, N * C - T) + x.shape[2:])], dim=1)
        return x.view(B, N, C, heads, -1).permute(0, 3, 1, 2, 4).repeat_interleave(H // heads, dim=1)

    def frames(x, heads, like):
        x = x.view(B, heads, H // heads, N, C, -1).sum(dim=2).permute(0, 2, 3, 1, 4).reshape(B, N * C, heads, -1)[:, :T]
        return x.to(like.dtype).reshape(like.shape)

    q, k, v = chunks(s["q"], G), chunks(s["k"], G), chunks(s["v"], H)
    rq, rk = _length(q), _length(k)
    q, k = q * rq, k * rk
    on = live.view(B, 1, N, C, 1)
    gate, beta = chunks(s["gate"][..., None], H), chunks(s["beta"][..., None], H)
    f = torch.where(on, 1.0 / (1.0 + torch.exp(-gate)), 1.0)
    log_f = torch.where(on, torch.clamp(gate, max=0.0) - torch.log1p(torch.exp(-gate.abs())), 0.0)
    beta = torch.where(on, 1.0 / (1.0 + torch.exp(-beta)), 0.0)
    c = log_f.double().cumsum(dim=3)                             # far larger than the differences that count
    low = torch.ones((C, C), dtype=torch.bool, device=q.device).tril()
    decay = torch.where(low, torch.exp((c - c.transpose(3, 4)).float().clamp(max=0.0)), 0.0)
    from_start, to_end = torch.exp(c.float()), torch.exp((c[..., -1:, :] - c).float())
    kk = k @ k.transpose(3, 4)
    A = (beta * decay * kk).tril(-1)
    P = decay * (q @ k.transpose(3, 4))
    solve = -A
    for i in range(1, C):                                        # (1 + A)^-1 row by row
        solve[..., i, :i] += (solve[..., i, :i, None].clone() * solve[..., :i, :i]).sum(dim=-2)
    solve += torch.eye(C, device=q.device)
    x, w = solve @ (beta * v), solve @ (beta * from_start * k)
    qs, ke = from_start * q, to_end * k
    S = s["initial"].detach()
    u, o, states = torch.empty_like(v), torch.empty_like(v), []
    for n in range(N):
        states.append(S)
        u[:, :, n] = x[:, :, n] - w[:, :, n] @ S
        o[:, :, n] = qs[:, :, n] @ S + P[:, :, n] @ u[:, :, n]
        S = from_start[:, :, n, -1:] * S + ke[:, :, n].transpose(2, 3) @ u[:, :, n]
    out = {"o": frames(torch.where(on, o, 0.0), H, s["v"]), "last": S}
    if not s["train"]:
        return out
    do = chunks(s["grad_o"], H)
    D = s["grad_last"]
    du0 = P.transpose(3, 4) @ do
    dr, ends, S_end = torch.empty_like(v), [None] * N, S
    for n in reversed(range(N)):
        ends[n] = D
        dr[:, :, n] = solve[:, :, n].transpose(2, 3) @ (du0[:, :, n] + ke[:, :, n] @ D)
        D = from_start[:, :, n, -1:] * D + qs[:, :, n].transpose(2, 3) @ do[:, :, n] - (beta * from_start * k)[:, :, n].transpose(2, 3) @ dr[:, :, n]
    out["initial"] = D
    S, D = torch.stack(states, dim=2), torch.stack(ends, dim=2)
    after = torch.cat([S[:, :, 1:], S_end[:, :, None]], dim=2)
    dP = (do @ u.transpose(3, 4)).tril()
    dA = -(dr @ u.transpose(3, 4)).tril(-1)
    do_S, dr_S, u_D = do @ S.transpose(3, 4), dr @ S.transpose(3, 4), u @ D.transpose(3, 4)
    dq = from_start * do_S + (dP * decay) @ k
    E = dA * beta * decay
    dk = to_end * u_D + (dP * decay).transpose(3, 4) @ q + E @ k + E.transpose(3, 4) @ k - beta * from_start * dr_S
    # what decays from frame j to frame i: products that cross the frame in question
    M = dP * P + dA * A
    state_part = from_start * ((q * do_S).sum(-1, keepdim=True) - beta * (k * dr_S).sum(-1, keepdim=True))
    write_part = to_end * (k * u_D).sum(-1, keepdim=True)
    dc = M.sum(-1, keepdim=True) - M.sum(-2)[..., None] + state_part - write_part
    dc[..., -1, 0] += (after * D).sum(dim=(-1, -2))
    dlog = dc.double().flip(3).cumsum(dim=3).flip(3).float()
    out["gate"] = frames(torch.where(on, dlog / (1.0 + torch.exp(gate)), 0.0), H, s["gate"])
    out["beta"] = frames((dr * u).sum(-1, keepdim=True) * (1.0 - beta), H, s["beta"])
    out["v"] = frames(beta * dr, H, s["v"])
    out["q"] = frames((dq - q * (q * dq).sum(-1, keepdim=True)) * rq, G, s["q"])
    out["k"] = frames((dk - k * (k * dk).sum(-1, keepdim=True)) * rk, G, s["k"])
    return out


def _plain_orth(s):
    a, b, c = QUINTIC
    out = []
    for update in s["updates"]:
        x = update.float()
        if x.shape[0] > x.shape[1]:
            x = x.t()
        x = x / x.square().sum().sqrt().clamp(min=1e-7)
        for _ in range(5):
            A = x @ x.t()
            x = a * x + (b * A + c * (A @ A)) @ x
        out.append((x.t() if update.shape[0] > update.shape[1] else x).to(update.dtype))
    return out


# ---------------------------------------------------------------------------------------------------------------- run


def run(state):
    op = state["op"]
    if not own:
        return {"logp": _plain_logp, "delta": _plain_delta, "orth": _plain_orth}[op](state)
    if op == "orth":
        from i6_native_ops_amd.training import orthogonalize
        return orthogonalize(state["updates"], steps=5)
    if op == "logp":
        from i6_native_ops_amd.training import target_log_probs
        out = dict(zip(("log_prob", "entropy", "top_log_probs", "top_classes"),
                       target_log_probs(state["logits"], state["targets"], state["lens"], alternatives=state["k"])))
        if state["train"]:
            wanted = ("log_prob", "entropy", "top_log_probs") if state["k"] else ("log_prob", "entropy")
            grads = [state[n] for n in ("grad_log_prob", "grad_entropy", "grad_top")][:len(wanted)]
            out["logits"], = torch.autograd.grad([out[n] for n in wanted], [state["logits"]], grads)
        return out
    from i6_native_ops_amd.training import gated_delta_rule
    names = ("q", "k", "v", "gate", "beta", "initial")
    inputs = [state[n] for n in names]
    o, last = gated_delta_rule(*inputs[:5], seq_lens=state["lens"], initial_state=inputs[5])
    out = {"o": o, "last": last}
    if state["train"]:
        out |= zip(names, torch.autograd.grad([o, last], inputs, [state["grad_o"], state["grad_last"]]))
    return out


# ------------------------------------------------------------------------------------------------------------ 64 bits


def _exact_logp(s):
    B, T, F = s["logits"].shape
    k = s["k"]
    shapes = {"log_prob": (B, T), "entropy": (B, T), "top_log_probs": (B, T, k), "top_classes": (B, T, k)}
    out = {n: torch.zeros(shape, dtype=torch.float64, device="cuda") for n, shape in shapes.items()}
    out["top_classes"] = torch.full((B, T, k), -1, dtype=torch.int32, device="cuda")
    if s["train"]:
        out["logits"] = torch.zeros((B, T, F), dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(s["lens"][b])
        if n == 0:
            continue
        z = s["logits"][b, :n].detach().double()
        # the others' sum apart from the largest's 1, of which it may be less than 2^-53
        top, first = z.max(dim=1, keepdim=True)
        others = (z - top).exp().scatter(1, first, 0.0).sum(dim=1, keepdim=True)
        log_p = z - top - torch.log1p(others)
        p = log_p.exp()
        plogp = torch.where(p > 0, p * log_p, 0.0)
        y = s["targets"][b, :n].long()[:, None]
        order = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :k]
        out["log_prob"][b, :n] = log_p.gather(1, y)[:, 0]
        out["entropy"][b, :n] = -plogp.sum(dim=1)
        out["top_log_probs"][b, :n] = log_p.gather(1, order)
        out["top_classes"][b, :n] = order.int()
        if s["train"]:
            gl, ge, gt = (s[m][b, :n].double() for m in ("grad_log_prob", "grad_entropy", "grad_top"))
            direct = torch.zeros_like(z).scatter_add_(1, y, gl[:, None]).scatter_add_(1, order, gt)
            direct -= torch.where(p > 0, p * (gl[:, None] + gt.sum(dim=1, keepdim=True)), 0.0)
            out["logits"][b, :n] = direct - ge[:, None] * (plogp - p * plogp.sum(dim=1, keepdim=True))
    return out


def _exact_delta(s):
    """Frame by frame.  Backward from states kept every 64 frames."""
    B, T, H, V = s["v"].shape
    G, K = s["k"].shape[2:]
    dev = s["v"].device
    lens = s["lens"]

    def at(name, t):
        """frame t of all sequences; zeros where there is none"""
        x = s[name][:, t].detach().double()
        x = torch.where((t < lens).view(B, *[1] * (x.dim() - 1)), x, 0.0)
        return x.repeat_interleave(H // x.shape[1], dim=1)

    def unit(x):
        return x / (x.square().sum(dim=-1, keepdim=True) + NORM_EPS).sqrt()

    def step(S, t):
        on = (t < lens).view(B, 1, 1, 1)
        f = torch.sigmoid(at("gate", t))[:, :, None, None]
        k, v, beta = unit(at("k", t)), at("v", t), torch.sigmoid(at("beta", t))[:, :, None]
        kept = f * S
        miss = v - (kept * k[..., None]).sum(dim=2)
        return torch.where(on, kept + k[..., None] * (beta * miss)[:, :, None], S), kept, miss

    S = s["initial"].detach().double()
    kept_states = {}
    o = torch.zeros((B, T, H, V), dtype=torch.float64, device=dev)
    for t in range(T):
        if t % 64 == 0 and s["train"]:
            kept_states[t] = S
        S = step(S, t)[0]
        o[:, t] = (S * unit(at("q", t))[..., None]).sum(dim=2) * (t < lens)[:, None, None]
    out = {"o": o, "last": S}
    if not s["train"]:
        return out
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device=dev) for n in ("q", "k", "v", "gate", "beta")}

    def through_unit(x, d):
        n = (x.square().sum(dim=-1, keepdim=True) + NORM_EPS).sqrt()
        return d / n - x * (x * d).sum(dim=-1, keepdim=True) / n ** 3

    def shared(x):
        return x.view(B, G, H // G, -1).sum(dim=2)

    dS = s["grad_last"].double()
    for first in reversed(range(0, T, 64)):
        S, span = kept_states.pop(first), []
        for t in range(first, min(T, first + 64)):
            after, kept, miss = step(S, t)
            span.append((t, S, after, kept, miss))
            S = after
        for t, before, after, kept, miss in reversed(span):
            on = (t < lens).view(B, 1, 1, 1)
            q, k, beta, f = at("q", t), at("k", t), torch.sigmoid(at("beta", t)), torch.sigmoid(at("gate", t))
            do = at("grad_o", t)
            grads["q"][:, t] = shared(through_unit(q, (after * do[:, :, None]).sum(dim=3)))
            d = dS + unit(q)[..., None] * do[:, :, None]
            written = beta[..., None] * miss
            du = (d * unit(k)[..., None]).sum(dim=2)
            dmiss = beta[..., None] * du
            dk = (d * written[:, :, None]).sum(dim=3) - (kept * dmiss[:, :, None]).sum(dim=3)
            grads["k"][:, t] = shared(through_unit(k, dk)) * on[..., 0]
            grads["v"][:, t] = dmiss * on[..., 0]
            grads["beta"][:, t] = (du * miss).sum(dim=2) * beta * (1.0 - beta) * on[:, 0, 0]
            dkept = d - unit(k)[..., None] * dmiss[:, :, None]
            grads["gate"][:, t] = (dkept * kept).sum(dim=(2, 3)) * torch.sigmoid(-at("gate", t)) * on[:, 0, 0]
            dS = torch.where(on, f[..., None, None] * dkept, dS)
    return {**out, **grads, "initial": dS}


def _exact_orth(s):
    """The same polynomials of the Gram matrix, multiplied out first."""
    a, b, c = QUINTIC
    out = []
    for update in s["updates"]:
        x = update.double()
        wide = x.shape[0] <= x.shape[1]
        x = x / torch.linalg.matrix_norm(x).clamp(min=1e-7)
        gram = x @ x.mT if wide else x.mT @ x
        one = torch.eye(gram.shape[0], dtype=torch.float64, device=x.device)
        total = one
        for _ in range(5):
            factor = torch.addmm(a * one, gram, b * one + c * gram)
            total = factor @ total
            gram = factor @ gram @ factor
        out.append(total @ x if wide else x @ total)
    return out


def exact(case, seed):
    if case["op"] == "delta" and case["T"] * (4 if case["train"] else 1) * (1 + case["B"] * case["H"] * case["K"] * case["V"] // 2_000_000) > 60_000:
        return None                          # frame by frame it takes too long
    return {"logp": _exact_logp, "delta": _exact_delta, "orth": _exact_orth}[case["op"]](prepare(case, seed))


# --------------------------------------------------------------------------------------------------------------- work


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "orth":
        small, large = sorted((case["rows"], case["cols"]))
        # five times: both triangles of a symmetric product are one, x x' and its square are symmetric
        flops = 5 * (small * small * large + small ** 3 + 2 * small * small * large)
        return {"bytes": 2 * size * case["layers"] * small * large, "flops": case["layers"] * flops}
    B, T = case["B"], case["T"]
    frames = B * T * (1 + case["shortest"]) / 2                # those of the sequences; results are dense
    train = case["train"]
    if case["op"] == "logp":
        F, k = case["F"], case["k"]
        grads = (size * F + 8 + 4 * k) if train else 0
        return {"bytes": frames * F * size + B * T * (4 + 8 + 8 * k + grads), "flops": frames * F * (20 if train else 10)}
    H, G, K, V = (case[n] for n in ("H", "G", "K", "V"))
    inputs = size * (2 * G * K + H * V + 2 * H)                  # of a frame
    state = 4 * B * H * K * V
    moved = frames * inputs + B * T * size * H * V + 2 * state
    if train:
        moved += frames * size * H * V + B * T * inputs + 2 * state
    # of a frame and head: the state decays, is read by the key, written to, read by the query; and the gradients of that
    return {"bytes": moved, "flops": frames * H * K * V * (23 if train else 7)}
