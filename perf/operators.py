"""The operators around the losses whose speed this repository looks after: what an emission model that is trained
on alignments or full sums computes besides them, through the public functions of ``i6_native_ops_amd.training``.

* ``linear_cross_entropy``: the output layer and the frame-wise cross entropy of an alignment, without the (B, T, F)
  logits, and the gradients of both;
* ``gated_recurrence``: a recurrence over the frames, h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate), its
  gradient, and its form for single frames;
* ``adamw_step``: the update of all parameters at once, with states in 32 bits or in 8.

With ``own`` false, ``run`` computes the same from elementary operations in 32 bits.
"""
import math

import torch

own = False

BLOCK = 256                     # values that share a scale where states are held in 8 bits
E4M3_MAX = 448.0                # largest finite value of the 8-bit format
LEAST_SCALE = 2.0 ** -100       # scale of a block of zeros
PHI = 2654435769                # 2^32 times the golden ratio's fraction
ROOT = 1779033703               # 2^32 times that of the square root of two
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01


def listed():
    return [
        # the output layer of the smallest model: ten classes, two short utterances; launches and host work
        dict(name="ce_tiny", op="ce", B=2, T=50, F=10, D=64, dtype="float32", train=True, shortest=0.8),
        # monophone states
        dict(name="ce_monophone", op="ce", B=32, T=500, F=264, D=512, dtype="bfloat16", train=True, shortest=0.8),
        # tied triphone states: the training step after align_viterbi on the headline workload
        dict(name="ce_cart", op="ce", B=32, T=1000, F=12001, D=512, dtype="bfloat16", train=True, shortest=0.8),
        # subword units, a large batch after subsampling, in 32 bits, an odd feature size
        dict(name="ce_units_fp32", op="ce", B=256, T=200, F=5001, D=500, dtype="float32", train=True, shortest=0.75),
        # the loss of held-out recordings of many minutes, without gradients
        dict(name="ce_longform_eval", op="ce", B=8, T=4000, F=12001, D=1024, dtype="bfloat16", train=False, shortest=0.5),
        # the recurrence while recognising: the next frame of 64 streams
        dict(name="rec_step", op="rec", B=64, T=1, D=1024, dtype="bfloat16", train=False, shortest=1.0),
        # ragged odd batch
        dict(name="rec_ragged_fp32", op="rec", B=19, T=437, D=321, dtype="float32", train=True, shortest=0.0),
        # the layer in training on the headline batch
        dict(name="rec_cart", op="rec", B=32, T=1000, D=1024, dtype="bfloat16", train=True, shortest=0.8),
        # one recording of five minutes, few channels for the chip
        dict(name="rec_recording", op="rec", B=1, T=30000, D=512, dtype="float32", train=False, shortest=1.0),
        # parameters of the smallest model, states in 32 bits
        dict(name="adamw_tiny", op="adamw", layers=2, D=64, F=10, dtype="float32", bits=32),
        # an encoder with tied triphone states, states in 32 bits
        dict(name="adamw_cart", op="adamw", layers=12, D=1024, F=12001, dtype="float32", bits=32),
        # a large one, states in 8 bits
        dict(name="adamw_large_8bit", op="adamw", layers=24, D=2048, F=12001, dtype="float32", bits=8),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choices(("ce", "rec", "adamw"), (5, 4, 3))[0]
    dtype = rng.choice(("float32", "bfloat16"))
    if op == "adamw":
        layers, D = rng.randint(1, 24), _log_uniform(rng, 16, 2048)
        F = _log_uniform(rng, 10, 12001)
        return dict(op=op, layers=layers, D=D, F=F, dtype=dtype, bits=rng.choice((8, 32)))
    shortest = round(rng.uniform(0.0, 1.0), 2)
    train = rng.random() < 0.7
    if op == "rec":
        D = _log_uniform(rng, 8, 2048)
        T = 1 if rng.random() < 0.2 else _log_uniform(rng, 2, 30000)
        most = 300_000_000 // max(10, int(math.log2(T) + 1))
        B = _log_uniform(rng, 1, max(1, min(256, most // (T * D))))
        return dict(op=op, B=B, T=T, D=min(D, max(8, most // (B * T))), dtype=dtype, train=train, shortest=shortest)
    D = _log_uniform(rng, 8, 1024)
    if rng.random() < 0.5:
        D = max(64, D // 64 * 64)
    F = _log_uniform(rng, 2, 12001)
    T = _log_uniform(rng, 1, 4000)
    B = _log_uniform(rng, 1, max(1, min(256, 32000 // T, 190_000_000_000 // (T * F * D))))
    return dict(op=op, B=B, T=T, F=F, D=D, dtype=dtype, train=train, shortest=shortest)


# ------------------------------------------------------------------------------------------------------------- inputs


def _lens(case, gen, dev):
    B, T = case["B"], case["T"]
    least = int(case["shortest"] * T)
    lens = torch.randint(least, T + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
    lens[B // 2] = T
    return lens


def _shapes(case):
    D, F = case["D"], case["F"]
    return case["layers"] * [(2 * D, D), (2 * D,), (D,)] + [(F, D), (F,)]


def _prepare_ce(case, gen, dev):
    B, T, F, D = case["B"], case["T"], case["F"], case["D"]
    dtype = getattr(torch, case["dtype"])
    # labels that last for a few frames, as an alignment has them
    runs = torch.randint(0, F, (B, T // 4 + 1), generator=gen, device=dev, dtype=torch.int32)
    targets = runs.repeat_interleave(4, dim=1)[:, :T].contiguous()
    weight = torch.randn((F, D), generator=gen, device=dev) / math.sqrt(D)
    bias = torch.randn((F,), generator=gen, device=dev) * 0.5
    # features of a model that has learned something: normalised, leaning towards their label's row
    hidden = torch.randn((B, T, D), generator=gen, device=dev) + 2.0 * weight[targets.long()]
    lens = _lens(case, gen, dev)
    # the mean over the frames of the batch
    state = dict(lens=lens, targets=targets, share=(1.0 / lens.sum().clamp(min=1)).float().expand(B, T).contiguous(), train=case["train"])
    for name, x in (("hidden", hidden), ("weight", weight), ("bias", bias)):
        state[name] = x.to(dtype).requires_grad_(case["train"])
    return state


def _prepare_rec(case, gen, dev):
    B, T, D = case["B"], case["T"], case["D"]
    dtype = getattr(torch, case["dtype"])
    state = dict(lens=_lens(case, gen, dev), train=case["train"])
    state["x"] = torch.randn((B, T, D), generator=gen, device=dev).to(dtype).requires_grad_(case["train"])
    # gates that keep the state for between one and some hundred frames
    keep = torch.linspace(-1.0, 5.0, D, device=dev)
    state["gate"] = (torch.randn((B, T, D), generator=gen, device=dev) + keep).to(dtype).requires_grad_(case["train"])
    state["initial"] = torch.randn((B, D), generator=gen, device=dev).requires_grad_(case["train"])
    if case["train"]:
        state["grad_h"] = torch.randn((B, T, D), generator=gen, device=dev).to(dtype)
        state["grad_last"] = torch.randn((B, D), generator=gen, device=dev)
    return state


def _prepare_adamw(case, gen, dev):
    dtype = getattr(torch, case["dtype"])
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for n in sizes:                       # one buffer for all tensors, as programs have that reduce it in one piece
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    used = torch.zeros(total, dtype=torch.bool, device=dev)
    for at, n in zip(starts, sizes):
        used[at:at + n] = True

    def normal():
        return torch.randn(total, generator=gen, device=dev) * used

    # gradients whose size varies over the tensors by a few powers of ten
    size = torch.exp(torch.randn(total // BLOCK, 1, generator=gen, device=dev) - 6.0).expand(-1, BLOCK).reshape(-1)
    p = (normal() * 0.05).to(dtype)
    g = (normal() * size).to(dtype)
    m, v = normal() * size * 0.2, (normal() * size).square_() * 0.5 + 0.5 * size.square() * used
    state = dict(step=1000, bits=case["bits"], flat=[p, g])
    if case["bits"] == 8:
        (m, ms), (v, vs) = _quantise(m, v, 999)
        state["flat"] += [m, v, ms, vs]
    else:
        state["flat"] += [m, v]

    def views(x, shaped=True, unit=1):
        if not shaped:
            return [x[at // BLOCK:at // BLOCK + -(-n // BLOCK)] for at, n in zip(starts, sizes)]
        return [x[at:at + n].view(s) for at, n, s in zip(starts, sizes, shapes)]

    state["lists"] = [views(x) for x in state["flat"][:4]]
    state["scales"] = list(zip(*(views(x, False) for x in state["flat"][4:]))) if case["bits"] == 8 else None
    return state


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    state = {"ce": _prepare_ce, "rec": _prepare_rec, "adamw": _prepare_adamw}[case["op"]](case, gen, dev)
    state["op"] = case["op"]
    return state


# -------------------------------------------------------------------------------------------------------- plain forms


def _plain_ce(s):
    B, T, D = s["hidden"].shape
    hidden, weight, bias = (s[k].detach().float() for k in ("hidden", "weight", "bias"))
    live = (torch.arange(T, device=hidden.device) < s["lens"][:, None]).reshape(-1, 1)
    index = s["targets"].reshape(-1, 1).long()
    rows = torch.where(live, hidden.reshape(-1, D), 0.0)
    logits = rows @ weight.t() + bias
    top = logits.amax(dim=1, keepdim=True)
    total_of = (logits - top).exp_()
    total = total_of.sum(dim=1, keepdim=True)
    loss = ((total.log() + top - logits.gather(1, index)) * live).view(B, T)
    if not s["train"]:
        return {"loss": loss}
    share = s["share"].reshape(-1, 1) * live
    grad = total_of.mul_(share / total)
    grad.scatter_add_(1, index, -share)
    dtype = s["hidden"].dtype
    return {"loss": loss, "hidden": (grad @ weight).view(B, T, D).to(dtype), "weight": (grad.t() @ rows).to(dtype), "bias": grad.sum(dim=0).to(dtype)}


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, from h = 0: spans of 1, 2, 4, ... frames joined in pairs."""
    T, span = a.shape[1], 1
    while span < T:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], dim=1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], dim=1)
        span *= 2
    return b


def _plain_rec(s):
    x, gate = s["x"].detach().float(), s["gate"].detach().float()
    initial = s["initial"].detach()
    T = x.shape[1]
    live = (torch.arange(T, device=x.device) < s["lens"][:, None])[:, :, None]
    f = torch.where(live, 1.0 / (1.0 + torch.exp(-gate)), 1.0)       # behind the end the state stays
    b = torch.where(live, (1.0 - f) * x, 0.0)
    b[:, 0] += f[:, 0] * initial
    h = _scan(f, b)
    out = {"h": torch.where(live, h, 0.0).to(s["x"].dtype), "last": h[:, -1]}
    if not s["train"]:
        return out
    d = torch.where(live, s["grad_h"].float(), 0.0)
    d[:, -1] += s["grad_last"]
    after = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], dim=1)
    d = _scan(after.flip(1), d.flip(1)).flip(1)
    before = torch.cat([initial[:, None], h[:, :-1]], dim=1)
    out["x"] = torch.where(live, d * (1.0 - f), 0.0).to(s["x"].dtype)
    out["gate"] = torch.where(live, d * (before - x) * f * (1.0 - f), 0.0).to(s["x"].dtype)
    out["initial"] = d[:, 0] * f[:, 0]
    return out


def _dither(step, dev):
    """For each place in a block two numbers in [0, 1) that decide which way the step rounds there.  From step to step
    they go round in irrational turns, so that over the steps every value is rounded up as often as it should be."""
    at = torch.arange(BLOCK, device=dev, dtype=torch.int64)
    turns = torch.stack([at * PHI + step * ROOT, at * ROOT + step * PHI]) & 0xFFFFFFFF
    return (turns >> 16).float() / 65536.0


def _quantum(y):
    """Distance of the 8-bit values around y."""
    exponent = (y.view(torch.int32) >> 23) & 255
    return ((exponent.clamp(min=121) - 3) << 23).view(torch.float32)


def _quantise(m, v, step):
    """Blocks of m and of the square root of v in 8 bits, with scales.  Both are rounded up with the probability that
    keeps the mean, of m and of v; a root that is not zero does not become zero."""
    um, uv = _dither(step, m.device)
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    scale = (m.abs().amax(dim=1, keepdim=True) / E4M3_MAX).clamp(min=LEAST_SCALE)
    y = m * (1.0 / scale)
    q = _quantum(y.abs())
    k = torch.floor(y.abs() / q + um) * q
    m8 = torch.copysign(k.clamp(max=E4M3_MAX), y).to(torch.float8_e4m3fn)
    r = v.sqrt()
    scale_r = (r.amax(dim=1, keepdim=True) / E4M3_MAX).clamp(min=LEAST_SCALE)
    y = r * (1.0 / scale_r)
    q = _quantum(y)
    low = torch.floor(y / q) * q
    up = (y * y - low * low > uv * (q * (low + low + q))) | ((low == 0) & (y > 0))
    r8 = torch.where(up, low + q, low).clamp(max=E4M3_MAX).to(torch.float8_e4m3fn)
    return (m8.view(-1), scale.view(-1)), (r8.view(-1), scale_r.view(-1))


def _plain_adamw(s):
    p, g, m, v = s["flat"][:4]
    step, bits = s["step"], s["bits"]
    if bits == 8:
        ms, vs = s["flat"][4:]
        m32 = (m.float().view(-1, BLOCK) * ms[:, None]).view(-1)
        v32 = (v.float().view(-1, BLOCK) * vs[:, None]).view(-1)
        v32 = v32 * v32
    else:
        m32, v32 = m, v
    g32 = g.float()
    m32 = m32 * BETA1 + g32 * (1.0 - BETA1)
    v32 = v32 * BETA2 + g32 * g32 * (1.0 - BETA2)
    size = v32.sqrt() * (1.0 / math.sqrt(1.0 - BETA2 ** step)) + EPS
    p.copy_(p.float() * (1.0 - LR * DECAY) - m32 / size * (LR / (1.0 - BETA1 ** step)))
    if bits == 8:
        (m8, ms8), (r8, vs8) = _quantise(m32, v32, step)
        m.copy_(m8), v.copy_(r8), ms.copy_(ms8), vs.copy_(vs8)
    else:
        m.copy_(m32), v.copy_(v32)


# ---------------------------------------------------------------------------------------------------------------- run


def run(state):
    op = state["op"]
    if op == "adamw":
        if own:
            from i6_native_ops_amd.training import adamw_step
            params, grads, m, v = state["lists"]
            adamw_step(params, grads, m, v, step=state["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, scales=state["scales"])
        else:
            _plain_adamw(state)
        state["step"] += 1
        names = ("params", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        return dict(zip(names, state["flat"][:1] + state["flat"][2:]))
    if not own:
        return _plain_ce(state) if op == "ce" else _plain_rec(state)
    from i6_native_ops_amd.training import gated_recurrence, linear_cross_entropy
    if op == "ce":
        inputs = [state[k] for k in ("hidden", "weight", "bias")]
        loss = linear_cross_entropy(inputs[0], inputs[1], state["targets"], state["lens"], bias=inputs[2])
        out = {"loss": loss}
        if state["train"]:
            out |= zip(("hidden", "weight", "bias"), torch.autograd.grad(loss, inputs, state["share"]))
        return out
    inputs = [state[k] for k in ("x", "gate", "initial")]
    h, last = gated_recurrence(inputs[0], inputs[1], state["lens"], initial_state=inputs[2])
    out = {"h": h, "last": last}
    if state["train"]:
        out |= zip(("x", "gate", "initial"), torch.autograd.grad([h, last], inputs, [state["grad_h"], state["grad_last"]]))
    return out


# ------------------------------------------------------------------------------------------------------------ 64 bits


def _exact_ce(s):
    inputs = [s[k].detach().double().requires_grad_(s["train"]) for k in ("hidden", "weight", "bias")]
    hidden, weight, bias = inputs
    B, T, D = hidden.shape
    at = torch.nonzero(torch.arange(T, device=hidden.device) < s["lens"][:, None], as_tuple=True)
    log_probs = torch.nn.functional.linear(hidden[at], weight, bias).log_softmax(dim=-1)
    picked = -log_probs.gather(1, s["targets"][at].long()[:, None])[:, 0]
    loss = torch.zeros((B, T), dtype=torch.float64, device=hidden.device).index_put(at, picked)
    if not s["train"]:
        return {"loss": loss}
    grads = torch.autograd.grad((loss * s["share"].double()).sum(), inputs)
    return {"loss": loss.detach(), **dict(zip(("hidden", "weight", "bias"), grads))}


def _exact_rec(s):
    x, gate, state = s["x"].detach().double(), s["gate"].detach().double(), s["initial"].detach().double()
    lens = s["lens"][:, None]
    B, T, D = x.shape
    f = torch.sigmoid(gate)
    h, before = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        before[:, t] = state
        state = torch.where(t < lens, torch.lerp(x[:, t], state, f[:, t]), state)
        h[:, t] = state * (t < lens)
    out = {"h": h, "last": state}
    if not s["train"]:
        return out
    dx, dg, d = torch.zeros_like(x), torch.zeros_like(x), s["grad_last"].double()
    for t in reversed(range(T)):
        live = t < lens
        d = torch.where(live, d + s["grad_h"][:, t].double(), d)
        dx[:, t] = d * torch.sigmoid(-gate[:, t]) * live
        dg[:, t] = d * (before[:, t] - x[:, t]) * f[:, t] * torch.sigmoid(-gate[:, t]) * live
        d = torch.where(live, d * f[:, t], d)
    return {**out, "x": dx, "gate": dg, "initial": d}


def _exact_round(y, up):
    """The 8-bit value under or over y >= 0: ``up(low, high)`` says which."""
    q = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3.0)
    low = torch.floor(y / q) * q
    return torch.where(up(low, low + q), low + q, low).clamp(max=E4M3_MAX)


def _exact_adamw(s):
    p, g, m, v = (x.double() for x in s["flat"][:4])
    step = s["step"]
    if s["bits"] == 8:
        m = m * s["flat"][4].double().repeat_interleave(BLOCK)
        v = (v * s["flat"][5].double().repeat_interleave(BLOCK)).square()
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g.square(), v, BETA2)
    ahead = (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)).sqrt() + EPS)
    out = {"params": p - LR * (ahead + DECAY * p)}
    if s["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    um, uv = _dither(step, p.device).double()
    m, r = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
    scale, scale_r = ((x.abs().amax(dim=1, keepdim=True) / E4M3_MAX).clamp(min=LEAST_SCALE) for x in (m, r))
    y = (m / scale).abs()
    m8 = _exact_round(y, lambda low, high: (y - low) / (high - low) + um >= 1.0) * m.sign()
    y = r / scale_r
    r8 = _exact_round(y, lambda low, high: (y.square() - low.square() > uv * (high.square() - low.square())) | ((low == 0) & (y > 0)))
    return {**out, "exp_avg": m8.view(-1), "exp_avg_sq": r8.view(-1), "exp_avg_scale": scale.view(-1), "exp_avg_sq_scale": scale_r.view(-1)}


def exact(case, seed):
    return {"ce": _exact_ce, "rec": _exact_rec, "adamw": _exact_adamw}[case["op"]](prepare(case, seed))


# --------------------------------------------------------------------------------------------------------------- work


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        # parameters and both states read and written, gradients read
        state = 4 * (1 + 4 / BLOCK) if case["bits"] == 8 else 16
        return {"bytes": n * (3 * size + state), "flops": 15 * n}
    B, T, D = case["B"], case["T"], case["D"]
    frames = B * T * (1 + case["shortest"]) / 2          # those of the sequences; results are dense
    if case["op"] == "rec":
        read = 3 * frames * D * size if case["train"] else 2 * frames * D * size
        write = 3 * B * T * D * size if case["train"] else B * T * D * size
        return {"bytes": read + write + (16 if case["train"] else 8) * B * D, "flops": (20 if case["train"] else 7) * frames * D}
    F = case["F"]
    read = size * (frames * D + F * D + F) + 4 * B * T
    write = 4 * B * T + (size * (B * T * D + F * D + F) if case["train"] else 0)
    # the logits once, and both products with their gradient
    return {"bytes": read + write, "flops": (6 if case["train"] else 2) * frames * F * D}
