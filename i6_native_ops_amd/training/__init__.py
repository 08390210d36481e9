"""What an emission model computes around the sequence losses, on MI355X.

``fbw_loss`` and ``align_viterbi`` start from log probabilities; the operators here stand in front of and behind them
in a training step on alignments, and in front of a search while recognising:

* ``linear_cross_entropy``: the output layer and the frame-wise cross entropy of an alignment (what ``align_viterbi``
  returns can be handed over as ``targets``), without the (B, T, F) logits;
* ``target_log_probs``: from such logits the log probabilities of targets, the entropy and the best alternatives of every frame,
  with gradients: confidences, rescoring, the classes a search goes on with;
* ``gated_recurrence``: a recurrence over the frames of a batch, with its gradient, and for single frames with a state;
* ``gated_delta_rule``: one whose state is a matrix for each head, written to by keys and read by queries, likewise;
* ``adamw_step`` / ``AdamW``: the update of all parameters at once, with states in 32 bits or in 8;
* ``orthogonalize`` / ``muon_step`` / ``Muon``: the orthogonal factors of updates of matrices, and the optimiser that goes along them.

The kernels are in libi6train.so (C ABI: include/i6train.h, i6logp.h, i6delta.h, i6orth.h).  As in the other modules nothing is compiled at import and
there is no fallback; problems only the device can see are raised by a later call or by ``check_status()``,
according to ``i6_native_ops_amd.fbw.set_status_mode``.  The reference has none of these operators.
"""
from typing import Iterable, List, Optional, Sequence, Tuple

import torch

from .._version import __version__  # noqa: F401

try:
    from . import training_core as core
except ImportError as exc:  # pragma: no cover - depends on the build state
    raise ImportError(
        "i6_native_ops_amd.training needs the built extension training_core; "
        "run `python -m i6_native_ops_amd.build`"
    ) from exc

BLOCK = 256     # values that share a scale where AdamW's states are held in 8 bits

check_status = core.check_status

__all__ = ["linear_cross_entropy", "target_log_probs", "gated_recurrence", "gated_delta_rule", "adamw_step", "AdamW", "orthogonalize", "muon_step", "Muon",
           "check_status", "core", "BLOCK"]


def linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.IntTensor,
    seq_lens: torch.IntTensor,
    bias: Optional[torch.Tensor] = None,
) -> torch.FloatTensor:
    """Frame-wise cross entropy of an output layer, ``-log_softmax(hidden @ weight.T + bias)`` at the targets, with
    the gradients with respect to ``hidden``, ``weight`` and ``bias``.  The logits are never stored.

    :param hidden: features of the frames, [B, T, D], float32 or bfloat16
    :param weight: [F, D], of the same type
    :param targets: int32 [B, T], e.g. the alignment of ``align_viterbi``; a negative target: the frame has none
    :param seq_lens: int32 [B]; frames behind the end are not looked at
    :param bias: [F], of the same type
    :return: float32 [B, T]; 0 in frames behind the end or without a target, NaN (and an error raised later) where a
        target is F or more
    """
    return core.linear_cross_entropy(hidden, weight, targets, seq_lens, bias)


def target_log_probs(
    logits: torch.Tensor,
    targets: torch.IntTensor,
    seq_lens: torch.IntTensor,
    alternatives: int = 0,
) -> Tuple[torch.FloatTensor, torch.FloatTensor, torch.FloatTensor, torch.IntTensor]:
    """Log probabilities of targets, the entropy and the best classes of every frame, in one pass over the scores of all classes, with the
    gradients of the first three with respect to ``logits``.

    :param logits: scores before the softmax (log probabilities are such, too), [B, T, F], float32 or bfloat16; -inf: a class without
        probability
    :param targets: int32 [B, T], e.g. the alignment of ``align_viterbi``; a negative target: the frame has none
    :param seq_lens: int32 [B]; frames behind the end are not looked at
    :param alternatives: k, number of classes to return for a frame, up to 64 and F
    :return: log probabilities of the targets [B, T] (0 without a target, NaN and an error raised later where it is F or more), entropies in
        nats [B, T], log probabilities [B, T, k] and classes (int32) [B, T, k] of the alternatives, the best first and the lowest index first
        among equal scores.  Behind the end: 0 and class -1.  A frame of -inf alone has log probabilities -inf, entropy 0 and gradient 0; one with NaN or
        +inf has NaN and class -1.
    """
    return core.target_log_probs(logits, targets, seq_lens, int(alternatives))


def gated_recurrence(
    x: torch.Tensor,
    gate: torch.Tensor,
    seq_lens: Optional[torch.IntTensor] = None,
    initial_state: Optional[torch.FloatTensor] = None,
) -> Tuple[torch.Tensor, torch.FloatTensor]:
    """Gated recurrence over the frames: with f = sigmoid(gate), ``h[t] = f[t] h[t-1] + (1 - f[t]) x[t]`` for every
    channel, and its gradient.

    :param x: [B, T, D], float32 or bfloat16
    :param gate: [B, T, D], before the sigmoid, of the same type
    :param seq_lens: int32 [B]; all T frames without.  Frames behind the end are not looked at
    :param initial_state: float32 [B, D], the state in front of the first frame; zeros without
    :return: h [B, T, D] in the type of x, 0 behind the end, and the state after the last frame of every sequence, float32
        [B, D].  The next frames of the same streams start from it: ``h, state = gated_recurrence(x, gate, initial_state=state)``
    """
    return core.gated_recurrence(x, gate, seq_lens, initial_state)


def gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    gate: torch.Tensor,
    beta: torch.Tensor,
    seq_lens: Optional[torch.IntTensor] = None,
    initial_state: Optional[torch.FloatTensor] = None,
) -> Tuple[torch.Tensor, torch.FloatTensor]:
    """A recurrence over the frames whose state S is a matrix for each head, and its gradient.  With f = sigmoid(gate), w = sigmoid(beta), and q and k scaled to
    length one (``k / sqrt(sum(k**2) + 1e-6)``): the state fades, ``S = f S``; what the key holds is replaced to the share w, ``S = S + outer(k, w (v - S.T @ k))``;
    and the query reads, ``o = S.T @ q``.

    :param q: [B, T, G, K], float32 or bfloat16, K up to 128; sums of squares below 2^127, as those of k
    :param k: of the same shape and type
    :param v: [B, T, H, V], of the same type, V up to 128; H is a multiple of G, and H / G neighbouring heads share a query and a key
    :param gate: [B, T, H], before the sigmoid, of the same type
    :param beta: [B, T, H], before the sigmoid, of the same type
    :param seq_lens: int32 [B]; all T frames without.  Frames behind the end are not looked at
    :param initial_state: float32 [B, H, K, V], the state in front of the first frame; zeros without
    :return: o [B, T, H, V] in the type of v, 0 behind the end, and the state after the last frame of every sequence, float32 [B, H, K, V].
        The next frames of the same streams start from it.  What is no number in v spoils its column of the head from its frame on, in k, gate or beta all of the head from the frame
        on, in q the frame's output; nothing in front of the frame.  Gradients of such a sequence's head are not defined
    """
    return core.gated_delta_rule(q, k, v, gate, beta, seq_lens, initial_state)


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    step: int,
    lr: float,
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    scales: Optional[Sequence[Tuple[torch.FloatTensor, torch.FloatTensor]]] = None,
) -> None:
    """One step of AdamW for all tensors, in place: ``torch.optim.AdamW``'s update.

    States are float32, or ``torch.float8_e4m3fn`` with ``scales``: for each tensor two float32 tensors with a scale
    for each 256 consecutive values.  In 8 bits ``exp_avg_sqs`` hold the square root of the second moment.

    :param params: contiguous tensors, all float32 or all bfloat16
    :param grads: of the same types and sizes
    :param step: number of this step, from 1.  It is part of the call: a captured step repeats this number, with its corrections, rate and
        roundings, at every replay
    """
    core.adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales or [], int(step), lr, betas[0], betas[1], eps, weight_decay)


def _load_states(optimizer: torch.optim.Optimizer, state_dict: dict) -> None:
    """The states keep their own types, which the base class would turn into those of the parameters."""
    torch.optim.Optimizer.load_state_dict(optimizer, state_dict)
    names = [i for g in state_dict["param_groups"] for i in g["params"]]
    params = [p for g in optimizer.param_groups for p in g["params"]]
    for name, p in zip(names, params):
        if name in state_dict["state"]:
            optimizer.state[p] = {k: v.detach().clone().to(p.device) if torch.is_tensor(v) else v for k, v in state_dict["state"][name].items()}


class AdamW(torch.optim.Optimizer):
    """AdamW on ``adamw_step``: one launch for the tensors of a parameter group.  ``step`` is not for capture into a graph, whose
    replays would all be the same step, and refuses it.

    :param state_bits: 32, or 8: a quarter of the optimiser's memory, and 16 instead of 28 bytes moved for each float32
        parameter in a step
    """

    def __init__(self, params: Iterable, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or eps < 0.0:
            raise ValueError("betas must be in [0, 1), eps must not be negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def _start(self, p: torch.Tensor, bits: int) -> dict:
        state = self.state[p]
        state["step"] = 0
        if bits == 8:
            blocks = (p.numel() + BLOCK - 1) // BLOCK
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                state[name + "_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step cannot be captured: every replay would be the step of this number, with its corrections and roundings")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                state = self.state[p] or self._start(p, group["state_bits"])
                calls.setdefault((p.device, p.dtype, state["step"] + 1), []).append((p, state))
            for (_, _, step), items in calls.items():
                scales = [(s["exp_avg_scale"], s["exp_avg_sq_scale"]) for _, s in items] if group["state_bits"] == 8 else None
                adamw_step([p for p, _ in items], [p.grad.contiguous() for p, _ in items], [s["exp_avg"] for _, s in items],
                           [s["exp_avg_sq"] for _, s in items], step, group["lr"], group["betas"], group["eps"], group["weight_decay"], scales)
                for _, state in items:       # a call that has been refused is no step
                    state["step"] = step
        return loss

    def load_state_dict(self, state_dict):
        _load_states(self, state_dict)


def orthogonalize(updates: Sequence[torch.Tensor], steps: int = 5) -> List[torch.Tensor]:
    """The matrices that the singular vectors of ``updates`` make with singular values near one: each update, divided by the root of its sum of squares, goes through
    ``steps`` times ``X = a X + (b A + c A @ A) @ X, A = X @ X.T`` with a, b, c = 3.4445, -4.775, 2.0315 (transposed where it has more rows than columns).

    :param updates: contiguous matrices of any sizes up to 32768, all float32 or all bfloat16; without a gradient
    :return: matrices of the same sizes and type
    """
    return core.orthogonalize(list(updates), int(steps))


def _rate(lr: float, shape, adjust_lr: str) -> float:
    rows, cols = shape
    if adjust_lr == "original":
        return lr * max(1.0, rows / cols) ** 0.5 if cols else lr
    if adjust_lr == "match_rms_adamw":
        return lr * 0.2 * max(rows, cols) ** 0.5
    raise ValueError("adjust_lr must be original or match_rms_adamw")


def muon_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    momenta: Sequence[torch.FloatTensor],
    lr: float,
    momentum: float = 0.95,
    nesterov: bool = True,
    weight_decay: float = 0.1,
    steps: int = 5,
    adjust_lr: str = "original",
) -> None:
    """One step of Muon for all matrices, in place: ``torch.optim.Muon``'s update, whose average of the gradients and products are held in float32 here (the
    products' operands in 22 bits).

    :param params: contiguous matrices, all float32 or all bfloat16
    :param grads: of the same types and sizes
    :param momenta: averages of the gradients, float32, of the same sizes.  Params, grads and momenta have memory of their own
    :param adjust_lr: the rate is multiplied by sqrt(max(1, rows / columns)) ("original") or by 0.2 sqrt(max(rows, columns)) ("match_rms_adamw")
    """
    rates = [_rate(lr, p.shape, adjust_lr) if p.dim() == 2 else lr for p in params]
    core.muon_step(list(params), list(grads), list(momenta), rates, momentum, bool(nesterov), lr * weight_decay, int(steps))


class Muon(torch.optim.Optimizer):
    """Muon on ``muon_step``: averaged gradients of matrices, orthogonalised.  For the weights between layers; biases, gains and output layers are for ``AdamW``.  ``step`` can be
    captured into a graph once every parameter has had one, or its state has been loaded."""

    def __init__(self, params: Iterable, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.1, steps: int = 5,
                 adjust_lr: str = "original"):
        if not 0.0 <= momentum < 1.0:
            raise ValueError("momentum must be in [0, 1)")
        _rate(lr, (1, 1), adjust_lr)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, adjust_lr=adjust_lr))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("Muon takes matrices; other parameters are for AdamW")

    @torch.no_grad()
    def step(self, closure=None):
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                state = self.state[p]
                if not state:
                    if capturing:
                        raise RuntimeError("Muon.step makes the averages of a parameter's gradients in its first step, which cannot be captured: every replay would begin them anew")
                    state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                calls.setdefault((p.device, p.dtype), []).append((p, state["momentum"]))
            for items in calls.values():
                muon_step([p for p, _ in items], [p.grad.contiguous() for p, _ in items], [m for _, m in items], group["lr"], group["momentum"], group["nesterov"],
                          group["weight_decay"], group["steps"], group["adjust_lr"])
        return loss

    def load_state_dict(self, state_dict):
        _load_states(self, state_dict)
