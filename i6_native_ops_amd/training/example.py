"""A small emission model trained and used with the operators of this package:  python -m i6_native_ops_amd.training.example

One recurrent layer over the frames of made-up utterances, three HMM states per label:

1. a few steps with the full-sum loss (``fbw_loss``), which needs no alignment;
2. the best path through each utterance's automaton with that model (``align_viterbi``);
3. training on this alignment frame by frame: ``linear_cross_entropy`` takes the alignment as it is and the output layer's
   weights, so the (B, T, F) logits are never there;
4. recognition of streams: frames arrive one by one, ``gated_recurrence`` goes on from the state of the last one.

All steps update the parameters with ``AdamW``, states in 8 bits.
"""
import math

import torch

from ..fast_viterbi import align_viterbi
from ..fbw import fbw_loss
from ..fsa import hmm_fsa
from . import AdamW, gated_recurrence, linear_cross_entropy

STATES = 3          # HMM states per label


class EmissionModel(torch.nn.Module):
    """Features -> inputs and gates of the recurrence -> states -> scores of the emission classes."""

    def __init__(self, features: int, channels: int, classes: int):
        super().__init__()
        self.project = torch.nn.Linear(features, 2 * channels)
        self.output = torch.nn.Linear(channels, classes)
        with torch.no_grad():       # gates that look back over a few frames at the start
            self.project.bias[channels:] = 0.5

    def hidden(self, frames, seq_lens=None, state=None):
        x, gate = self.project(frames).chunk(2, dim=-1)
        return gated_recurrence(x, gate, seq_lens, initial_state=state)

    def log_probs(self, hidden):
        return torch.log_softmax(self.output(hidden), dim=-1)


def utterances(n: int, labels: int, features: int, seed: int, device="cuda"):
    """(frames [B, T, features], their number [B], labels [B, L], states that produced the frames [B, T])"""
    gen = torch.Generator().manual_seed(seed)
    means = torch.randn((labels * STATES, features), generator=torch.Generator().manual_seed(0)) * 0.7
    said = torch.randint(0, labels, (n, 8), generator=gen, dtype=torch.int32)
    frames, states, lens = [], [], []
    for row in said:
        path = [int(label) * STATES + k for label in row for k in range(STATES)]
        stay = torch.randint(1, 5, (len(path),), generator=gen)
        seq = torch.tensor(path).repeat_interleave(stay)
        states.append(seq)
        lens.append(len(seq))
        frames.append(means[seq] + 0.7 * torch.randn((len(seq), features), generator=gen))
    T = max(lens)
    pad = torch.zeros
    frames = torch.stack([torch.cat([f, pad(T - len(f), features)]) for f in frames])
    states = torch.stack([torch.cat([s, pad(T - len(s), dtype=torch.long)]) for s in states])
    return frames.to(device), torch.tensor(lens, dtype=torch.int32, device=device), said.to(device), states.to(device)


def train(steps: int = 40, labels: int = 6, features: int = 16, channels: int = 64, sequences: int = 24, state_bits: int = 8, verbose: bool = False):
    """Trains the model as described above and returns what a caller may want to look at."""
    torch.manual_seed(1)
    device = torch.device("cuda")
    frames, seq_lens, said, states = utterances(sequences, labels, features, seed=2)
    label_lens = torch.full((sequences,), said.shape[1], dtype=torch.int32, device=device)
    live = torch.arange(frames.shape[1], device=device) < seq_lens[:, None]
    n_frames = int(live.sum())
    half = math.log(0.5)
    to_sum = hmm_fsa(said, label_lens, STATES, -half, -half)        # weights are costs for the sum ...
    to_align = hmm_fsa(said, label_lens, STATES, half, half)        # ... and log probabilities for the best path
    model = EmissionModel(features, channels, labels * STATES).to(device)
    opt = AdamW(model.parameters(), lr=1e-2, state_bits=state_bits)

    def right(log_probs):
        return float(((log_probs.argmax(-1) == states) & live).sum()) / n_frames

    seen = {"full_sum": [], "cross_entropy": []}
    for step in range(steps):
        opt.zero_grad()
        hidden, _ = model.hidden(frames, seq_lens)
        loss = fbw_loss(model.log_probs(hidden), to_sum, seq_lens)
        loss[0].sum().backward()          # the gradient of a sum over the frames, whatever it is multiplied by
        opt.step()
        seen["full_sum"].append(float(loss[0].sum().detach()) / n_frames)

    with torch.no_grad():
        hidden, _ = model.hidden(frames, seq_lens)
        log_probs = model.log_probs(hidden)
        alignment, _ = align_viterbi(log_probs, to_align, seq_lens)
    seen["aligned_right"] = float(((alignment == states) & live).sum()) / n_frames
    seen["right_after_full_sum"] = right(log_probs)

    # gradients are means over the frames from here on, far smaller than the sums above: the optimiser starts anew
    opt = AdamW(model.parameters(), lr=1e-2, state_bits=state_bits)
    for step in range(steps):
        opt.zero_grad()
        hidden, _ = model.hidden(frames, seq_lens)
        loss = linear_cross_entropy(hidden, model.output.weight, alignment, seq_lens, bias=model.output.bias)
        (loss.sum() / n_frames).backward()
        opt.step()
        seen["cross_entropy"].append(float(loss.sum().detach()) / n_frames)

    # frames of all streams as they arrive
    with torch.no_grad():
        state = torch.zeros((sequences, channels), device=device)
        scores = []
        for t in range(frames.shape[1]):
            h, state = model.hidden(frames[:, t:t + 1], state=state)
            scores.append(model.log_probs(h))
        streamed = torch.cat(scores, dim=1)
        whole = model.log_probs(model.hidden(frames, seq_lens)[0])
    seen["right"] = right(whole)
    seen["streamed_differs"] = float(((streamed - whole).abs() * live[:, :, None]).max())
    if verbose:
        print(f"full sum per frame      {seen['full_sum'][0]:.3f} -> {seen['full_sum'][-1]:.3f}, frames right {seen['right_after_full_sum']:.3f}")
        print(f"alignment               {seen['aligned_right']:.3f} of the frames as they were made")
        print(f"cross entropy per frame {seen['cross_entropy'][0]:.3f} -> {seen['cross_entropy'][-1]:.3f}, frames right {seen['right']:.3f}")
        print(f"frame by frame: scores differ by {seen['streamed_differs']:.1e} at most")
    return seen


if __name__ == "__main__":
    train(verbose=True)
