"""The recurrence with two channels a lane, which batches of many sequences and channels in bfloat16 get: several turns of the
workgroups, states kept in between, ends of every kind, and the same bits as with single channels."""
import pytest
import torch

from tests.test_training_gpu import close, rec_expected, rec_problem, rec_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,D", [(130, 300, 130), (257, 129, 64), (256, 65, 128), (256, 1, 66), (300, 14, 98), (86, 200, 270)])
def test_recurrence_in_pairs(B, T, D):
    problem = rec_problem(B, T, D, torch.bfloat16, seed=B + T + D)
    x, gate, lens, _, (dh, _) = problem
    lens[:5] = torch.tensor([0, 1, T, -3, T + 9], dtype=torch.int32, device="cuda")
    want = rec_expected(*problem)
    behind = torch.arange(T, device="cuda") >= lens[:, None]
    for v in (x, gate, dh):
        v[behind] = float("nan")
    got = rec_run(*problem)
    for k in got:
        close(got[k], *want[k], k)
        if k in ("h", "x", "gate"):
            assert (got[k][behind] == 0).all()


@pytest.mark.parametrize("B,T,D", [(130, 300, 130), (257, 129, 64), (256, 20, 66)])
def test_pairs_and_single_channels_round_alike(B, T, D):
    x, gate, lens, state, grads = rec_problem(B, T, D, torch.bfloat16, seed=3)
    want = rec_run(x, gate, lens, state, grads)
    odd = torch.zeros((T, B, D + 1), dtype=torch.bfloat16, device="cuda")       # rows that begin at odd places: single channels
    odd[:, :, 1:] = x.transpose(0, 1)
    for xs, gs, dh in ((odd.transpose(0, 1)[:, :, 1:], gate, grads[0]), (x, gate, odd.transpose(0, 1)[:, :, 1:])):
        ref = want if dh is grads[0] else rec_run(x, gate, lens, state, (dh.contiguous(), grads[1]))
        got = rec_run(xs, gs, lens, state, (dh, grads[1]))
        for k in got:
            assert torch.equal(got[k], ref[k]), k
