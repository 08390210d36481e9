"""Log probabilities of targets where there are thousands of frames: rows have a wave each up to other lengths than among few frames, forward and backward.  Bounds as in test_logp_gpu.py,
whose terms (64 one after another, 96 more for long rows) cover a lane's 80 of 20 pieces of eight by twos."""
import pytest
import torch

from tests.test_logp_gpu import INF, check, expected, problem, run

pytestmark = pytest.mark.gpu

FEW, MANY = torch.float32, torch.bfloat16
SIZES = [(FEW, 500), (FEW, 1537), (FEW, 2500), (FEW, 2560), (FEW, 2561), (FEW, 2900), (FEW, 3100), (FEW, 5001), (FEW, 5120), (FEW, 5121),
         (MANY, 500), (MANY, 2900), (MANY, 4999), (MANY, 5120), (MANY, 5121), (MANY, 6144), (MANY, 6145), (MANY, 10240), (MANY, 10241)]


@pytest.mark.parametrize("dtype,F", SIZES)
@pytest.mark.parametrize("k,B,T", [(5, 5, 820), (0, 1, 4096), (64, 4096, 1)])
def test_many_frames(dtype, F, k, B, T):
    if k == 64 and F > 3100:
        B = 4097
    logits, targets, lens, k, grads = problem(B, T, F, k, dtype, seed=F + k, lens=[T] * B if T == 1 or B == 1 else [T, 0, T - 1, 1, T])
    rows, y = logits.view(B * T, F), targets.view(-1)
    lowest = torch.finfo(dtype).min
    rows[3] = -INF
    rows[4, 1:] = lowest
    rows[5, ::2] = -INF
    rows[6, : F - max(1, k // 2)] = -INF
    rows[7] = 1.5
    rows[8] = (torch.arange(F, device="cuda") % 5).to(dtype)
    rows[9] = torch.round(rows[9])
    rows[10] = torch.arange(F, device="cuda").float().mul(1 / 64).to(dtype)
    rows[11] = -rows[10]
    y[5], y[12] = 0, -1
    check(run(logits, targets, lens, k, grads), expected(logits, targets, lens, k, grads))


@pytest.mark.parametrize("dtype,F", [(FEW, 2500), (FEW, 5001), (MANY, 4999), (MANY, 10001)])
def test_many_frames_whose_rows_begin_anywhere(dtype, F):
    logits, targets, lens, k, grads = problem(6, 700, F, 3, dtype, seed=F)
    wide = torch.zeros((6, 700, F + 5), dtype=dtype, device="cuda")
    wide[..., 3:F + 3] = logits
    got, want = run(wide[..., 3:F + 3], targets, lens, k, grads), expected(logits, targets, lens, k, grads)
    check(got, want)


@pytest.mark.parametrize("dtype,F", [(FEW, 2500), (FEW, 5001), (MANY, 4999), (MANY, 10001)])
def test_many_frames_that_are_no_distribution(dtype, F):
    logits, targets, lens, k, grads = problem(1, 4100, F, 3, dtype, lens=[4100])
    logits[0, 100, F // 2], logits[0, 2000, F - 1], logits[0, 4099] = float("nan"), INF, float("nan")
    got = run(logits, targets, lens, k, grads)
    bad = torch.tensor([100, 2000, 4099], device="cuda")
    for n in ("log_prob", "entropy", "top", "logits"):
        assert torch.isnan(got[n][0, bad]).all(), n
    assert (got["classes"][0, bad] == -1).all()
    want = expected(logits.nan_to_num(0.0, 0.0), targets, lens, k, grads)
    keep = torch.ones(4100, dtype=torch.bool, device="cuda")
    keep[bad] = False
    check({n: x[:, keep] for n, x in got.items()}, {n: (w[:, keep], b[:, keep] if b is not None else None) for n, (w, b) in want.items()})


def test_alternatives_that_are_no_classes_are_passed_over():
    """At the C level a caller may hand over any alternatives: those outside of the row's classes count for nothing, and nothing is written for them."""
    import ctypes

    import i6_native_ops_amd.training as training
    from tests.test_more_training_cpu import Logp
    lib = ctypes.CDLL(training.__file__.replace("__init__.py", "libi6train.so"))
    B, T, F, k = 1, 3, 37, 4
    logits, targets, lens, _, grads = problem(B, T, F, k, FEW, lens=[T])
    room = torch.full((3, T, F), 5.0, device="cuda")                 # memory of its own on both sides
    floats = [torch.empty(n, device="cuda") for n in (B * T, B * T, B * T * k, B * T * 4)]
    classes = torch.empty(B * T * k, dtype=torch.int32, device="cuda")
    at = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
    p = Logp(B=B, T=T, F=F, k=k, dtype=0, logits=logits.data_ptr(), targets=targets.data_ptr(), lens=lens.data_ptr(), l_b=T * F, l_t=F, t_b=T, t_t=1)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.i6logp_forward(ctypes.byref(p), at(floats[0]), at(floats[1]), at(floats[2]), at(classes), at(floats[3]), stream) == 0
    gt = grads[2].clone()
    classes.view(T, k)[:, 1], classes.view(T, k)[:, 3] = F, -7       # both would be within `room`
    assert lib.i6logp_backward(ctypes.byref(p), at(floats[3]), at(classes), None, None, at(gt), at(room[1]), stream) == 0
    torch.cuda.synchronize()
    assert (room[0] == 5.0).all() and (room[2] == 5.0).all()
    # what comes in for them is in the frame's sum, but no class has it
    z = logits[0].double()
    direct = torch.zeros_like(z)
    direct.scatter_add_(1, classes.view(T, k)[:, ::2].long(), gt[0, :, ::2].double())
    want = direct - torch.softmax(z, -1) * gt[0].double().sum(-1, keepdim=True)
    assert float((room[1].double() - want).abs().max()) <= 2.0 ** -20 * float(gt.abs().sum(-1).max())
