"""AdamW: values that are no numbers beside others."""
import pytest
import torch

from tests.test_training_gpu import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e25])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_bad_gradient_in_8_bits_spoils_one_value(dtype, bad):
    """The other values of its block go on as they would without it; the bad one stays no number (1e25: its square is infinite)."""
    from i6_native_ops_amd.training import adamw_step
    g = gen(12)
    n, at = 1000, 300
    start = torch.randn(n, generator=g, device="cuda").to(dtype)
    runs = []
    for value in (bad, 0.0):
        p = start.clone()
        m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        scales = (torch.ones(4, device="cuda"), torch.ones(4, device="cuda"))
        h = gen(13)
        for step in range(1, 6):
            grad = torch.randn(n, generator=h, device="cuda").to(dtype)
            grad[at] = value if step == 2 else 0.0
            adamw_step([p], [grad], [m], [v], step=step, lr=1e-2, scales=[scales])
        runs.append((p, m.float(), v.float(), *scales))
    places = torch.arange(n, device="cuda")
    for i in range(3):
        # a first moment of 1e24 is a number, and the largest of its block: what is small beside it is 0 there, as anywhere
        others = places // 256 != at // 256 if bad == 1e25 and i < 2 else places != at
        a, b = runs[0][i], runs[1][i]
        assert torch.isfinite(a[others]).all() and torch.equal(a[others], b[others]), i
    assert torch.isnan(runs[0][2][at])
    if bad != 1e25:
        assert torch.isnan(runs[0][0][at]) and torch.isnan(runs[0][1][at])
        assert torch.equal(runs[0][3], runs[1][3])
    assert torch.equal(runs[0][4], runs[1][4])


def test_optimiser_steps_are_not_captured(monkeypatch):
    """A replay would repeat the number of the captured step, and with it its corrections and roundings."""
    from i6_native_ops_amd.training import AdamW
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = AdamW([p], lr=1e-2)
    p.grad = torch.ones_like(p)
    opt.step()
    held = p.detach().clone()
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="AdamW.step cannot be captured"):
            opt.step()
    assert opt.state[p]["step"] == 1 and torch.equal(p.detach(), held)
    opt.step()
    assert opt.state[p]["step"] == 2


def test_steps_that_fail_are_not_counted():
    from i6_native_ops_amd.training import AdamW
    p = torch.nn.Parameter(torch.ones(4, 6, device="cuda"))
    q = torch.nn.Parameter(torch.ones(4, 6, device="cuda").T)          # not contiguous: refused
    opt = AdamW([p, q], lr=1e-2)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.step()
    assert opt.state[p].get("step", 0) == 0
    q.grad = None
    opt.step()
    assert opt.state[p]["step"] == 1
