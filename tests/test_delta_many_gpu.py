"""The gated delta rule with so many heads that a workgroup has all of a head's more than 64 columns.  Every sequence of one head against the definition would take minutes on the host:
three of them, the longest among these, and all against calls with few heads, whose columns are two workgroups'."""
import pytest
import torch

from tests.test_delta_gpu import DTYPES, NAMES, check, expected, problem, run

pytestmark = pytest.mark.gpu


def some(p, sequences):
    return {n: x if x is None else x[sequences].contiguous() for n, x in p.items()}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,G,K,V", [(17, 70, 8, 8, 24, 72), (17, 70, 8, 4, 24, 128), (17, 70, 8, 8, 64, 72), (17, 131, 8, 2, 64, 128), (17, 70, 8, 8, 128, 72), (17, 70, 8, 8, 128, 128), (65, 20, 4, 2, 33, 100)])
def test_many_heads_of_more_than_64_columns(B, T, H, G, K, V, dtype):
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(K + V)).tolist()
    lens[0], lens[3], lens[5] = T, T - 1, 0
    p = problem(B, T, H, G, K, V, dtype, seed=K + V, lens=lens)
    got = run(p)
    chosen = [0, 3, B - 1]
    few = some(p, chosen)
    check(few, {n: x[chosen] for n, x in got.items()}, expected(few))
    for first in range(0, B, 4):
        part = list(range(first, min(B, first + 4)))
        again = run(some(p, part))
        assert all(torch.equal(again[n], got[n][part]) for n in got), first
    with torch.no_grad():
        from i6_native_ops_amd.training import gated_delta_rule
        o, last = gated_delta_rule(*(p[n] for n in NAMES[:5]), seq_lens=p["lens"], initial_state=p["initial"])
    assert torch.equal(o, got["o"]) and torch.equal(last, got["last"])
