"""CPU-side checks of the second set of operators around the losses: exported symbols, refusals before anything is launched, sizes that are too large."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, TOO_SMALL, TOO_LARGE = -1, -2, -4
P, N = ctypes.c_void_p, ctypes.c_int64


class Logp(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("B", "T", "F", "k", "dtype")] + [("logits", P), ("l_b", N), ("l_t", N), ("targets", P), ("t_b", N), ("t_t", N), ("lens", P)]


class Delta(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("B", "T", "H", "G", "K", "V", "dtype")] + [
        f for x in ("q", "k", "v", "gate", "beta") for f in ((x, P), (x + "_b", N), (x + "_t", N), (x + "_h", N))] + [("lens", P), ("initial", P)]


class Orth(ctypes.Structure):
    _fields_ = [("update", P), ("result", P), ("momentum", P), ("rows", ctypes.c_int), ("cols", ctypes.c_int), ("keep", ctypes.c_float), ("rate", ctypes.c_float)]


@pytest.fixture(scope="module")
def lib():
    import i6_native_ops_amd.training  # noqa: F401
    return ctypes.CDLL(os.path.join(ROOT, "i6_native_ops_amd", "training", "libi6train.so"))


@pytest.mark.parametrize("header,count", [("i6logp.h", 2), ("i6delta.h", 3), ("i6orth.h", 2)])
def test_library_exports_every_declared_symbol(lib, header, count):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
    names = set(re.findall(r"\b(%s_\w+)\s*\(" % header[:-2], text))
    assert len(names) == count
    for n in names:
        assert getattr(lib, n) is not None


def logp(**more):
    return Logp(**{**dict(B=2, T=3, F=10, k=2, dtype=0, logits=256, targets=256, lens=256, l_b=30, l_t=10, t_b=3, t_t=1), **more})


def test_logp_refusals(lib):
    def forward(p, *out):
        return lib.i6logp_forward(ctypes.byref(p) if p else None, *out, None)
    outs = [P(256)] * 5
    assert forward(None, *outs) == INVALID
    for bad in (dict(B=0), dict(T=-1), dict(F=0), dict(k=-1), dict(k=11), dict(F=100, k=65), dict(dtype=2), dict(logits=None), dict(targets=None), dict(lens=None)):
        assert forward(logp(**bad), *outs) == INVALID, bad
    assert forward(logp(), None, P(256), P(256), P(256), None) == INVALID
    assert forward(logp(), P(256), P(256), None, P(256), None) == INVALID
    assert forward(logp(F=(1 << 28) + 1), *outs) == TOO_LARGE
    assert forward(logp(B=1 << 11, T=1 << 11, F=513), *outs) == TOO_LARGE
    assert forward(logp(B=1 << 13, T=1 << 13, F=512), *outs) == TOO_LARGE
    assert lib.i6logp_backward(ctypes.byref(logp()), None, P(256), None, None, None, P(256), None) == INVALID
    assert lib.i6logp_backward(ctypes.byref(logp()), P(256), None, None, None, None, P(256), None) == INVALID


def delta(**more):
    return Delta(**{**dict(B=2, T=100, H=4, G=2, K=64, V=64, dtype=1, q=256, k=256, v=256, gate=256, beta=256), **more})


def delta_sizes(lib, p, train=1):
    n = [ctypes.c_size_t() for _ in range(3)]
    return lib.i6delta_sizes(ctypes.byref(p) if p else None, train, *(ctypes.byref(x) for x in n)), [x.value for x in n]


def test_delta_refusals(lib):
    assert delta_sizes(lib, None)[0] == INVALID
    for bad in (dict(B=0), dict(T=0), dict(H=0), dict(G=3), dict(K=0), dict(V=0), dict(dtype=7), dict(q=None), dict(beta=None)):
        assert delta_sizes(lib, delta(**bad))[0] == INVALID, bad
    for bad in (dict(B=65536), dict(K=129), dict(V=129), dict(H=65536, G=1), dict(T=(1 << 28) + 1), dict(B=1, T=(1 << 28), H=2), dict(B=1, H=1, G=1, T=(1 << 28) + 1), dict(B=65535, H=65535, G=1, T=1), dict(B=1, T=1 << 30, H=2)):
        assert delta_sizes(lib, delta(**bad))[0] == TOO_LARGE, bad
    assert delta_sizes(lib, delta(B=1, H=1, G=1, T=1 << 28))[0] == 0
    rc, (kept, forward, backward) = delta_sizes(lib, delta())
    assert rc == 0 and kept > 0 and backward > 0
    assert delta_sizes(lib, delta(), 0)[1][0] == 0
    p, at, size = delta(), P(256), ctypes.c_size_t
    assert lib.i6delta_forward(ctypes.byref(p), None, at, None, size(0), None, size(0), None) == INVALID
    assert lib.i6delta_forward(ctypes.byref(p), at, at, at, size(kept - 1), at, size(1 << 40), None) == TOO_SMALL
    back = [at, N(0), N(0), N(0), at, at, size(kept), at, at, at, at, at, at, at, size(backward - 1), None]
    assert lib.i6delta_backward(ctypes.byref(p), *back) == TOO_SMALL
    back[14], back[7] = size(backward), None
    assert lib.i6delta_backward(ctypes.byref(p), *back) == INVALID


def test_orth_refusals(lib):
    def sizes(*tensors, dtype=0):
        n = ctypes.c_size_t(7)
        table = (Orth * max(1, len(tensors)))(*tensors)
        return lib.i6orth_workspace_size(table, len(tensors), dtype, ctypes.byref(n)), n.value
    good = dict(update=256, result=256, rows=5, cols=9)
    assert sizes() == (0, 0)
    assert sizes(Orth(**good))[0] == 0
    assert sizes(Orth(**{**good, "rows": 0, "update": None})) == (0, 0)
    assert sizes(Orth(**{**good, "rows": -1}))[0] == INVALID
    assert sizes(Orth(**{**good, "result": None}))[0] == INVALID
    assert sizes(Orth(**good), Orth(**{**good, "momentum": 256}))[0] == INVALID
    assert sizes(Orth(**{**good, "cols": 32769}))[0] == TOO_LARGE
    assert sizes(Orth(**good), dtype=3)[0] == INVALID
    assert lib.i6orth_workspace_size(None, 1, 0, ctypes.byref(ctypes.c_size_t())) == INVALID
    rc, need = sizes(Orth(**good))
    t = Orth(**good)
    step = lambda n, mu, bytes: lib.i6orth_step(ctypes.byref(t), 1, 0, n, ctypes.c_double(mu), 0, P(256), ctypes.c_size_t(bytes), None)  # noqa: E731
    assert step(-1, 0.9, need) == INVALID and step(5, 1.0, need) == INVALID and step(5, 0.9, need - 1) == TOO_SMALL


def test_cpu_tensors_are_refused():
    from i6_native_ops_amd.training import Muon, gated_delta_rule, muon_step, orthogonalize, target_log_probs
    x = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        target_log_probs(x, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        gated_delta_rule(x[..., None], x[..., None], x[..., None], x, x)
    with pytest.raises(RuntimeError, match="contiguous CUDA matrix"):
        orthogonalize([x[0]])
    with pytest.raises(RuntimeError, match="contiguous CUDA matrix"):
        muon_step([x[0]], [x[0]], [x[0]], lr=0.1)
    assert orthogonalize([]) == []
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(x)])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(x[0])], adjust_lr="none")
