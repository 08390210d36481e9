"""CPU-side checks of the operators around the losses: the library exports what its header declares, refuses bad
arguments before anything is launched, and its kernels keep to their registers."""
import ctypes
import json
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "i6_native_ops_amd", "training", "libi6train.so")


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "i6train.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(i6train_\w+)\s*\(", text))
    import i6_native_ops_amd.training  # noqa: F401
    lib = ctypes.CDLL(LIB)
    assert len(names) == 10
    for n in names:
        assert getattr(lib, n) is not None


def test_header_and_python_agree():
    from i6_native_ops_amd import training
    text = open(os.path.join(ROOT, "include", "i6train.h")).read()
    assert int(re.search(r"#define I6TRAIN_BLOCK (\d+)", text).group(1)) == training.BLOCK


def test_null_arguments_are_refused_on_the_host():
    import i6_native_ops_amd.training  # noqa: F401
    lib = ctypes.CDLL(LIB)
    lib.i6train_strerror.restype = ctypes.c_char_p
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.i6train_ce_workspace_size(None, ctypes.byref(a), ctypes.byref(b)) == -1
    assert lib.i6train_ce_forward(None, None, None, ctypes.c_size_t(0), None) == -1
    assert lib.i6train_rec_workspace_size(None, ctypes.byref(a)) == -1
    assert lib.i6train_rec_states_size(None, ctypes.byref(a)) == -1
    zero = [ctypes.c_double(x) for x in (1e-3, 0.9, 0.999, 1e-8, 0.0)]
    assert lib.i6train_adamw(None, 1, 0, 32, ctypes.c_int64(1), *zero, None) == -1
    assert lib.i6train_adamw(None, 0, 0, 16, ctypes.c_int64(1), *zero, None) == -1
    assert lib.i6train_adamw(None, 0, 0, 32, ctypes.c_int64(1), *zero, None) == 0       # no tensors: nothing to do
    assert b"invalid" in lib.i6train_strerror(-1)
    assert len({lib.i6train_strerror(c) for c in (0, -1, -2, -3, -4, -11, -99)}) == 7


def test_cpu_tensors_are_refused():
    from i6_native_ops_amd.training import adamw_step, gated_recurrence, linear_cross_entropy
    x = torch.zeros(2, 3, 4)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="hidden must be a CUDA tensor"):
        linear_cross_entropy(x, torch.zeros(5, 4), torch.zeros(2, 3, dtype=torch.int32), i)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        gated_recurrence(x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        adamw_step([x], [x], [x], [x], step=1, lr=1e-3)
    adamw_step([], [], [], [], step=1, lr=1e-3)


def test_kernels_keep_to_their_registers():
    from i6_native_ops_amd import build
    res = json.load(open(os.path.join(os.path.dirname(LIB), "kernel_resources.json")))
    assert res.get("_sources_sha256") == build.sources_digest(build.TRAINING), "rebuild (python -m i6_native_ops_amd.build)"
    kernels = {k: v for k, v in res.items() if k != "_sources_sha256"}
    assert any("adamw_step" in k for k in kernels) and any("rec_forward" in k for k in kernels)
    for name, r in kernels.items():
        if "adamw_step" in name:
            assert r["scratch"] == 0 and r["occupancy"] == 8, (name, r)      # bound by memory: all the waves there is room for
        else:
            assert r["scratch"] == 0, (name, r)
