"""Sizes that no launch takes are refused by name, before anything is launched."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOO_LARGE = -4


class CeProblem(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int), ("T", ctypes.c_int), ("F", ctypes.c_int), ("D", ctypes.c_int), ("dtype", ctypes.c_int),
                ("hidden", ctypes.c_void_p), ("hidden_stride_b", ctypes.c_int64), ("hidden_stride_t", ctypes.c_int64),
                ("weight", ctypes.c_void_p), ("weight_stride_f", ctypes.c_int64), ("bias", ctypes.c_void_p),
                ("targets", ctypes.c_void_p), ("targets_stride_b", ctypes.c_int64), ("targets_stride_t", ctypes.c_int64),
                ("seq_lens", ctypes.c_void_p)]


class RecProblem(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int), ("T", ctypes.c_int), ("D", ctypes.c_int), ("dtype", ctypes.c_int),
                ("x", ctypes.c_void_p), ("x_stride_b", ctypes.c_int64), ("x_stride_t", ctypes.c_int64),
                ("gate", ctypes.c_void_p), ("gate_stride_b", ctypes.c_int64), ("gate_stride_t", ctypes.c_int64),
                ("seq_lens", ctypes.c_void_p), ("initial", ctypes.c_void_p)]


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")] + [("n", ctypes.c_int64)]


@pytest.fixture(scope="module")
def lib():
    import i6_native_ops_amd.training  # noqa: F401
    return ctypes.CDLL(os.path.join(ROOT, "i6_native_ops_amd", "training", "libi6train.so"))


def ce_sizes(lib, B, T, F, D, dtype):
    p = CeProblem(B=B, T=T, F=F, D=D, dtype=dtype, hidden=256, weight=256, targets=256, seq_lens=256, hidden_stride_b=T * D, hidden_stride_t=D,
                  weight_stride_f=D, targets_stride_b=T, targets_stride_t=1)
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    return lib.i6train_ce_workspace_size(ctypes.byref(p), ctypes.byref(a), ctypes.byref(b))


@pytest.mark.parametrize("dtype", [0, 1])
def test_cross_entropy_limits(lib, dtype):
    assert ce_sizes(lib, 32, 1000, 12001, 512, dtype) == 0
    assert ce_sizes(lib, 1, 1 << 22, 12001, 64, dtype) == 0                 # 47 x 32768 tiles
    assert ce_sizes(lib, 1 << 12, 1 << 10, 1 << 18, 64, dtype) == TOO_LARGE  # 2^25 tiles of 256 threads: more than 2^32 threads
    assert ce_sizes(lib, 1 << 12, 1 << 10, 1 << 22, 64, dtype) == TOO_LARGE
    assert ce_sizes(lib, 1, (1 << 22) + 1, 100, 64, dtype) == TOO_LARGE
    assert ce_sizes(lib, 1, 600, 1 << 22, 64, dtype) == 0


def test_recurrence_limits(lib):
    def states(B, T, D):
        p = RecProblem(B=B, T=T, D=D, dtype=0, x=256, gate=256, x_stride_b=T * D, x_stride_t=D, gate_stride_b=T * D, gate_stride_t=D)
        n = ctypes.c_size_t()
        return lib.i6train_rec_workspace_size(ctypes.byref(p), ctypes.byref(n))
    assert states(65535, 1, 1024) == 0 and states(1, 1 << 30, 1) == 0 and states(1, 1, 1 << 28) == 0
    assert states(1, 1, 1 << 29) == TOO_LARGE                               # 2^23 workgroups of 512 threads


def test_adamw_limits(lib):
    t = Tensor(*[256] * 6, n=(1 << 36) + 1)
    numbers = [ctypes.c_double(x) for x in (1e-3, 0.9, 0.999, 1e-8, 0.0)]
    assert lib.i6train_adamw(ctypes.byref(t), 1, 0, 32, ctypes.c_int64(1), *numbers, None) == TOO_LARGE
