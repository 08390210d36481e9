"""What the C ABI of the orthogonalised updates says about calls before anything is launched: matrices without values, and the size of its workspace."""
import ctypes
import os

import pytest

from tests.test_more_training_cpu import INVALID, Orth

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def sizes():
    import i6_native_ops_amd.training  # noqa: F401
    lib = ctypes.CDLL(os.path.join(ROOT, "i6_native_ops_amd", "training", "libi6train.so"))

    def call(*tensors, dtype=0):
        n = ctypes.c_size_t(7)
        return lib.i6orth_workspace_size((Orth * max(1, len(tensors)))(*tensors), len(tensors), dtype, ctypes.byref(n)), n.value
    return call


def matrix(rows, cols, momentum=None):
    return Orth(update=256 if rows * cols else None, result=256 if rows * cols else None, momentum=momentum, rows=rows, cols=cols)


@pytest.mark.parametrize("order", ["first", "middle", "last"])
def test_matrices_without_values_say_nothing_about_momenta(sizes, order):
    """A tensor without values has no address, so it looks like one without a momentum; wherever it stands, the others decide."""
    with_momenta, empty = [matrix(5, 9, 256), matrix(300, 200, 256)], matrix(0, 5)
    at = {"first": 0, "middle": 1, "last": 2}[order]
    rc, need = sizes(*with_momenta[:at], empty, *with_momenta[at:])
    assert rc == 0 and need == sizes(*with_momenta)[1]
    without = [matrix(5, 9), matrix(300, 200)]
    assert sizes(*without[:at], Orth(rows=0, cols=5, momentum=256), *without[at:])[0] == 0
    assert sizes(empty, matrix(5, 9), matrix(5, 9, 256))[0] == INVALID
