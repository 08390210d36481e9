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


def test_workspace_is_that_of_the_matrices_at_work(sizes):
    """Three times the matrix (as it is and twice turned) and two square ones, 4 bytes a value each, sides rounded up to 64: for the matrices of one launch, not for all of the call."""
    def own(rows, cols):
        up = lambda n: (n + 63) // 64 * 64  # noqa: E731
        n, m = min(rows, cols), max(rows, cols)
        return 4 * (n * up(m) + 2 * m * up(n) + 2 * n * up(n)) + 8 * 256 + 8 * 256     # and sums; each part rounded up to 256 bytes

    shared = 64 << 20
    for rows, cols in [(4096, 11008), (300, 200), (2048, 1024)]:
        one = sizes(matrix(rows, cols))[1]
        assert 0.99 * own(rows, cols) <= one <= own(rows, cols) + shared
        for count in (2, 34, 35, 200):
            need = sizes(*[matrix(rows, cols)] * count)[1]
            at_work = min(count, 34, max(1, (4 << 30) // own(rows, cols)))
            assert 0.99 * at_work * own(rows, cols) <= need <= at_work * own(rows, cols) + shared, (rows, cols, count)
    # matrices that a workgroup does alone need none but where they go the others' way, without iterations
    assert sizes(*[matrix(64, 64)] * 1000)[1] <= 34 * own(64, 64) + shared
    assert sizes(*[matrix(64, 64)] * 1000)[1] == sizes(*[matrix(64, 64)] * 34)[1]
    # one larger than 4 GB is worked on alone
    assert sizes(matrix(20000, 20000), matrix(20000, 20000), matrix(5, 5))[1] <= own(20000, 20000) + shared
