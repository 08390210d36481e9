"""The losses, the alignment and the operators around them in one small model."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state_bits", [8, 32])
def test_example_trains_aligns_and_streams(state_bits):
    from i6_native_ops_amd.training import example
    seen = example.train(steps=30, state_bits=state_bits)
    assert seen["full_sum"][-1] < 0.7 * seen["full_sum"][0]
    assert seen["cross_entropy"][-1] < 0.7 * seen["cross_entropy"][0]
    assert seen["aligned_right"] > 0.5 and seen["right"] > seen["right_after_full_sum"] - 0.05
    assert seen["streamed_differs"] < 1e-4
