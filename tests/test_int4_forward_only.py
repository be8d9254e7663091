"""Layers over 4-bit weights refuse the calls of training before they launch anything."""
import pytest
import torch


@pytest.fixture
def weight():
    from swiftrt_b200.int4 import Int4Weight
    w = object.__new__(Int4Weight)              # (one with tensors needs a device)
    w.shape = (8, 4)
    return w


def test_training_calls_are_refused(weight):
    import swiftrt_b200 as srt
    x, dy = torch.zeros(2, 8), torch.zeros(2, 4)
    dense = srt.Dense(weight, None, srt.ActivationType.relu)
    gated = srt.GatedDense(weight, weight)
    for call in (lambda: dense.forward_keep(x), lambda: dense.backward(x, dy, dy), lambda: gated.forward_keep(x), lambda: gated.backward(x, (dy, dy), dy)):
        with pytest.raises(ValueError, match="no backward pass"):
            call()
