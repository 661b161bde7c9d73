"""The 8-bit operators' Python entries without a GPU: arguments that are not tensors on the GPU."""
import pytest
import torch

from hecate_amd import i8


class OnGpu:
    """what the entries ask a tensor for its place"""
    is_cuda = True

    def __init__(self, i=0):
        self.device = torch.device("cuda", i)

    def get_device(self):
        return self.device.index


def test_every_argument_is_a_tensor_on_the_same_gpu():
    x = OnGpu()
    i8._on("f", x, OnGpu(), OnGpu())
    for other in (None, 3, [x], OnGpu(1), torch.zeros(2)):
        with pytest.raises(RuntimeError, match="f: "):
            i8._on("f", x, OnGpu(), other)
        if not isinstance(other, OnGpu):
            with pytest.raises(RuntimeError, match="f: "):
                i8._on("f", other, x)
