"""Sizes past 32 bits are refused before they reach the C entries, whose sizes are 32-bit; without a GPU."""
import pytest
import torch

from hecate_amd import i8, moe8


@pytest.mark.parametrize("shape", [((1 << 32) + 4, 16), (4, (1 << 32) + 16), (1 << 31, 16)])
def test_a_matrix_of_more_than_31_bits(shape):
    with pytest.raises(RuntimeError, match="2147483647"):
        i8._two("x", torch.empty(shape, device="meta"))
    assert tuple(i8._two("x", torch.empty(((1 << 31) - 1, 16), device="meta"))) == ((1 << 31) - 1, 16)


def test_workspaces():
    big = 1 << 32
    for f in (lambda: i8.linear_work("cpu", big + 4, 16, 64), lambda: i8.linear_work("cpu", 4, 16, big + 64),
              lambda: i8.mlp_work("cpu", big + 4, 64, 32), lambda: i8.mlp_work("cpu", 4, big + 64, 32),
              lambda: moe8.layer_work("cpu", big + 4, 64, 32, 8, 2), lambda: moe8.layer_work("cpu", 4, 64, 32, 8, big + 2)):
        with pytest.raises(RuntimeError):
            f()
