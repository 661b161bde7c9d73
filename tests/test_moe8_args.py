"""The 8-bit expert layer's Python entry without a GPU: a shared expert is six tensors."""
import pytest
import torch

from hecate_amd import moe8


@pytest.mark.parametrize("count", [0, 3, 4, 5, 7])
def test_shared_expert_of_another_number_of_tensors(count):
    z = torch.zeros
    x, wr = z((2, 64)), z((4, 64))
    w, d, s, sd = z((4, 32, 64), dtype=torch.int8), z((4, 64, 32), dtype=torch.int8), z((4, 32)), z((4, 64))
    with pytest.raises(RuntimeError, match="six tensors"):
        moe8.layer(x, wr, None, w, w, d, s, s, sd, z((2, 2), dtype=torch.int64), z((2, 2)), z((2, 64)), z(8, dtype=torch.uint8), 2.5, 0,
                   (w[0],) * count)
