"""The 8-bit expert layer (hecate_amd.moe8) on the GPU: rows that are not finite."""
import pytest
import torch

from test_gpu_moe8 import BF, F16, F32, Layer, log, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 6, 16])
@pytest.mark.parametrize("n", [0, 9])
def test_rows_that_are_not_finite_without_a_resident_pick(dev, T, n):
    """a row with a NaN picks the lowest ids; where none of them is resident (and there is no shared expert) its output is NaN all the
    same, and the rows beside it are what they are without it"""
    log("not finite, nothing resident", T, n)
    L = Layer(30, n, 12, 256, 128, 4, False, 21, dev)
    x = rows(T, 256, BF, 5, dev).clone()
    bad = sorted({0, T // 2, T - 1})
    want = L(x, F32)[0]
    for k, r in enumerate(bad):
        x[r, 7 * k] = (float("nan"), float("inf"), -float("inf"))[k]
    for odt in (F32, BF, F16):
        out, sel, _ = L(x, odt)
        assert sel[0].tolist() == [0, 1, 2, 3]
        o = out.cpu()
        assert bool(o[bad].isnan().all())
        keep = [r for r in range(T) if r not in bad]
        assert torch.equal(o[keep], want.cpu()[keep].to(odt))
