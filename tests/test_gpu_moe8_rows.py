"""The 8-bit expert layer (hecate_amd.moe8) on the GPU: rows that are not finite, and the whole numbers of the gated rows."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from hecate_amd import i8, moe8
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


def test_gated_rows_become_the_whole_numbers_of_the_mlp(dev):
    """gated values next to the borders between whole numbers, in the layer and in the gated MLP: half to even of the true quotient.
    x = (127, 64, 64, ..) has scale 1, so g = 64 / 2 = 32, silu(32) = 32 in fp32 (e^-32 < 2^-25), u = 64 su and h = 2048 su: any
    fp32 value. With wd the identity an output is its gated row's whole number times the row's scale"""
    H = I = 768
    x = torch.full((1, H), 64.0, dtype=BF, device=dev)
    x[0, 0] = 127.0
    one = torch.zeros((I, H), dtype=torch.int8, device=dev)
    one[:, 1] = 1
    eye = torch.eye(H, I, dtype=torch.int8, device=dev)
    sg, sd = torch.full((I,), 0.5, device=dev), torch.ones(H, device=dev)
    for top in (3.4150088, 1.8574041, 1.1617918):
        a = np.float32(top)
        near = ((np.arange(127) + 0.5) * float(a) / 127).astype(np.float32)
        h = np.concatenate([near, np.nextafter(near, np.float32(0)), np.nextafter(near, np.float32(9))])
        h = np.concatenate([[a], h, -h, np.zeros(I - 1 - 2 * h.size, np.float32)]).astype(np.float32)
        want = np.array([round(127 * Fraction(float(v)) / Fraction(float(a))) for v in h], dtype=np.float64)
        su = torch.from_numpy(h / np.float32(2048)).to(dev)
        y = torch.empty((1, H), device=dev)
        i8.mlp(x, one, one, eye, sg, su, sd, y, i8.mlp_work(dev, 1, H, I))
        s = float(a / np.float32(127))
        assert np.array_equal(np.rint(y[0].double().cpu().numpy() / s), want)
        # one expert, its weight 1: a / (a + 1e-20)
        sel, rw, out = torch.empty((1, 1), dtype=torch.int64, device=dev), torch.empty((1, 1), device=dev), torch.empty((1, H), device=dev)
        moe8.layer(x, torch.zeros((1, H), device=dev), None, one[None], one[None], eye[None], sg[None], su[None], sd[None], sel, rw, out,
                   moe8.layer_work(dev, 1, H, I, 1, 1), 1.0)
        assert float(rw) == 1.0
        got = np.rint(out[0].double().cpu().numpy() / s)
        assert np.array_equal(got, want), (int((got != want).sum()), "of", want.size)


def test_no_tokens(dev):
    """no tokens: nothing is launched, and no workspace is needed"""
    L = Layer(8, 8, 0, 64, 32, 2, True, 23, dev)
    out, sel, rw = L(torch.empty((0, 64), dtype=BF, device=dev), F32, work=L.work(4))
    assert out.shape == (0, 64) and sel.shape == (0, 2) and rw.shape == (0, 2)
    moe8.layer(out, L.wr.to(dev), None, *L.dw, *L.ds, sel, rw, torch.empty_like(out), None, 2.5)
