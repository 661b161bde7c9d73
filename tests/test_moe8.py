"""The 8-bit expert layer's checks of arguments, without a GPU (the addresses below are never read)."""
import ctypes

import pytest
import torch

from hecate_amd import _lib, moe8

A = 1 << 20


def test_layer_refuses():
    L = _lib.lib()
    P3 = ctypes.c_void_p * 3
    good = dict(x=A, xdt=1, ldx=64, T=4, wr=2 * A, bias=None, E=16, topk=2, scale=2.5, wg=3 * A, wu=4 * A, wd=5 * A, sg=6 * A, su=7 * A,
                sd=8 * A, n=16, lo=0, H=64, I=32, shw=None, shs=None, sel=9 * A, rw=10 * A, y=11 * A, ydt=1, ldy=64, work=12 * A, st=None)

    def refused(word, **k):
        assert L.hmoe_moe8_layer(*{**good, **k}.values()) == 1 and word.encode() in L.hmoe_last_error(), L.hmoe_last_error()

    refused("tokens", T=17)
    refused("tokens", T=-1)
    refused("hidden size", H=72)
    refused("hidden size", H=7184, ldx=7184, ldy=7184)
    refused("hidden size", I=8)
    refused("hidden size", I=0)
    refused("hidden size", I=4112)
    refused("experts", E=513)
    refused("experts", topk=17)
    refused("experts", topk=0)
    refused("experts", E=1, n=1)
    refused("resident", lo=1)
    refused("resident", lo=-1)
    refused("resident", n=-1)
    refused("resident", n=17)
    refused("dtype", xdt=3)
    refused("dtype", ydt=-1)
    refused("row stride", x=None)
    refused("row stride", x=A + 1)
    refused("row stride", ldx=63)
    refused("row stride", ldy=63)
    refused("row stride", y=11 * A + 1)
    refused("router", wr=None)
    refused("router", wr=2 * A + 4)
    refused("router", bias=A + 2)
    refused("expert weights", wu=None)
    refused("expert weights", wd=5 * A + 8)
    refused("expert weights", sd=8 * A + 2)
    refused("shared", shw=P3(A, A, A))
    refused("shared", shw=P3(A, A, 0), shs=P3(A, A, A))
    refused("shared", shw=P3(A, A, A), shs=P3(A, A, A + 2))
    refused("sel", sel=None)
    refused("sel", work=None)
    refused("sel", work=12 * A + 64)
    refused("overlaps", y=A + 128)
    assert L.hmoe_moe8_layer(*{**good, "T": 0, "x": None}.values()) == 0
    assert L.hmoe_moe8_work_bytes(17, 64, 32, 16, 2) == 0 and L.hmoe_moe8_work_bytes(16, 64, 32, 16, 2) > 0
    assert all(L.hmoe_moe8_work_bytes(t, 64, 32, 16, 2) <= L.hmoe_moe8_work_bytes(t + 1, 64, 32, 16, 2) for t in range(1, 16))


def test_python_entry_refuses():
    z = torch.zeros
    x, wr = z((2, 64)), z((4, 64))
    w, d, s, sd = z((4, 32, 64), dtype=torch.int8), z((4, 64, 32), dtype=torch.int8), z((4, 32)), z((4, 64))
    with pytest.raises(RuntimeError, match="device"):
        moe8.layer(x, wr, None, w, w, d, s, s, sd, z((2, 2), dtype=torch.int64), z((2, 2)), z((2, 64)), z(8, dtype=torch.uint8), 2.5)
    with pytest.raises(RuntimeError, match="not a layer"):
        moe8.layer_work("cpu", 17, 64, 32, 4, 2)
    with pytest.raises(RuntimeError, match="contiguous"):
        moe8._w("wg", w.transpose(1, 2), (4, 64, 32), torch.int8)
