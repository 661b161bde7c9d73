"""The 8-bit integer operators' checks of arguments, without a GPU: the C entries and the Python ones refuse before any
launch (the addresses below are never read)."""
import pytest
import torch

from hecate_amd import _lib, i8

A = 1 << 20
F32, BF16, F16 = 0, 1, 2


def refused(rc, word):
    assert rc == 1 and word.encode() in _lib.lib().hmoe_last_error(), (rc, _lib.lib().hmoe_last_error())


def test_quantize_refuses():
    f = _lib.lib().hmoe_i8_quantize
    good = dict(x=A, dt=BF16, ldx=64, M=4, K=64, q=2 * A, ldq=64, s=3 * A, st=None)
    bad = lambda **k: f(*{**good, **k}.values())
    refused(bad(dt=5), "dtype")
    refused(bad(K=24), "depth")
    refused(bad(K=0), "depth")
    refused(bad(K=131072, ldx=131072, ldq=131072), "depth")
    refused(bad(M=-1), "rows")
    refused(bad(M=(1 << 20) + 1), "rows")
    refused(bad(x=None), "x address")
    refused(bad(x=A + 1), "x address")
    refused(bad(dt=F32, x=A + 2), "x address")
    refused(bad(ldx=63), "row stride")
    refused(bad(ldx=1 << 62), "row stride")
    refused(bad(q=None), "q:")
    refused(bad(q=A + 8), "q:")
    refused(bad(ldq=72), "q:")
    refused(bad(s=None), "q:")
    refused(bad(q=A + 256), "overlaps")
    assert bad(M=0, x=None, q=None) == 0


def test_matmul_refuses():
    f = _lib.lib().hmoe_i8_matmul
    good = dict(q=A, ldq=64, s=2 * A, M=4, w=3 * A, ldw=64, ws=4 * A, N=8, K=64, bias=None, y=5 * A, dt=F32, ldy=8, st=None)
    bad = lambda **k: f(*{**good, **k}.values())
    refused(bad(K=40), "depth")
    refused(bad(M=-2), "rows")
    refused(bad(N=0), "output channels")
    refused(bad(q=A + 4), "q:")
    refused(bad(ldq=65), "q:")
    refused(bad(ldq=1 << 28), "q:")
    refused(bad(ldw=1 << 28), "weights")
    refused(bad(w=None), "weights")
    refused(bad(w=3 * A + 8), "weights")
    refused(bad(ldw=48), "weights")
    refused(bad(ws=None), "weights")
    refused(bad(bias=A + 2), "bias")
    refused(bad(dt=3), "dtype")
    refused(bad(y=None), "output")
    refused(bad(y=5 * A + 2), "output")
    refused(bad(ldy=7), "output")
    refused(bad(y=A + 64), "overlaps")
    assert bad(M=0, q=None, y=None) == 0


def test_linear_and_mlp_refuse():
    L = _lib.lib()
    good = dict(x=A, dt=F16, ldx=64, M=4, w=3 * A, ldw=64, ws=4 * A, N=8, K=64, bias=None, y=5 * A, ydt=F32, ldy=8, work=6 * A, st=None)
    bad = lambda **k: L.hmoe_i8_linear(*{**good, **k}.values())
    refused(bad(K=8), "depth")
    refused(bad(work=None), "workspace")
    refused(bad(work=6 * A + 8), "workspace")
    refused(bad(y=A), "overlaps")
    refused(bad(dt=-1), "dtype")
    refused(bad(ldw=60), "weights")
    good2 = dict(x=A, dt=F16, ldx=64, M=4, H=64, I=32, wg=2 * A, wu=3 * A, wd=4 * A, sg=5 * A, su=6 * A, sd=7 * A, y=8 * A, ydt=F32, ldy=64,
                 work=9 * A, st=None)
    bad = lambda **k: L.hmoe_i8_mlp(*{**good2, **k}.values())
    refused(bad(H=72, ldx=72), "depth")
    refused(bad(I=40), "intermediate")
    refused(bad(I=0), "intermediate")
    refused(bad(wu=None), "weights")
    refused(bad(sd=None), "weights")
    refused(bad(work=None), "workspace")
    refused(bad(y=A + 2, ydt=BF16), "overlaps")
    refused(bad(ldy=63), "output")
    assert bad(M=0, x=None) == 0
    assert L.hmoe_i8_linear_work_bytes(0, 8, 64) == 0 and L.hmoe_i8_linear_work_bytes(3, 8, 64) >= 3 * 64 + 12
    assert L.hmoe_i8_mlp_work_bytes(5, 64, 32) >= 5 * (64 + 4 + 32 * 5 + 4)


def test_python_entries_refuse_host_tensors():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    w, s = torch.zeros((8, 64), dtype=torch.int8), torch.zeros(8)
    out, work = torch.zeros((2, 8)), torch.zeros(4096, dtype=torch.uint8)
    for f in (lambda: i8.quantize(x, torch.zeros((2, 64), dtype=torch.int8), torch.zeros(2)),
              lambda: i8.linear(x, w, s, out, work),
              lambda: i8.matmul(torch.zeros((2, 64), dtype=torch.int8), torch.zeros(2), w, s, out),
              lambda: i8.mlp(x, w, w, w, s, s, s, out, work)):
        with pytest.raises(RuntimeError, match="device"):
            f()


def test_python_checks_shapes_and_types():
    x = torch.zeros((4, 64))
    with pytest.raises(RuntimeError, match="contiguous rows"):
        i8._rows("x", x.t(), 64, 4)
    with pytest.raises(RuntimeError, match="overlap"):
        i8._rows("x", x[:1].expand(4, 64), 4, 64)
    with pytest.raises(RuntimeError, match="must be"):
        i8._rows("x", x, 4, 63)
    with pytest.raises(RuntimeError, match="must be"):
        i8._rows("q", x, 4, 64, torch.int8)
    assert i8._rows("x", torch.zeros((4, 80))[:, :64], 4, 64) == 80
    assert i8._rows("x", x[:1], 1, 64) == 64
    with pytest.raises(RuntimeError, match="fp32"):
        i8._vec("s", torch.zeros(4, dtype=torch.float16), 4)
    with pytest.raises(RuntimeError, match="int8"):
        i8._mat("w", torch.zeros((8, 64)), 8, 64)
    with pytest.raises(RuntimeError, match="int8"):
        i8._mat("w", torch.zeros((8, 128), dtype=torch.int8)[:, :64], 8, 64)
    with pytest.raises(RuntimeError, match="workspace"):
        i8._work("linear", torch.zeros(16, dtype=torch.uint8), 17)
