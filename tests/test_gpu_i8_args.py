"""The 8-bit operators' Python entries on the GPU: every argument that is not what it should be raises RuntimeError, and nothing is
written."""
import pytest
import torch

from hecate_amd import i8, moe8

pytestmark = pytest.mark.gpu


def calls(dev):
    """(entry, its arguments, those that may be None)"""
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=dev)
    b, i = torch.int8, torch.int64
    T, H, I, E, N = 2, 64, 32, 4, 16
    x, work = z(T, H, dt=torch.bfloat16), z(1 << 20, dt=torch.uint8)
    w = (z(I, H, dt=b), z(I, H, dt=b), z(H, I, dt=b), z(I), z(I), z(H))
    we = tuple(torch.stack([t] * E) for t in w)
    return {
        "quantize": (i8.quantize, [x, z(T, H, dt=b), z(T)], ()),
        "matmul": (i8.matmul, [z(T, H, dt=b), z(T), z(N, H, dt=b), z(N), z(T, N), z(N)], (5,)),
        "linear": (i8.linear, [x, z(N, H, dt=b), z(N), z(T, N), work, z(N)], (5,)),
        "mlp": (i8.mlp, [x, *w, z(T, H), work], ()),
        "layer": (moe8.layer, [x, z(E, H), z(E), *we, z(T, 2, dt=i), z(T, 2), z(T, H), work, 2.5, 0, w], (2, 15)),
    }


@pytest.mark.parametrize("name", ["quantize", "matmul", "linear", "mlp", "layer"])
def test_arguments_left_out(dev, name):
    f, args, optional = calls(dev)[name]
    f(*args)
    for k, a in enumerate(args):
        if k in optional:
            f(*args[:k], None, *args[k + 1:])
        elif isinstance(a, torch.Tensor):
            for other in (None, 3, [a]):
                with pytest.raises(RuntimeError):
                    f(*args[:k], other, *args[k + 1:])
            with pytest.raises(RuntimeError, match="device"):
                f(*args[:k], a.cpu(), *args[k + 1:])
    torch.cuda.synchronize()


def test_shared_experts_of_another_number_of_tensors(dev):
    f, args, _ = calls(dev)["layer"]
    w = args[15]
    for bad in ((), w[:3], w[:4], w[:5], w + (w[5],), w[0], w[:5] + (None,)):
        with pytest.raises(RuntimeError):
            f(*args[:15], bad)
    f(*args[:15], list(w))
    torch.cuda.synchronize()


@pytest.mark.parametrize("lo", [1 << 32, -(1 << 32), (1 << 32) + 1, 1, -1])
def test_first_resident_expert(dev, lo):
    """lo is what it is, not its low 32 bits"""
    f, args, _ = calls(dev)["layer"]
    with pytest.raises(RuntimeError):
        f(*args[:14], lo, args[15])
    torch.cuda.synchronize()
