"""x and the output as column ranges of one buffer (they share no byte): the 8-bit operators give what they give apart."""
import pytest
import torch

from hecate_amd import i8, moe8
from test_gpu_i8 import BF, F16, F32, log, rows, weight
from test_gpu_moe8 import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [2, 16, 40, 300])
@pytest.mark.parametrize("first", [True, False])
def test_products(dev, M, first):
    """M rows of x beside their outputs, x first or behind them"""
    log("columns", M, first)
    K, N, I = 272, 144, 80
    x = rows(M, K, BF, M)
    w, ws = weight(N, K, 1)
    work = i8.linear_work(dev, M, N, K)
    want = i8.linear(x, w, ws, torch.empty((M, N), dtype=BF, device=dev), work).clone()
    buf = torch.zeros((M, K + N), dtype=BF, device=dev)
    xb, yb = (buf[:, :K], buf[:, K:]) if first else (buf[:, N:], buf[:, :N])
    xb.copy_(x)
    i8.linear(xb, w, ws, yb, work)
    assert torch.equal(yb, want) and torch.equal(xb, x)

    (wg, sg), (wu, su), (wd, sd) = weight(I, K, 1), weight(I, K, 2), weight(K, I, 3)
    mw = i8.mlp_work(dev, M, K, I)
    want = i8.mlp(x, wg, wu, wd, sg, su, sd, torch.empty((M, K), dtype=F16, device=dev), mw).clone()
    buf = torch.zeros((M, 2 * K), dtype=BF, device=dev)
    xb, yb = (buf[:, :K], buf[:, K:].view(F16)) if first else (buf[:, K:], buf[:, :K].view(F16))
    xb.copy_(x)
    i8.mlp(xb, wg, wu, wd, sg, su, sd, yb, mw)
    assert torch.equal(yb, want) and torch.equal(xb, x)

    q, s = torch.empty((M, K), dtype=torch.int8, device=dev), torch.empty(M, device=dev)
    i8.quantize(x, q, s)
    raw = torch.zeros((M, 3 * K + 4 * N), dtype=torch.int8, device=dev)      # x, q and a product of it, a row behind another
    at = (0, 2 * K, 3 * K) if first else (4 * N + K, 4 * N, 0)
    xb, qb, yb = raw[:, at[0]:at[0] + 2 * K].view(BF), raw[:, at[1]:at[1] + K], raw[:, at[2]:at[2] + 4 * N].view(F32)
    xb.copy_(x)
    sb = torch.empty_like(s)
    i8.quantize(xb, qb, sb)
    assert torch.equal(qb, q) and torch.equal(sb, s) and torch.equal(xb, x)
    i8.matmul(qb, sb, w, ws, yb)
    assert torch.equal(yb, i8.matmul(q, s, w, ws, torch.empty((M, N), device=dev))) and torch.equal(qb, q)


@pytest.mark.parametrize("T", [2, 5, 16])
def test_layer(dev, T):
    L = Layer(12, 12, 0, 272, 144, 3, True, 17, dev)
    x = rows(T, 272, BF, T)
    want = L(x, BF)[0]
    buf = torch.zeros((T, 2 * 272), dtype=BF, device=dev)
    for xb, yb in ((buf[:, :272], buf[:, 272:]), (buf[:, 272:], buf[:, :272])):
        xb.copy_(x)
        L(xb, BF, out=yb)
        assert torch.equal(yb, want) and torch.equal(xb, x)
