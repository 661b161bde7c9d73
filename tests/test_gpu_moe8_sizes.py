"""Every form of the 8-bit expert layer's kernel (the lines of a hidden row that a wave takes: 1, 2, 4, 6, 7; of an intermediate row: 1, 2,
4) against its definition in 64 bits, with one token and with 16."""
import numpy as np
import pytest
import torch

import i8ref as R
from test_gpu_moe8 import BF, F16, F32, Layer, log, rows

pytestmark = pytest.mark.gpu


class ByExpert(Layer):
    """the same reference with each expert's weights widened once"""

    def reference(self, x):
        xd = x.double().cpu().numpy()
        a = 1.0 / (1.0 + np.exp(-(xd @ self.wr.double().numpy().T)))
        key = a + (self.bias.double().numpy() if self.bias is not None else 0.0)
        sel = np.argsort(-key, axis=1, kind="stable")[:, :self.topk]
        top = np.take_along_axis(a, sel, 1)
        rw = self.scale * top / (top.sum(1, keepdims=True) + 1e-20)
        q, m = R.rows8(x)
        y, slack, size = (np.zeros(xd.shape) for _ in range(3))

        def add(t, w, e):
            yy, ss, aa = R.mlp(q[t], m[t], *e)
            y[t] += w * yy
            slack[t] += w * ss
            size[t] += w * aa

        for i in range(self.n):
            t, j = np.nonzero(sel == i + self.lo)
            if t.size:
                add(t, rw[t, j][:, None], [v[i] for v in self.w] + [v[i] for v in self.s])
        if self.sh is not None:
            add(np.arange(xd.shape[0]), 1.0, self.sh)
        return y, sel, rw, slack, size


@pytest.mark.parametrize("E,n,lo,H,I,topk,shared", [
    (6, 6, 0, 2048, 1408, 3, True), (9, 7, 1, 1040, 1040, 4, False),                  # 2 and 2
    (3, 3, 0, 4096, 2064, 2, True), (4, 3, 0, 2576, 4096, 3, False),                  # 4 and 4
    (3, 2, 1, 6144, 4096, 2, False), (2, 2, 0, 4624, 2576, 1, True),                  # 6 and 4
    (3, 3, 0, 7168, 2048, 2, True), (6, 5, 0, 6160, 1040, 4, False),                  # 7 and 2
    (2, 2, 0, 7168, 4096, 1, True), (4, 4, 0, 7168, 2064, 3, False)])                 # 7 and 4
def test_every_form(dev, E, n, lo, H, I, topk, shared):
    L = ByExpert(E, n, lo, H, I, topk, shared, E + H + I, dev)
    work = L.work(16)
    for T, dtype, odt in ((1, BF, F32), (16, F16, BF), (3, F32, F16), (16, BF, F32)):
        log("form", E, n, lo, H, I, topk, shared, T)
        x = rows(T, H, dtype, T + H, dev)
        got = L(x, odt, work)
        torch.cuda.synchronize()
        L.check(x, odt, got)
