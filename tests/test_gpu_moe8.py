"""The whole 8-bit expert layer (hecate_amd.moe8) on the GPU against its definition in 64 bits (tests/i8ref.py): the selection
exactly, the weights and the output within their roundings."""
import numpy as np
import pytest
import torch

import i8ref as R
from hecate_amd import moe8

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def log(*a):
    print(*a, flush=True)


class Layer:
    """random experts and router on the host and on the device"""

    def __init__(self, E, n, lo, H, I, topk, shared, seed, dev, bias=True):
        g = torch.Generator().manual_seed(seed)
        self.E, self.n, self.lo, self.H, self.I, self.topk, self.scale = E, n, lo, H, I, topk, 2.5

        def mat(*shape):
            w = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
            return w, (0.5 + torch.rand(shape[:-1], generator=g)) / (73.0 * shape[-1] ** 0.5)

        self.wr = torch.randn((E, H), generator=g) / H ** 0.5
        self.bias = 0.05 * torch.randn(E, generator=g) if bias else None
        mats = [mat(n, I, H), mat(n, I, H), mat(n, H, I)]
        self.w, self.s = [m[0] for m in mats], [m[1] for m in mats]
        sh = [mat(I, H), mat(I, H), mat(H, I)] if shared else None
        self.sh = [m[0] for m in sh] + [m[1] for m in sh] if shared else None
        self.d = lambda t: None if t is None else t.to(dev)
        self.dev = dev
        self.dw, self.ds = [t.to(dev) for t in self.w], [t.to(dev) for t in self.s]
        self.dsh = [t.to(dev) for t in self.sh] if shared else None

    def work(self, T):
        return moe8.layer_work(self.dev, T, self.H, self.I, self.E, self.topk)

    def __call__(self, x, odt, work=None, out=None):
        T = x.shape[0]
        sel = torch.full((T, self.topk), -1, dtype=torch.int64, device=self.dev)
        rw = torch.full((T, self.topk), -1.0, device=self.dev)
        out = torch.full((T, self.H), 7.0, dtype=odt, device=self.dev) if out is None else out
        moe8.layer(x, self.wr.to(self.dev), self.d(self.bias), *self.dw, *self.ds, sel, rw, out, self.work(T) if work is None else work,
                   self.scale, self.lo, self.dsh)
        return out, sel, rw

    def reference(self, x):
        xd = x.double().cpu().numpy()
        with np.errstate(all="ignore"):
            a = 1.0 / (1.0 + np.exp(-(xd @ self.wr.double().numpy().T)))
        key = a + (self.bias.double().numpy() if self.bias is not None else 0.0)
        key = np.where(np.isnan(key), -np.inf, key)
        sel = np.argsort(-key, axis=1, kind="stable")[:, :self.topk]
        top = np.take_along_axis(a, sel, 1)
        rw = self.scale * top / (top.sum(1, keepdims=True) + 1e-20)
        q, m = R.rows8(x)
        y = np.zeros(xd.shape)
        slack = np.zeros(xd.shape)
        size = np.zeros(xd.shape)                         # what the sum's roundings scale with
        def add(t, w, e):
            yy, ss, aa = R.mlp(q[t:t + 1], m[t:t + 1], *e)
            y[t] += (w * yy)[0]
            slack[t] += (abs(w) * ss)[0]
            size[t] += (abs(w) * aa)[0]
        for t in range(xd.shape[0]):
            for j in range(self.topk):
                i = sel[t, j] - self.lo
                if 0 <= i < self.n:
                    add(t, rw[t, j], [v[i] for v in self.w] + [v[i] for v in self.s])
            if self.sh is not None:
                add(t, 1.0, self.sh)
        return y, sel, rw, slack, size

    def check(self, x, odt, got, gaps=True):
        out, sel, rw = got
        y, rsel, rrw, slack, size = self.reference(x)
        assert np.array_equal(sel.cpu().numpy(), rsel)
        assert np.allclose(rw.cpu().numpy(), rrw, rtol=2 * R.U, atol=0, equal_nan=True)
        o = out.float().cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(o), np.isnan(y))
        # a piece of the depth of an expert's term carries the roundings of its cast, two scales, their product and the weight
        # (6 u of at most `size`), the sum over at most 17 experts and 8 pieces one rounding each (25 u)
        b = R.product_bound(y, y, odt) + (slack + (6 + 25) * R.U * size) * (1 + 2 * R.HALF[odt])
        bad = np.abs(o - y) > b
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(o - y)[bad][:4], b[bad][:4])


def rows(T, H, dtype, seed, dev, pad=0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn((T, H + pad), generator=g)
    t[:, :: max(1, H // 3)] *= 6.0
    return t.to(dtype).to(dev)[:, :H]


SIZES = [  # E, n, lo, H, I, topk, shared
    (1, 1, 0, 16, 16, 1, False), (3, 3, 0, 48, 80, 2, True), (8, 8, 0, 256, 128, 2, True), (60, 40, 11, 512, 352, 4, False),
    (64, 1, 63, 144, 272, 6, True), (20, 20, 0, 1024, 704, 16, True), (128, 100, 0, 2048, 144, 8, False), (512, 512, 0, 96, 32, 16, True),
    (7, 7, 0, 6144, 2048, 3, True), (4, 4, 0, 7168, 48, 4, False), (4, 4, 0, 48, 4096, 4, True), (257, 200, 57, 176, 1104, 5, True),
    (5, 5, 0, 4096, 1536, 2, True), (9, 9, 0, 7168, 208, 8, False), (6, 6, 0, 1040, 2064, 2, True)]


@pytest.mark.parametrize("E,n,lo,H,I,topk,shared", SIZES)
@pytest.mark.parametrize("T", [1, 2, 5, 16])
def test_layer(dev, E, n, lo, H, I, topk, shared, T):
    log("layer", E, n, lo, H, I, topk, shared, T)
    L = Layer(E, n, lo, H, I, topk, shared, E + H, dev, bias=E % 3 != 0)
    work = L.work(16)
    forms = [(BF, BF, 0), (F16, F32, 8), (F32, F16, 3)]
    for k, (dtype, odt, pad) in enumerate(forms if T == 5 else [forms[(T + E) % 3]]):
        x = rows(T, H, dtype, T + H + k, dev, pad)
        got = L(x, odt, work)
        torch.cuda.synchronize()
        L.check(x, odt, got)


def test_no_expert_resident(dev):
    """only picks that live elsewhere, with and without a shared expert: the shared expert's rows, or zeros"""
    L = Layer(16, 0, 16, 64, 32, 4, False, 1, dev)
    out, sel, rw = L(rows(3, 64, BF, 1, dev), F32)
    assert bool((out == 0).all()) and bool((sel >= 0).all())
    L = Layer(16, 2, 14, 64, 32, 1, True, 2, dev)
    L.bias[14:] = -float("inf")
    x = rows(4, 64, BF, 1, dev)
    L.check(x, F32, L(x, F32))


def test_equal_scores_take_the_lowest_ids(dev):
    L = Layer(40, 40, 0, 128, 64, 8, True, 3, dev, bias=False)
    L.wr[:] = L.wr[0]
    x = rows(6, 128, F16, 4, dev)
    got = L(x, F32)
    assert np.array_equal(got[1].cpu().numpy(), np.tile(np.arange(8), (6, 1)))
    L.check(x, F32, got)


def test_bias_that_closes_experts_and_saturated_scores(dev):
    """a bias of -inf closes an expert until nothing else is left; scores that round to one tie; scores that underflow give zeros"""
    L = Layer(12, 12, 0, 64, 48, 5, False, 5, dev)
    L.bias[:9] = -float("inf")
    x = rows(5, 64, BF, 6, dev)
    got = L(x, F32)
    L.check(x, F32, got)
    assert sorted(got[1][0, :3].tolist()) == [9, 10, 11] and got[1][0, 3:].tolist() == [0, 1]
    L = Layer(12, 12, 0, 64, 48, 5, False, 7, dev, bias=False)
    L.wr[:] = 0
    L.wr[:, 0] = 1000.0
    x = torch.ones((2, 64), dtype=BF, device=dev)
    x[1, 0] = -1.0
    L.check(x, F32, L(x, F32))


def test_rows_that_are_not_finite(dev):
    L = Layer(30, 30, 0, 256, 128, 6, True, 9, dev)
    x = rows(6, 256, BF, 3, dev).clone()
    x[1, 5] = float("nan")
    x[3, 250] = float("inf")
    x[4] = 0
    out, sel, rw = L(x, F32)
    o = out.cpu()
    assert bool(o[1].isnan().all()) and bool(o[3].isnan().all()) and bool((o[4] == 0).all())
    assert not bool(o[[0, 2, 5]].isnan().any())
    assert int(sel.min()) >= 0 and int(sel.max()) < 30
    assert sel[1].tolist() == list(range(6))
    keep = [0, 2, 5]
    y, rsel, _, _, _ = L.reference(x[keep])
    assert np.array_equal(sel.cpu().numpy()[keep], rsel) and np.allclose(o.numpy()[keep], y, rtol=1e-2, atol=1e-2 * np.abs(y).max())


def test_same_bits_every_time_captured_and_side_by_side(dev):
    """two layers on two streams at once, and replays of a captured call between eager ones: the bits of one call alone"""
    L = Layer(64, 64, 0, 1024, 512, 8, True, 11, dev)
    wr, bias = L.wr.to(dev), L.bias.to(dev)
    for T in (1, 7, 16):
        xs = [rows(T, 1024, BF, 20 + k, dev) for k in range(2)]
        bufs = [(torch.empty((T, 8), dtype=torch.int64, device=dev), torch.empty((T, 8), device=dev),
                 torch.zeros((T, 1024), dtype=BF, device=dev), L.work(16)) for _ in range(5)]

        def go(k, x):
            sel, rw, out, work = bufs[k]
            moe8.layer(x, wr, bias, *L.dw, *L.ds, sel, rw, out, work, 2.5, 0, L.dsh)

        go(0, xs[0]); go(1, xs[1])
        torch.cuda.synchronize()
        st = [torch.cuda.Stream() for _ in range(2)]
        for k in range(2):
            st[k].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st[k]):
                for _ in range(20):
                    go(2 + k, xs[k])
        torch.cuda.synchronize()
        for k in range(2):
            for i in range(3):
                assert torch.equal(bufs[k][i], bufs[2 + k][i]), (T, k, i)
        x = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(4, x)
        for k in range(4):
            x.copy_(rows(T, 1024, BF, 40 + k, dev))
            go(0, x)
            bufs[4][2].zero_()
            g.replay()
            torch.cuda.synchronize()
            for i in range(3):
                assert torch.equal(bufs[0][i], bufs[4][i]), (T, k, i)


def test_rows_beside_the_output_stay(dev):
    L = Layer(8, 8, 0, 272, 144, 2, True, 13, dev)
    buf = torch.full((5, 272 + 6), 7.0, dtype=F16, device=dev)
    x = rows(3, 272, F16, 5, dev)
    out, sel, rw = L(x, F16, out=buf[1:4, :272])
    L.check(x, F16, (out, sel, rw))
    assert bool((buf[0] == 7).all()) and bool((buf[4] == 7).all()) and bool((buf[:, 272:] == 7).all())


@pytest.mark.parametrize("E,n,lo,H,I,topk,shared", [(46, 46, 0, 1840, 288, 5, True), (16, 11, 3, 528, 496, 7, False), (12, 12, 0, 2576, 304, 3, True),
                                                    (5, 5, 0, 4624, 112, 2, True), (200, 200, 0, 512, 1024, 8, True)])
@pytest.mark.parametrize("T", [1, 4, 13, 16])
def test_layer_of_many_rows(dev, E, n, lo, H, I, topk, shared, T):
    """slots of one row and of many in the down batches, each number of loads of a router's row"""
    log("layer of many rows", E, n, lo, H, I, topk, shared, T)
    L = Layer(E, n, lo, H, I, topk, shared, E + H, dev)
    x = rows(T, H, F16, T + H, dev, 5)
    got = L(x, F32, L.work(T))
    torch.cuda.synchronize()
    L.check(x, F32, got)
