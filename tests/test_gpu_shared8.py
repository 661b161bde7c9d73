"""The int4 layer with a shared expert in 8 bits (tier.shared_int8, i8.mlp): decode, prefill and the decode stack against the
routed part by the layer without one and the shared part from its definition in 64 bits."""
import numpy as np
import pytest
import torch

import i8ref as R8

pytestmark = pytest.mark.gpu
H, I = 6144, 2048
N_LONG = 40                       # a long prefill's limit in these tests (tier.LONG_ROWS)


@pytest.fixture(scope="module")
def layers():
    """the same layer without a shared expert and with one in 8 bits"""
    from hecate_amd import synth, tier
    dev = torch.device("cuda:0")
    lay = synth.make_layer(0, dev, resident=range(24))
    m8 = tier.shared_int8(*lay.shared_rows())
    bank = lay.bank
    return (tier.MoELayer(lay.wg, lay.bias, bank, None, lo=0, n_hot=24), tier.MoELayer(lay.wg, lay.bias, bank, m8, lo=0, n_hot=24), lay)


def shared_rows(lay, x):
    """the shared expert's fp32 rows by the layer's own call, held against their definition"""
    from hecate_amd import i8
    T = x.shape[0]
    rows = lay.mlp8(x, torch.full((T, H), float("nan"), device=x.device), i8.mlp_work(x.device, T, H, I))
    pick = torch.as_tensor(np.unique(np.linspace(0, T - 1, min(T, 24)).astype(int)))
    q, a = R8.rows8(x[pick])
    y, slack, _ = R8.mlp(q, a, *lay.shared8)
    d = np.abs(rows[pick].double().cpu().numpy() - y)
    assert (d <= R8.product_bound(y, y, torch.float32) + slack).all(), d.max()
    assert float(np.abs(y).max()) > 0
    return rows


@pytest.mark.parametrize("R", [1, 2, 5, 8, 9, 16])
def test_decode(layers, R):
    from hecate_amd import synth
    none, lay, _ = layers
    print("decode", R, flush=True)
    x = synth.gen_x(70 + R, R, lay.device)
    routed = torch.zeros((R, H), device=lay.device)
    none.decode(x, y=routed, out=False)
    y0 = torch.randn((R, H), generator=torch.Generator().manual_seed(R)).to(lay.device)
    y = y0.clone()
    out = lay.decode(x, y=y).clone()
    z = torch.zeros_like(y)
    assert lay.decode(x, y=z, out=False) is None
    torch.cuda.synchronize()
    # the launches add one sum of their parts into y
    rows = shared_rows(lay, x)
    assert torch.equal(z, rows + routed) and torch.equal(y, y0 + z) and float(routed.abs().max()) > 0
    assert torch.equal(out, z.bfloat16())
    assert torch.equal(lay.decode(x), out)                               # (no y)
    part = torch.zeros_like(y)
    lay.decode(x, y=part, out=False, with_shared=False)
    assert torch.equal(part, routed)
    for ph in (1, 2, 4, 8):                                              # the launches apart
        o = lay.decode(x, phases=ph)
    assert torch.equal(o, out)
    lay.route(x)
    y = y0.clone()
    lay.experts_decode(R, y)
    want = y0 + rows
    none.route(x)
    none.experts_decode(R, want)
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError):
        lay.decode(x, y=None, out=False)


@pytest.mark.parametrize("ordered", [True, False])
@pytest.mark.parametrize("T", [17, 39, 41, 300])
def test_prefill(layers, monkeypatch, T, ordered):
    from hecate_amd import synth, tier
    monkeypatch.setattr(tier, "LONG_ROWS", N_LONG)
    none, lay, _ = layers
    print("prefill", T, ordered, flush=True)
    none.deterministic = lay.deterministic = ordered
    x = synth.gen_x(90 + T, T, lay.device)
    try:
        for _ in range(2):                                               # (the second call finds the first's buffers)
            out = lay.prefill(x).clone()
        pf = lay._pf
        y = torch.zeros((T, H), device=lay.device)
        lay.prefill_experts(pf.xh[:T], y)
        rows = shared_rows(lay, pf.xh[:T])
        none.prefill(x)
        routed = torch.zeros((T, H), device=lay.device)
        none.prefill_experts(none._pf.xh[:T], routed)
        if T <= N_LONG:
            # one sum of a row's picks, added once
            assert torch.equal(y, rows + routed) and torch.equal(out, y.bfloat16())
            return
        none.deterministic = True
        none.prefill(x)
        # eight picks, each at most the largest down product (their weights, at most 2.5 together, applied to it or not), and the
        # shared row: nine additions in one order and in another, each rounded to fp32
        # (the products' buffer holds as many rows as the plan has picks of resident experts; behind them is what was there before)
        most = 8.0 * float(none._pf.scr[2][:int(none._pf.meta[0])].abs().max())
        d = 18 * R8.U * (most + rows.abs().double())
        assert bool(((y.double() - rows.double() - routed.double()).abs() <= d).all())
        # (a half step of bf16, of a value that is d from y's)
        assert bool(((out.double() - y.double()).abs() <= 2.0 ** -8 * (y.abs().double() + d) + d).all())
    finally:
        none.deterministic = lay.deterministic = True


@pytest.mark.parametrize("R", [1, 4])
def test_stack(layers, R):
    """the stack's forms give the same bits, eager, captured and replayed between eager work"""
    from hecate_amd import stack, synth
    none, lay, f16 = layers
    w = [torch.ones(H, device=lay.device) for _ in range(3)]
    s = stack.DecodeStack([f16, lay, none], w, R)
    s.x.copy_(synth.gen_x(5, R, lay.device))
    a = s.step(fused=False).clone()
    assert torch.equal(s.step().clone(), a)
    s.capture()
    for k in range(3):
        s.x.copy_(synth.gen_x(6 + k, R, lay.device))
        want = s.step().clone()
        s.h.zero_()
        got = s.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want), k


def test_matrices_in_8_bits(layers):
    """shared_int8 is i8.quantize of the rows"""
    _, lay, f16 = layers
    for m, (w8, s) in zip(f16.shared_rows(), ((0, 3), (1, 4), (2, 5))):
        q, a = R8.rows8(m[:64])
        assert np.array_equal(lay.shared8[w8][:64].cpu().numpy().astype(np.float64), q)
        assert np.allclose(lay.shared8[s][:64].double().cpu().numpy(), a[:, 0] / 127.0, rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("T", [1, 6, 30])
def test_captured(layers, T):
    """decode (1, 6) and prefill (30) captured, replayed between eager calls of the same layer's twin"""
    from hecate_amd import synth, tier
    _, lay, _ = layers
    twin = tier.MoELayer(lay.wg, lay.bias, lay.bank, lay.shared8, lo=0, n_hot=24)
    x = synth.gen_x(3, T, lay.device)
    lay.forward(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = lay.forward(x)
    for k in range(3):
        x.copy_(synth.gen_x(30 + k, T, lay.device))
        want = twin.forward(x).clone()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), k
