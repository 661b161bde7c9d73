"""The 8-bit integer operators (hecate_amd.i8) on the GPU against their definitions in 64 bits (tests/i8ref.py): the whole
numbers and scales exactly, the products within their roundings."""
import numpy as np
import pytest
import torch

import i8ref as R
from hecate_amd import i8

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def log(*a):
    print(*a, flush=True)


def rows(M, K, dtype, seed, pad=0, dev="cuda", big=8.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn((M, K + pad), generator=g)
    t[:, :: max(1, K // 3)] *= big
    return t.to(dtype).to(dev)[:, :K]


def weight(N, K, seed, dev="cuda"):
    g = torch.Generator().manual_seed(seed + 1000)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    s = (0.5 + torch.rand(N, generator=g)) / (73.0 * K ** 0.5)
    return w.to(dev), s.to(dev)


def quantized(x):
    M, K = x.shape
    q = torch.full((M, K), 99, dtype=torch.int8, device=x.device)
    s = torch.full((M,), -1.0, device=x.device)
    i8.quantize(x, q, s)
    torch.cuda.synchronize()
    return q, s


def check_rows(x):
    q, s = quantized(x)
    qr, a = R.rows8(x)
    assert np.array_equal(q.cpu().numpy().astype(np.float64), qr)
    with np.errstate(all="ignore"):
        sr = (a[:, 0].astype(np.float32) / np.float32(127.0))
    assert np.array_equal(s.cpu().numpy(), sr, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K,pad", [(1, 16, 0), (1, 6144, 0), (3, 2048, 24), (7, 1360, 3), (65, 144, 8), (129, 4096, 0), (2, 16384, 0)])
def test_quantize(dev, dtype, M, K, pad):
    log("quantize", dtype, M, K, pad)
    check_rows(rows(M, K, dtype, M * 31 + K, pad))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_quantize_borders_and_extremes(dev, dtype):
    """ties between whole numbers, the type's largest and smallest values, rows of zeros and rows that are not finite"""
    top = float(torch.finfo(dtype).max)
    tiny = float(torch.finfo(dtype).smallest_normal)
    K = 256
    x = torch.zeros((16, K), dtype=torch.float64)
    n = torch.arange(-127, 128, dtype=torch.float64)
    x[0, :255] = n / 2                                    # a = 63.5: every odd n a whole number, every even n one too
    x[1, :254] = n[:-1] + 0.5                             # halves of a row of 127: exact ties
    x[1, 255] = 127.0
    x[2, :255] = n / 254                                  # a = 0.5: levels of n, many rounded to the type
    x[3, :255] = n * (top / 127)
    x[3, 255] = top
    x[4, :255] = n * tiny / 127
    x[5, 7] = tiny / 4                                    # a subnormal alone
    x[6, 3] = -top
    x[7, :255] = n + 0.5
    x[7, 9] = float("nan")
    x[8, 200] = float("inf")
    x[9, 0] = -float("inf")
    x[10, 0], x[10, 1] = 1.0, 1.0 / 254                   # a tie at a half (where the type holds it)
    x[11, :255] = n * tiny
    x[12, 0], x[12, 1:] = top, tiny
    x[13, :] = 1.0
    x[14, :128] = -3.0
    check_rows(x.to(dtype).to(dev))


def test_quantize_every_16_bit_quotient(dev):
    """every bf16 magnitude in [2^-9, 1] under rows whose largest value runs over a binade, and the fp16 ones around it"""
    for dtype, bits in ((BF, 7), (F16, 10)):
        vals = torch.cat([torch.arange(2 ** bits, 2 ** (bits + 1), dtype=torch.float64) * 2.0 ** (e - bits) for e in range(-9, 0)])
        tops = 1.0 + torch.arange(0, 2 ** bits, 1 if bits == 7 else 13, dtype=torch.float64) * 2.0 ** -bits
        K = -(-(vals.numel() + 1) // 16) * 16
        x = torch.zeros((tops.numel(), K), dtype=torch.float64)
        x[:, :vals.numel()] = vals
        x[:, vals.numel()] = tops
        log("quantize all", dtype, tuple(x.shape))
        check_rows(x.to(dtype).to(dev))


def check_out(out, p, y):
    got = out.float().cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    top = float(torch.finfo(out.dtype).max)
    b = R.product_bound(p, y, out.dtype)
    ok = np.isnan(y) | (np.abs(got - y) <= b) | ((np.abs(y) > top * (1 - R.HALF[out.dtype])) & np.isinf(got))
    i = np.argmax(np.where(ok, 0, np.abs(got - y)))
    assert ok.all(), (np.unravel_index(i, y.shape), got.flat[i], y.flat[i], b.flat[i])


PRODUCTS = [(1, 1, 16), (1, 17, 48), (2, 2048, 6144), (5, 250, 1360), (13, 33, 64), (16, 16, 128), (17, 129, 144), (63, 65, 2048),
            (64, 64, 80), (65, 257, 208), (130, 31, 6144), (200, 515, 272), (257, 384, 1024), (1, 640, 32), (3, 1501, 16), (520, 300, 656)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("odt", [BF, F16, F32])
def test_matmul(dev, M, N, K, odt):
    log("matmul", M, N, K, odt)
    g = torch.Generator().manual_seed(M + N + K)
    q = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
    s = 0.01 + torch.rand(M, generator=g)
    w, ws = weight(N, K, M + N)
    bias = torch.randn(N, generator=g) if (M + N) % 2 else None
    out = torch.full((M, N), 7.0, dtype=odt, device=dev)
    i8.matmul(q.to(dev), s.to(dev), w, ws, out, None if bias is None else bias.to(dev))
    torch.cuda.synchronize()
    p = R.product(q.double().numpy(), s.double().numpy()[:, None] * 127.0, w, ws)
    check_out(out, p, p if bias is None else p + bias.double().numpy())


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype,odt,pad", [(BF, BF, 0), (F16, F32, 8), (F32, F16, 3), (BF, F32, 5)])
def test_linear(dev, M, N, K, dtype, odt, pad):
    """rows cut out of a wider buffer, the output into one; what lies between the rows stays as it was"""
    log("linear", M, N, K, dtype, odt, pad)
    x = rows(M, K, dtype, M + K, pad)
    w, ws = weight(N, K, N)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(N)).to(dev) if N % 2 else None
    buf = torch.full((M + 2, N + pad), 7.0, dtype=odt, device=dev)
    out = buf[1:M + 1, :N]
    work = i8.linear_work(dev, M, N, K)
    i8.linear(x, w, ws, out, work, bias)
    torch.cuda.synchronize()
    q, a = R.rows8(x)
    p = R.product(q, a, w, ws)
    check_out(out, p, p if bias is None else p + bias.double().cpu().numpy())
    assert (buf[0] == 7.0).all() and (buf[M + 1] == 7.0).all() and (pad == 0 or bool((buf[:, N:] == 7.0).all()))


def test_extreme_weights_fill_the_accumulator(dev):
    """-128 x -128 over the largest depth: the sum just fits 32 bits"""
    K = 131056
    for M in (1, 3, 33, 200):
        q = torch.full((M, K), -128, dtype=torch.int8, device=dev)
        w = torch.full((20, K), -128, dtype=torch.int8, device=dev)
        one = torch.ones(M, device=dev)
        out = torch.empty((M, 20), device=dev)
        i8.matmul(q, one, w, torch.ones(20, device=dev), out)
        assert bool((out == float(np.float32(128.0 * 128.0 * K))).all())


# sizes that fall on each of the product's tile shapes in turn (i8_gemm1.hip), whole tiles and ragged ones, the depth ending
# inside a stage
TILES = [(7, 4100, 80), (16, 4096, 1024), (17, 2050, 80), (30, 2048, 400), (33, 4100, 144), (64, 2080, 656), (100, 4100, 80), (65, 4096, 384),
         (129, 6150, 80), (200, 4096, 144), (500, 4100, 80), (512, 4096, 128), (1000, 4100, 80), (1024, 4096, 144), (2000, 4100, 80),
         (2048, 6144, 128), (4100, 2050, 336)]


@pytest.mark.parametrize("M,N,K", TILES)
def test_matmul_tile_shapes(dev, M, N, K):
    log("tiles", M, N, K)
    g = torch.Generator().manual_seed(M + N + K)
    q = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
    s = 0.01 + torch.rand(M, generator=g)
    w, ws = weight(N, K, M + N)
    bias = torch.randn(N, generator=g)
    p = R.product(q.double().numpy(), s.double().numpy()[:, None] * 127.0, w, ws)
    for odt, b in ((BF, bias), (F32, None), (F16, bias)):
        buf = torch.full((M + 1, N + 8), 7.0, dtype=odt, device=dev)
        i8.matmul(q.to(dev), s.to(dev), w, ws, buf[:M, :N], None if b is None else b.to(dev))
        torch.cuda.synchronize()
        check_out(buf[:M, :N], p, p if b is None else p + b.double().numpy())
        assert bool((buf[M] == 7.0).all()) and bool((buf[:, N:] == 7.0).all())


def test_rows_that_are_not_finite_stay_apart(dev):
    """a NaN or an infinity makes its own row NaN and no other; a row of zeros gives the bias"""
    for M in (1, 4, 40, 300):
        x = rows(M, 512, BF, M).clone()
        if M > 1:
            x[1, 500] = float("nan")
            x[2, 0] = float("inf")
            x[3] = 0
        w, ws = weight(96, 512, 5)
        out = torch.empty((M, 96), device=dev)
        bias = torch.randn(96, device=dev)
        i8.linear(x, w, ws, out, i8.linear_work(dev, M, 96, 512), bias)
        q, a = R.rows8(x)
        p = R.product(q, a, w, ws)
        check_out(out, p, p + bias.double().cpu().numpy())
        if M > 1:
            assert bool(out[1:3].isnan().all()) and bool((out[3] == bias).all())


MLPS = [(1, 6144, 2048), (1, 16, 16), (2, 144, 48), (4, 2048, 1408), (13, 512, 272), (16, 1024, 704), (40, 256, 144), (77, 2048, 512),
        (150, 384, 1040), (300, 1024, 256), (16, 6144, 2048),
        # each of the gated product's tile shapes (i8_gemm2.hip)
        (17, 80, 2064), (100, 1040, 1040), (40, 80, 4112), (65, 144, 4096), (129, 80, 6160), (200, 128, 2048), (300, 80, 6160), (512, 128, 4096),
        (1000, 80, 4112), (2048, 144, 2048), (120, 6144, 2048)]


@pytest.mark.parametrize("M,H,I", MLPS)
@pytest.mark.parametrize("dtype,odt", [(BF, BF), (F16, F32)])
def test_mlp(dev, M, H, I, dtype, odt):
    log("mlp", M, H, I, dtype, odt)
    x = rows(M, H, dtype, M + H + I)
    (wg, sg), (wu, su), (wd, sd) = weight(I, H, 1), weight(I, H, 2), weight(H, I, 3)
    out = torch.full((M, H), 7.0, dtype=odt, device=dev)
    work = i8.mlp_work(dev, M, H, I)
    for _ in range(2):                                    # (the second call finds the first's workspace)
        i8.mlp(x, wg, wu, wd, sg, su, sd, out, work)
    torch.cuda.synchronize()
    y, slack, _ = R.mlp(*R.rows8(x), wg, wu, wd, sg, su, sd)
    d = np.abs(out.float().cpu().numpy() - y)
    b = R.product_bound(y, y, odt) + slack * (1 + 2 * R.HALF[odt])
    assert (d <= b).all(), (d.max(), np.argmax(d - b))


def test_mlp_rows_of_zeros_and_not_finite(dev):
    for M in (3, 30, 200):
        x = rows(M, 256, F16, M).clone()
        x[0] = 0
        x[1, 3] = float("inf")
        (wg, sg), (wu, su), (wd, sd) = weight(128, 256, 1), weight(128, 256, 2), weight(256, 128, 3)
        out = torch.empty((M, 256), dtype=F16, device=dev)
        i8.mlp(x, wg, wu, wd, sg, su, sd, out, i8.mlp_work(dev, M, 256, 128))
        assert bool((out[0] == 0).all()) and bool(out[1].isnan().all()) and not bool(out[2:].isnan().any())


def test_empty(dev):
    w, ws = weight(32, 64, 1)
    x = torch.empty((0, 64), dtype=BF, device=dev)
    out = torch.empty((0, 32), dtype=BF, device=dev)
    i8.linear(x, w, ws, out, i8.linear_work(dev, 0, 32, 64))
    i8.quantize(x, torch.empty((0, 64), dtype=torch.int8, device=dev), torch.empty(0, device=dev))
    i8.matmul(torch.empty((0, 64), dtype=torch.int8, device=dev), torch.empty(0, device=dev), w, ws, out)


def test_same_bits_every_time_captured_and_on_another_stream(dev):
    """the same call twice, from a captured graph replayed between eager calls, and on a side stream: the same bits"""
    for M in (1, 9, 100, 700):
        x = rows(M, 1024, BF, M)
        (wg, sg), (wu, su), (wd, sd) = weight(512, 1024, 1), weight(512, 1024, 2), weight(1024, 512, 3)
        outs = [torch.zeros((M, 1024), dtype=BF, device=dev) for _ in range(3)]
        lin = [torch.zeros((M, 512), device=dev) for _ in range(3)]
        work = [i8.mlp_work(dev, M, 1024, 512) for _ in range(3)]
        lw = [i8.linear_work(dev, M, 512, 1024) for _ in range(3)]

        def go(i):
            i8.mlp(x, wg, wu, wd, sg, su, sd, outs[i], work[i])
            i8.linear(x, wg, sg, lin[i], lw[i])

        go(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(lin[0], lin[1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(2)
        for k in range(3):
            x.copy_(rows(M, 1024, BF, M + k + 1))
            go(0)
            outs[2].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], outs[2]) and torch.equal(lin[0], lin[2]), (M, k)


# few rows (i8_few.hip): 8 and 16 weight rows a tile, one and several turns of the loads, several tiles a workgroup, tails of each
FEW = [(1, 9, 40960), (1, 20, 16400), (2, 4101, 16000), (3, 100, 13312), (8, 9, 4112), (8, 6150, 1040), (7, 515, 5136), (9, 37, 5120), (12, 8200, 528),
       (10, 77, 2576), (16, 30, 1536), (15, 8193, 1008), (16, 260, 2976), (5, 33, 9504)]


@pytest.mark.parametrize("M,N,K", FEW)
def test_few_rows(dev, M, N, K):
    w, ws = weight(N, K, M + N)
    for dtype, odt, pad in ((BF, F32, 0), (F16, BF, 8), (F32, F16, 1), (None, F32, 0)):
        log("few", M, N, K, dtype, odt, pad)
        bias = torch.randn(N, generator=torch.Generator().manual_seed(N)).to(dev) if pad else None
        x = rows(M, K, dtype or BF, M + K, pad)
        q, a = R.rows8(x)
        buf = torch.full((M + 2, N + pad), 7.0, dtype=odt, device=dev)
        if dtype is None:
            q8, s = torch.zeros((M, K + 16), dtype=torch.int8, device=dev)[:, :K], torch.zeros(M, device=dev)
            i8.quantize(x, q8, s)
            i8.matmul(q8, s, w, ws, buf[1:M + 1, :N], bias)
        else:
            i8.linear(x, w, ws, buf[1:M + 1, :N], i8.linear_work(dev, M, N, K), bias)
        torch.cuda.synchronize()
        p = R.product(q, a, w, ws)
        check_out(buf[1:M + 1, :N], p, p if bias is None else p + bias.double().cpu().numpy())
        assert bool((buf[0] == 7.0).all()) and bool((buf[M + 1] == 7.0).all()) and bool((buf[:, N:] == 7.0).all())


@pytest.mark.parametrize("M,H,I", [(1, 512, 9216), (3, 4096, 4112), (8, 1040, 2064), (12, 528, 4112), (16, 1024, 48), (9, 2064, 80)])
def test_few_rows_of_the_mlp(dev, M, H, I):
    test_mlp(dev, M, H, I, BF, F32)
    test_mlp(dev, M, H, I, F32, F16)
