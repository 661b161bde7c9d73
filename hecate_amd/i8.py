"""Products in 8-bit integers with a scale for each token and each output channel, and the gated MLP made of them.

Weights are int8 [N, K] row-major with one fp32 scale a row (the form in which the reference keeps its shared expert,
runtime/tier/tier_split.py:252-263); rows of x are quantised on the fly: s = max |x| / 127, q = x / s rounded half to
even. A row of zeros gives zeros; a row with a NaN or an infinity gives NaN in the whole output row. The integer sums are
exact, everything else is fp32, and the output is rounded once to its type (bf16, fp16 or fp32). K is a multiple of 16;
any number of rows, 0 included, and of output channels. x, q and out may have a row stride (x.stride(0)); w is
contiguous.

Work runs on the current torch stream of x's device and allocates nothing; a workspace (linear_work, mlp_work) is the
caller's, any contents work, and calls that share one must not overlap. Errors raise RuntimeError.
"""
import torch

from ._lib import call, dt_of, lib, on_device, ptr, stream_of


def _rows(what, t, M, K, dtype=None):
    """the row stride of a [M, K] tensor whose rows are contiguous"""
    if t.dim() != 2 or t.shape[0] != M or t.shape[1] != K or (K > 1 and t.stride(1) != 1) or (dtype is not None and t.dtype != dtype):
        raise RuntimeError(f"{what} must be [{M}, {K}]{'' if dtype is None else ' ' + str(dtype)} with contiguous rows, "
                           f"got {tuple(t.shape)} {t.dtype}")
    ld = t.stride(0)
    if M > 1 and ld < K:
        raise RuntimeError(f"{what}: rows overlap (stride {ld})")
    return max(ld, K)


def _vec(what, t, n):
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise RuntimeError(f"{what} must be {n} contiguous fp32 values")


def _mat(what, w, N, K):
    if w.dtype != torch.int8 or w.shape != (N, K) or not w.is_contiguous():
        raise RuntimeError(f"{what} must be contiguous int8 [{N}, {K}], got {tuple(w.shape)} {w.dtype}")


def _work(what, t, nbytes):
    if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() < nbytes:
        raise RuntimeError(f"{what}: the workspace must be contiguous uint8 of at least {nbytes} bytes")


def _run(dev, name, *args):
    """the C entry on dev's current stream, with dev as the current device"""
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return call(name, *args, stream_of(dev))
    call(name, *args, stream_of(dev))


def quantize(x, q, s):
    """x [M, K] (bf16, fp16 or fp32) as int8 q [M, K] and fp32 scales s [M]"""
    on_device("i8.quantize", x, q, s)
    M, K = x.shape
    ldx, ldq = _rows("i8.quantize: x", x, M, K), _rows("i8.quantize: q", q, M, K, torch.int8)
    _vec("i8.quantize: s", s, M)
    _run(x.device, "hmoe_i8_quantize", ptr(x), dt_of(x), ldx, M, K, ptr(q), ldq, ptr(s))
    return q, s


def matmul(q, s, w, ws, out, bias=None):
    """out [M, N] = s[m] ws[n] (q [M, K] w [N, K]^T) (+ bias [N] fp32) of rows that are in 8 bits already"""
    on_device("i8.matmul", q, s, w, ws, out, bias)
    M, K = q.shape
    N = w.shape[0]
    ldq, ldy = _rows("i8.matmul: q", q, M, K, torch.int8), _rows("i8.matmul: out", out, M, N)
    _mat("i8.matmul: w", w, N, K)
    _vec("i8.matmul: s", s, M)
    _vec("i8.matmul: ws", ws, N)
    if bias is not None:
        _vec("i8.matmul: bias", bias, N)
    _run(q.device, "hmoe_i8_matmul", ptr(q), ldq, ptr(s), M, ptr(w), K, ptr(ws), N, K, ptr(bias), ptr(out), dt_of(out), ldy)
    return out


def linear_work(device, M, N, K):
    """workspace of linear for up to M rows"""
    return torch.empty(max(int(lib().hmoe_i8_linear_work_bytes(M, N, K)), 16), dtype=torch.uint8, device=torch.device(device))


def linear(x, w, ws, out, work, bias=None):
    """out [M, N] = quantize(x [M, K]) w [N, K]^T (+ bias [N] fp32)"""
    on_device("i8.linear", x, w, ws, out, work, bias)
    M, K = x.shape
    N = w.shape[0]
    ldx, ldy = _rows("i8.linear: x", x, M, K), _rows("i8.linear: out", out, M, N)
    _mat("i8.linear: w", w, N, K)
    _vec("i8.linear: ws", ws, N)
    if bias is not None:
        _vec("i8.linear: bias", bias, N)
    _work("i8.linear", work, lib().hmoe_i8_linear_work_bytes(M, N, K))
    _run(x.device, "hmoe_i8_linear", ptr(x), dt_of(x), ldx, M, ptr(w), K, ptr(ws), N, K, ptr(bias), ptr(out), dt_of(out), ldy,
         ptr(work))
    return out


def mlp_work(device, M, H, I):
    """workspace of mlp for up to M rows"""
    return torch.empty(max(int(lib().hmoe_i8_mlp_work_bytes(M, H, I)), 16), dtype=torch.uint8, device=torch.device(device))


def mlp(x, wg, wu, wd, sg, su, sd, out, work):
    """out [M, H] = linear(h; wd, sd), h = silu(linear(x; wg, sg)) linear(x; wu, su) held in fp32 and quantised row by row;
    wg, wu int8 [I, H], wd int8 [H, I]"""
    on_device("i8.mlp", x, wg, wu, wd, sg, su, sd, out, work)
    M, H = x.shape
    I = wg.shape[0]
    ldx, ldy = _rows("i8.mlp: x", x, M, H), _rows("i8.mlp: out", out, M, H)
    _mat("i8.mlp: wg", wg, I, H)
    _mat("i8.mlp: wu", wu, I, H)
    _mat("i8.mlp: wd", wd, H, I)
    _vec("i8.mlp: sg", sg, I)
    _vec("i8.mlp: su", su, I)
    _vec("i8.mlp: sd", sd, H)
    _work("i8.mlp", work, lib().hmoe_i8_mlp_work_bytes(M, H, I))
    _run(x.device, "hmoe_i8_mlp", ptr(x), dt_of(x), ldx, M, H, I, ptr(wg), ptr(wu), ptr(wd), ptr(sg), ptr(su), ptr(sd), ptr(out),
         dt_of(out), ldy, ptr(work))
    return out
