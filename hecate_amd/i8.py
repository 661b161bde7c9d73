"""Products in 8-bit integers with a scale for each token and each output channel, and the gated MLP made of them.

Weights are int8 [N, K] row-major with one fp32 scale a row (the form in which the reference keeps its shared expert,
runtime/tier/tier_split.py:252-263); rows of x are quantised on the fly: s = max |x| / 127, q = x / s rounded half to
even. A row of zeros gives zeros; a row with a NaN or an infinity gives NaN in the whole output row. The integer sums are
exact, everything else is fp32, and the output is rounded once to its type (bf16, fp16 or fp32). K is a multiple of 16 up to
131056; rows up to 2^20, 0 included, output channels 1 to 2^20. x, q and out may have a row stride (x.stride(0); below 2^28 for
the q of a product, and a multiple of 16 for any q), and be column ranges of one buffer; w is contiguous.

Work runs on the current torch stream of x's device and allocates nothing; a workspace (linear_work, mlp_work) is the
caller's, any contents work, and calls that share one must not overlap. Errors raise RuntimeError.
"""
from functools import lru_cache

import torch

from ._lib import check, lib, on_device

_MAX = (1 << 31) - 1                      # the C entries' sizes are 32-bit; a larger one would be cut to its low bits
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}            # the dtype codes of include/hecate_moe.h (HMOE_DT_*)


_device, _stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _dt(what, t):
    d = _DT.get(t.dtype)
    if d is None:
        raise RuntimeError(f"{what}: dtype {t.dtype} not supported here (float32, bfloat16, float16)")
    return d


def _rows(what, t, M, K, dtype=None):
    """the row stride of a [M, K] tensor whose rows are contiguous"""
    if t.shape != (M, K) or (dtype is not None and t.dtype != dtype):
        raise RuntimeError(f"{what} must be [{M}, {K}]{'' if dtype is None else ' ' + str(dtype)} with contiguous rows, "
                           f"got {tuple(t.shape)} {t.dtype}")
    return _stride(what, t, M, K)


def _stride(what, t, M, K):
    """the same of a tensor whose shape is known"""
    ld, step = t.stride()
    if K > 1 and step != 1:
        raise RuntimeError(f"{what} must be [{M}, {K}] with contiguous rows, got strides {t.stride()}")
    if M <= 1:
        return K
    if ld < K:
        raise RuntimeError(f"{what}: rows overlap (stride {ld})")
    return ld


def _vec(what, t, n):
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise RuntimeError(f"{what} must be {n} contiguous fp32 values")


def _mat(what, w, N, K):
    if w.dtype != torch.int8 or w.shape != (N, K) or not w.is_contiguous():
        raise RuntimeError(f"{what} must be contiguous int8 [{N}, {K}], got {tuple(w.shape)} {w.dtype}")


def _work(what, t, nbytes):
    if t is None or t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() < nbytes:
        raise RuntimeError(f"{what}: the workspace must be contiguous uint8 of at least {nbytes} bytes")


def _two(what, x):
    sh = x.shape
    if len(sh) != 2:
        raise RuntimeError(f"{what} must have two dimensions, got {tuple(sh)}")
    if sh[0] > _MAX or sh[1] > _MAX:
        raise RuntimeError(f"{what}: {tuple(sh)}: more than {_MAX} rows or columns")
    return sh


def _on(what, x, *ts):
    """raise unless every argument is a tensor on x's GPU (on_device, by the devices' numbers); x stands for one that may be left out"""
    try:
        i = x.get_device()
        if i >= 0 and x.is_cuda:
            for t in ts:
                if t.get_device() != i:
                    break
            else:
                return
    except AttributeError:
        pass
    on_device(what, x, *ts)
    raise RuntimeError(f"{what}: an argument that has to be a tensor is None or a number")


@lru_cache(maxsize=256)
def _bytes(name, *sizes):
    if any(n > _MAX for n in sizes):
        raise RuntimeError(f"{name}: a size of {sizes} is more than {_MAX}")
    return int(getattr(lib(), name)(*sizes))


def _run(dev, name, *args):
    """the C entry on dev's current stream, with dev as the current device (raw queries: a call of a few microseconds pays
    for every Python object that it makes)"""
    i = dev.index
    if i != _device():
        with torch.cuda.device(dev):
            rc = getattr(lib(), name)(*args, _stream(i))
    else:
        rc = getattr(lib(), name)(*args, _stream(i))
    if rc:
        check(rc, name)


def quantize(x, q, s):
    """x [M, K] (bf16, fp16 or fp32) as int8 q [M, K] and fp32 scales s [M]"""
    _on("i8.quantize", x, q, s)
    M, K = _two("i8: x", x)
    ldx, ldq = _stride("i8.quantize: x", x, M, K), _rows("i8.quantize: q", q, M, K, torch.int8)
    _vec("i8.quantize: s", s, M)
    _run(x.device, "hmoe_i8_quantize", x.data_ptr(), _dt("i8: x", x), ldx, M, K, q.data_ptr(), ldq, s.data_ptr())
    return q, s


def matmul(q, s, w, ws, out, bias=None):
    """out [M, N] = s[m] ws[n] (q [M, K] w [N, K]^T) (+ bias [N] fp32) of rows that are in 8 bits already"""
    _on("i8.matmul", q, s, w, ws, out, q if bias is None else bias)
    M, K = _two("i8: q", q)
    N = _two("i8: w", w)[0]
    if q.dtype != torch.int8:
        raise RuntimeError(f"i8.matmul: q must be int8, got {q.dtype}")
    ldq, ldy = _stride("i8.matmul: q", q, M, K), _rows("i8.matmul: out", out, M, N)
    _mat("i8.matmul: w", w, N, K)
    _vec("i8.matmul: s", s, M)
    _vec("i8.matmul: ws", ws, N)
    if bias is not None:
        _vec("i8.matmul: bias", bias, N)
    _run(q.device, "hmoe_i8_matmul", q.data_ptr(), ldq, s.data_ptr(), M, w.data_ptr(), K, ws.data_ptr(), N, K,
         None if bias is None else bias.data_ptr(), out.data_ptr(), _dt("i8: out", out), ldy)
    return out


def linear_work(device, M, N, K):
    """workspace of linear for up to M rows"""
    return torch.empty(max(_bytes("hmoe_i8_linear_work_bytes", M, N, K), 16), dtype=torch.uint8, device=torch.device(device))


def linear(x, w, ws, out, work, bias=None):
    """out [M, N] = quantize(x [M, K]) w [N, K]^T (+ bias [N] fp32)"""
    _on("i8.linear", x, w, ws, out, work, x if bias is None else bias)
    M, K = _two("i8: x", x)
    N = _two("i8: w", w)[0]
    ldx, ldy = _stride("i8.linear: x", x, M, K), _rows("i8.linear: out", out, M, N)
    _mat("i8.linear: w", w, N, K)
    _vec("i8.linear: ws", ws, N)
    if bias is not None:
        _vec("i8.linear: bias", bias, N)
    _work("i8.linear", work, _bytes("hmoe_i8_linear_work_bytes", M, N, K))
    _run(x.device, "hmoe_i8_linear", x.data_ptr(), _dt("i8: x", x), ldx, M, w.data_ptr(), K, ws.data_ptr(), N, K,
         None if bias is None else bias.data_ptr(), out.data_ptr(), _dt("i8: out", out), ldy, work.data_ptr())
    return out


def mlp_work(device, M, H, I):
    """workspace of mlp for up to M rows"""
    return torch.empty(max(_bytes("hmoe_i8_mlp_work_bytes", M, H, I), 16), dtype=torch.uint8, device=torch.device(device))


def mlp(x, wg, wu, wd, sg, su, sd, out, work):
    """out [M, H] = linear(h; wd, sd), h = silu(linear(x; wg, sg)) linear(x; wu, su) held in fp32 and quantised row by row;
    wg, wu int8 [I, H], wd int8 [H, I]"""
    _on("i8.mlp", x, wg, wu, wd, sg, su, sd, out, work)
    M, H = _two("i8: x", x)
    I = _two("i8.mlp: wg", wg)[0]
    ldx, ldy = _stride("i8.mlp: x", x, M, H), _rows("i8.mlp: out", out, M, H)
    _mat("i8.mlp: wg", wg, I, H)
    _mat("i8.mlp: wu", wu, I, H)
    _mat("i8.mlp: wd", wd, H, I)
    _vec("i8.mlp: sg", sg, I)
    _vec("i8.mlp: su", su, I)
    _vec("i8.mlp: sd", sd, H)
    _work("i8.mlp", work, _bytes("hmoe_i8_mlp_work_bytes", M, H, I))
    _run(x.device, "hmoe_i8_mlp", x.data_ptr(), _dt("i8: x", x), ldx, M, H, I, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), sg.data_ptr(),
         su.data_ptr(), sd.data_ptr(), out.data_ptr(), _dt("i8: out", out), ldy, work.data_ptr())
    return out
