"""A whole mixture-of-experts layer for up to 16 tokens with experts in 8 bits (the formats and roundings of i8.py).

    sel, rw   the topk experts of each token by sigmoid(wr x) + bias, equal ones in the order of their ids, and their
              weights scale a / (sum of the selected a + 1e-20), a = sigmoid(wr x) (the reference's selection,
              runtime/core/exl3_router.py:94-127, its scores summed in 64 bits here)
    out       the sum over the selected experts that are resident (lo <= id < lo + n) of weight x gated MLP, and the
              shared expert's MLP, in fp32, rounded once

Weights are int8 row-major: wg, wu [n, I, H], wd [n, H, I], fp32 scales sg, su [n, I], sd [n, H]; wr fp32 [E, H], bias fp32
[E] or None; shared is None or (wg, wu, wd, sg, su, sd) of one expert without the leading axis. H and I are multiples of 16 up
to 7168 and 4096, E at most 512, topk at most 16. A score that is NaN is selected last; a row with a NaN or an infinity gives NaN,
whether an expert of its own is resident or not.

Work runs on the current torch stream of x's device and allocates nothing; the workspace (layer_work) is the caller's, any
contents work, and calls that share one must not overlap. Errors raise RuntimeError.
"""
import ctypes

import torch

from ._lib import ptr
from .i8 import _bytes, _dt, _on, _rows, _run, _two, _vec, _work

_P3 = ctypes.c_void_p * 3


def layer_work(device, T, H, I, E, topk):
    """workspace of layer for up to T tokens"""
    nbytes = _bytes("hmoe_moe8_work_bytes", T, H, I, E, topk)
    if nbytes == 0:
        raise RuntimeError(f"moe8.layer_work: {T} tokens, H {H}, I {I}, {topk} of {E} experts: not a layer this operator takes")
    return torch.empty(nbytes, dtype=torch.uint8, device=torch.device(device))


def _w(what, t, shape, dtype):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise RuntimeError(f"moe8.layer: {what} must be contiguous {dtype} {list(shape)}, got {tuple(t.shape)} {t.dtype}")


def layer(x, wr, bias, wg, wu, wd, sg, su, sd, sel, rw, out, work, scale, lo=0, shared=None):
    """one layer of x [T, H] (bf16, fp16 or fp32) into sel int64 [T, topk], rw fp32 [T, topk] and out [T, H]"""
    if shared is not None and len(shared) != 6:
        raise RuntimeError(f"moe8.layer: shared must be six tensors (wg, wu, wd, sg, su, sd) or None, got {len(shared)}")
    _on("moe8.layer", x, wr, wg, wu, wd, sg, su, sd, sel, rw, out, x if bias is None else bias, x if work is None else work,
        *(shared or ()))
    T, H = _two("moe8.layer: x", x)
    E = _two("moe8.layer: wr", wr)[0]
    if wg.dim() != 3:
        raise RuntimeError(f"moe8.layer: wg must be [n, I, H], got {tuple(wg.shape)}")
    n, I = wg.shape[0], wg.shape[1]
    topk = _two("moe8.layer: sel", sel)[1]
    if not 0 <= lo <= E - n:
        raise RuntimeError(f"moe8.layer: resident experts [{lo}, {lo} + {n}) of {E}")
    ldx, ldy = _rows("moe8.layer: x", x, T, H), _rows("moe8.layer: out", out, T, H)
    i8, f32 = torch.int8, torch.float32
    for what, t, shape, dtype in (("wr", wr, (E, H), f32), ("wg", wg, (n, I, H), i8), ("wu", wu, (n, I, H), i8), ("wd", wd, (n, H, I), i8),
                                  ("sg", sg, (n, I), f32), ("su", su, (n, I), f32), ("sd", sd, (n, H), f32),
                                  ("sel", sel, (T, topk), torch.int64), ("rw", rw, (T, topk), f32)):
        _w(what, t, shape, dtype)
    if bias is not None:
        _vec("moe8.layer: bias", bias, E)
    sw = ss = None
    if shared is not None:
        for what, t, shape, dtype in zip(("shared wg", "shared wu", "shared wd", "shared sg", "shared su", "shared sd"), shared,
                                         ((I, H), (I, H), (H, I), (I,), (I,), (H,)), (i8, i8, i8, f32, f32, f32)):
            _w(what, t, shape, dtype)
        sw, ss = _P3(*map(ptr, shared[:3])), _P3(*map(ptr, shared[3:]))
    if T:
        _work("moe8.layer", work, _bytes("hmoe_moe8_work_bytes", T, H, I, E, topk))
    _run(x.device, "hmoe_moe8_layer", ptr(x), _dt("moe8.layer: x", x), ldx, T, ptr(wr), ptr(bias), E, topk, float(scale), ptr(wg), ptr(wu),
         ptr(wd), ptr(sg), ptr(su), ptr(sd), n, int(lo), H, I, sw, ss, ptr(sel), ptr(rw), ptr(out), _dt("moe8.layer: out", out), ldy,
         ptr(work))
    return out
