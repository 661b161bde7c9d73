"""Timed cases of the 8-bit integer operators: the matrix product with a scale for each token and each channel, on rows
that are in 8 bits already (matmul) and on rows that it quantises itself (linear), the gated MLP made of three such
products, and a whole mixture-of-experts layer of such experts for a few tokens.

Where `own` is false, run() computes them in elementary torch operations; where it is true, through hecate_amd.i8 and
hecate_amd.moe8."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a long chunk's down projection on quantised rows: the largest product; and a decode batch of an odd number of rows
        dict(name="matmul 8192x6144x2048 bf16", op="matmul", M=8192, N=6144, K=2048, out="bf16", bias=False),
        dict(name="matmul 13x6144x2048 f16 bias", op="matmul", M=13, N=6144, K=2048, out="f16", bias=True),
        # one token through an up projection: latency and weight streaming
        dict(name="linear 1x2048x6144 bf16", op="linear", M=1, N=2048, K=6144, x="bf16", out="bf16", bias=False, pad=0),
        # a ragged serving batch: odd rows, rows cut out of a wider buffer
        dict(name="linear 61x2048x6144 f16", op="linear", M=61, N=2048, K=6144, x="f16", out="f16", bias=False, pad=24),
        # odd rows and channels, a depth that ends inside a tile, 32-bit rows in and out
        dict(name="linear 333x1501x1360 f32", op="linear", M=333, N=1501, K=1360, x="f32", out="f32", bias=True, pad=0),
        # a 2048-token chunk through gate and up at once
        dict(name="linear 2048x4096x6144 bf16", op="linear", M=2048, N=4096, K=6144, x="bf16", out="bf16", bias=False, pad=0),
        # the shared expert at one token, at an odd prompt and at a 2048-token chunk
        dict(name="mlp 1 bf16", op="mlp", M=1, H=6144, I=2048, x="bf16", out="bf16"),
        dict(name="mlp 77 f16", op="mlp", M=77, H=6144, I=2048, x="f16", out="f16"),
        dict(name="mlp 2048 bf16", op="mlp", M=2048, H=6144, I=2048, x="bf16", out="bf16"),
        # the whole layer: one token, a 16-row step, and a smaller layer of which a device holds a part of the experts
        dict(name="layer 1 of 256 experts", op="layer", T=1, H=6144, I=2048, E=256, n=256, lo=0, topk=8, shared=True, x="bf16", out="bf16"),
        dict(name="layer 16 of 256 experts", op="layer", T=16, H=6144, I=2048, E=256, n=256, lo=0, topk=8, shared=True, x="bf16", out="bf16"),
        dict(name="layer 5, 40 of 60 experts", op="layer", T=5, H=2048, I=1408, E=60, n=40, lo=11, topk=4, shared=False, x="f16", out="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    x = rng.choice(["bf16", "f16"])
    op = rng.choice(["matmul", "linear", "mlp", "layer"])
    if op in ("matmul", "linear"):
        M = _log(rng, 1, 8192)
        c = dict(op=op, M=M, N=_log(rng, 33, 6144), K=16 * _log(rng, 8, 384 if M < 4096 else 128), out=rng.choice(["bf16", "f16", "f32"]),
                 bias=rng.random() < 0.5)
        return c if op == "matmul" else dict(c, x=rng.choice(["bf16", "f16", "f32"]), pad=8 * rng.randint(0, 5))
    if op == "mlp":
        return dict(op=op, M=_log(rng, 1, 2048), H=16 * _log(rng, 16, 384), I=16 * _log(rng, 8, 128), x=x, out=x)
    E = _log(rng, 8, 256)
    n = rng.choice([E, rng.randint(1, E)])
    return dict(op=op, T=rng.randint(1, 16), H=16 * _log(rng, 16, 384), I=16 * _log(rng, 8, 128), E=E, n=n, lo=rng.randint(0, E - n),
                topk=rng.randint(1, min(8, E)), shared=rng.random() < 0.5, x=x, out=x)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _rows(gen, M, K, kind, pad=0):
    """normed activations: unit rows with a few channels 16 times as large, as the residual stream of a trained model has"""
    t = torch.randn((M, K + pad), generator=gen, device="cuda")
    t[:, torch.randint(0, K, (max(1, K // 512),), generator=gen, device="cuda")] *= 16.0
    return t.to(TYPES[kind])[:, :K]


def _weight(gen, *shape):
    """8-bit weights in [-127, 127] and the fp32 scale of each output channel, such that products of unit rows are of order one"""
    w = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    s = (0.5 + torch.rand(shape[:-1], generator=gen, device="cuda")) / (73.0 * math.sqrt(shape[-1]))
    return w, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, op = case, case["op"]
    if op in ("matmul", "linear"):
        w, ws = _weight(gen, c["N"], c["K"])
        b = torch.randn(c["N"], generator=gen, device="cuda") if c["bias"] else None
        s = dict(op=op, w=w, ws=ws, b=b, out=torch.empty((c["M"], c["N"]), dtype=TYPES[c["out"]], device="cuda"), work=None)
        if op == "linear":
            return dict(s, x=_rows(gen, c["M"], c["K"], c["x"], c["pad"]))
        q = (30.0 * torch.randn((c["M"], c["K"]), generator=gen, device="cuda")).round().clamp(-127, 127).to(torch.int8)
        return dict(s, q=q, qs=(0.5 + torch.rand(c["M"], generator=gen, device="cuda")) / 30.0)
    H, I = c["H"], c["I"]
    if op == "mlp":
        x = _rows(gen, c["M"], H, c["x"])
        mats = [_weight(gen, I, H), _weight(gen, I, H), _weight(gen, H, I)]
        return dict(op=op, x=x, w=[m[0] for m in mats], ws=[m[1] for m in mats],
                    out=torch.empty((c["M"], H), dtype=TYPES[c["out"]], device="cuda"), work=None)
    x = _rows(gen, c["T"], H, c["x"])
    n = c["n"]
    wr = torch.randn((c["E"], H), generator=gen, device="cuda") * (1.0 / math.sqrt(H))
    bias = 0.05 * torch.randn(c["E"], generator=gen, device="cuda")
    mats = [_weight(gen, n, I, H), _weight(gen, n, I, H), _weight(gen, n, H, I)]
    sh = [_weight(gen, I, H), _weight(gen, I, H), _weight(gen, H, I)] if c["shared"] else None
    return dict(op=op, x=x, wr=wr, bias=bias, w=[m[0] for m in mats], ws=[m[1] for m in mats],
                shared=[t for t, _ in sh] + [t for _, t in sh] if sh else None, lo=c["lo"], topk=c["topk"], scale=2.5,
                sel=torch.empty((c["T"], c["topk"]), dtype=torch.int64, device="cuda"),
                rw=torch.empty((c["T"], c["topk"]), device="cuda"),
                out=torch.empty((c["T"], H), dtype=TYPES[c["out"]], device="cuda"), work=None)


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    s, op = state, state["op"]
    if own:
        from hecate_amd import i8, moe8
        out = s["out"]
        if op == "matmul":
            i8.matmul(s["q"], s["qs"], s["w"], s["ws"], out, s["b"])
            return out
        x = s["x"]
        if op == "linear":
            if s["work"] is None:
                s["work"] = i8.linear_work(x.device, x.shape[0], *s["w"].shape)
            i8.linear(x, s["w"], s["ws"], out, s["work"], s["b"])
            return out
        if op == "mlp":
            if s["work"] is None:
                s["work"] = i8.mlp_work(x.device, x.shape[0], x.shape[1], s["w"][0].shape[0])
            i8.mlp(x, *s["w"], *s["ws"], out, s["work"])
            return out
        if s["work"] is None:
            s["work"] = moe8.layer_work(x.device, x.shape[0], x.shape[1], s["w"][0].shape[1], s["wr"].shape[0], s["topk"])
        moe8.layer(x, s["wr"], s["bias"], *s["w"], *s["ws"], s["sel"], s["rw"], out, s["work"], s["scale"], s["lo"], s["shared"])
        return out, s["sel"], s["rw"]
    if op in ("matmul", "linear"):
        q, sc = _quantize(s["x"]) if op == "linear" else (s["q"].float(), s["qs"][:, None])
        y = (q @ s["w"].float().t()) * sc * s["ws"]
        return (y if s["b"] is None else y + s["b"]).to(s["out"].dtype)
    if op == "mlp":
        return _mlp(*_quantize(s["x"]), *s["w"], *s["ws"]).to(s["out"].dtype)
    return _layer(s)


def _quantize(x):
    """the whole numbers (as fp32) and scales of the rows. 127 x has at most 18 bits for a 16-bit x, so its 32-bit quotient is a
    half exactly where the true one is; 32-bit rows are divided in 64 bits"""
    t = x.double() if x.dtype == torch.float32 else x.float()
    a = t.abs().amax(-1, keepdim=True)
    q = torch.round(t * 127.0 / torch.where(a > 0, a, torch.ones_like(a)))
    return q.float(), a.float() / 127.0


def _mlp(q, sc, wg, wu, wd, sg, su, sd):
    """q [..., M, H] whole numbers with row scales through one expert's weights, or one expert's for each leading index"""
    g = (q @ wg.float().transpose(-1, -2)) * sc * sg.unsqueeze(-2)
    u = (q @ wu.float().transpose(-1, -2)) * sc * su.unsqueeze(-2)
    p, sp = _quantize_h(g * torch.sigmoid(g) * u)
    return (p @ wd.float().transpose(-1, -2)) * sp * sd.unsqueeze(-2)


def _quantize_h(h):
    a = h.abs().amax(-1, keepdim=True)
    return torch.round(h * 127.0 / torch.where(a > 0, a, torch.ones_like(a))), a / 127.0


def _layer(s):
    x, k, n = s["x"], s["topk"], s["w"][0].shape[0]
    T = x.shape[0]
    a = torch.sigmoid(x.double() @ s["wr"].double().t())       # (scores next to each other decide the selection)
    sel = torch.sort(a + s["bias"].double(), dim=-1, descending=True, stable=True).indices[:, :k]
    top = a.gather(1, sel)
    rw = (s["scale"] * top / (top.sum(-1, keepdim=True) + 1e-20)).float()
    at = sel - s["lo"]
    here = (at >= 0) & (at < n)
    e = torch.where(here, at, torch.zeros_like(at)).reshape(-1)
    q, sc = _quantize(x)
    pick = lambda t: t[:, None].expand(T, k, t.shape[1]).reshape(T * k, 1, t.shape[1])
    d = _mlp(pick(q), pick(sc), *(m[e] for m in s["w"]), *(m[e] for m in s["ws"])).reshape(T, k, -1)
    y = (d * torch.where(here, rw, torch.zeros_like(rw))[..., None]).sum(1)
    if s["shared"] is not None:
        y = y + _mlp(q, sc, *s["shared"])
    return y.to(s["out"].dtype), sel, rw


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("matmul", "linear"):
        y = _product(s["x"], s["w"], s["ws"]) if op == "linear" else (
            torch.einsum("mk,nk->mn", s["q"].double(), s["w"].double()) * torch.outer(s["qs"].double(), s["ws"].double()))
        return y if s["b"] is None else y + s["b"].double()
    if op == "mlp":
        return _expert(s["x"], *s["w"], *s["ws"])
    x, k, lo = s["x"], s["topk"], s["lo"]
    score = 1.0 / (1.0 + torch.exp(-torch.einsum("th,eh->te", x.double(), s["wr"].double())))
    key = score + s["bias"].double()
    y = torch.zeros((x.shape[0], x.shape[1]), dtype=torch.float64, device=x.device)
    sel = torch.empty_like(s["sel"])
    rw = torch.empty(s["rw"].shape, dtype=torch.float64, device=x.device)
    for t in range(x.shape[0]):
        left = key[t].clone()
        for j in range(k):                                       # the largest left, of equal ones the first
            i = int((left == left.max()).nonzero()[0])
            sel[t, j] = i
            left[i] = -math.inf
        rw[t] = s["scale"] * score[t, sel[t]] / (score[t, sel[t]].sum() + 1e-20)
        for j in range(k):
            i = int(sel[t, j]) - lo
            if 0 <= i < s["w"][0].shape[0]:
                y[t] += rw[t, j] * _expert(x[t:t + 1], *(m[i] for m in s["w"]), *(m[i] for m in s["ws"]))[0]
    if s["shared"] is not None:
        y += _expert(x, *s["shared"])
    return y, sel, rw


def _levels(x):
    """whole numbers rounded half to even, and the rows' largest magnitudes"""
    x = x.double()
    a = torch.linalg.vector_norm(x, ord=math.inf, dim=-1, keepdim=True)
    v = 127.0 * x / a.clamp(min=1e-300)
    f = torch.floor(v)
    r = v - f
    up = (r > 0.5) | ((r == 0.5) & (torch.remainder(f, 2.0) == 1.0))
    return f + up.double(), a


def _product(x, w, ws):
    q, a = _levels(x)
    return torch.einsum("mk,nk->mn", q, w.double()) * (a / 127.0) * ws.double()[None, :]


def _expert(x, wg, wu, wd, sg, su, sd):
    g = _product(x, wg, sg)
    return _product(g / (1.0 + torch.exp(-g)) * _product(x, wu, su), wd, sd)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op in ("matmul", "linear"):
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": M * (K * SIZE[c["x"]] if op == "linear" else K + 4) + N * (K + 4 + 4 * c["bias"]) + M * N * SIZE[c["out"]], "flops": 2 * M * N * K}
    H, I = c["H"], c["I"]
    expert = 3 * H * I + 4 * (2 * I + H)
    if op == "mlp":
        return {"bytes": expert + c["M"] * H * (SIZE[c["x"]] + SIZE[c["out"]]), "flops": 6 * c["M"] * H * I}
    T, E, n, k = c["T"], c["E"], c["n"], c["topk"]
    distinct = n * (1.0 - (1.0 - k / E) ** T)                   # as expected of even routing
    rows = T * H * (SIZE[c["x"]] + SIZE[c["out"]]) + 12 * T * k
    return {"bytes": (distinct + c["shared"]) * expert + 4 * E * (H + 1) + rows,
            "flops": 6 * T * (k * n / E + c["shared"]) * H * I + 2 * T * E * H}
