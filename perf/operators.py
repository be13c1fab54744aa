"""The operators of 4-bit weights and 8-bit rows: cases, inputs, and their plain forms.

Blocks of 32 values along a row share a scale 2^(b - 127), b a byte. Weights are e2m1 (two to a byte, the first in the low
half), rows of activations e4m3. The scale of a block is the smallest power of two with which its largest magnitude is at
most the format's largest value (6 and 448)."""
import math

import torch

own = False

BLOCK = 32
DEV = "cuda:0"
EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence's token through the output projection of a layer 4,096 wide: the smallest call of a decode step
        {"name": "product 1x4096x4096", "op": "product", "rows": 1, "n": 4096, "k": 4096, "glu": False, "wide": True},
        # the same token through the gated pair of a feed-forward of 14,336
        {"name": "gated 1x14336x4096", "op": "product", "rows": 1, "n": 14336, "k": 4096, "glu": True, "wide": False},
        # eight sequences through its down projection: a long k
        {"name": "product 8x4096x14336", "op": "product", "rows": 8, "n": 4096, "k": 14336, "glu": False, "wide": True},
        # a larger batch, widths off every tile
        {"name": "product 37x1999x5472", "op": "product", "rows": 37, "n": 1999, "k": 5472, "glu": False, "wide": False},
        # eight sequences' 8-bit rows through the qkv projection
        {"name": "product8 8x6144x4096", "op": "product8", "rows": 8, "n": 6144, "k": 4096},
        # a prompt's 8-bit rows through a narrow layer, rows and columns off every tile
        {"name": "product8 1021x1376x2080", "op": "product8", "rows": 1021, "n": 1376, "k": 2080},
        # an ordinary prompt through the down projection
        {"name": "product8 512x4096x14336", "op": "product8", "rows": 512, "n": 4096, "k": 14336},
        # several prompts in one step through gates and ups: the largest
        {"name": "product8 4096x28672x4096", "op": "product8", "rows": 4096, "n": 28672, "k": 4096},
        # a decode step's norm
        {"name": "norm 8x4096", "op": "norm", "rows": 8, "n": 4096, "bias": False, "wide": True},
        # a prompt's norm at a width of 8,192
        {"name": "norm 2048x8192", "op": "norm", "rows": 2048, "n": 8192, "bias": True, "wide": False},
        # the activation of a decode step
        {"name": "swiglu 8x14336", "op": "swiglu", "rows": 8, "n": 14336},
        # and of several prompts
        {"name": "swiglu 4096x14336", "op": "swiglu", "rows": 4096, "n": 14336},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("product", "product", "product8", "product8", "norm", "swiglu"))
    if op == "product":
        rows, glu = _log(rng, 1, 64), rng.random() < 0.4
        n = _log(rng, 48, 14336 if glu else 28672)
        k = BLOCK * _log(rng, 2, 512)
        while n * k * (2 if glu else 1) > 28672 * 4096:
            k = BLOCK * max(2, k // (2 * BLOCK))
        return {"op": op, "rows": rows, "n": n, "k": k, "glu": glu, "wide": not glu and rng.random() < 0.5}
    if op == "product8":
        rows, n, k = _log(rng, 1, 4096), _log(rng, 48, 28672), BLOCK * _log(rng, 2, 512)
        while n * k > 28672 * 4096 or rows * n * k > 4096 * 28672 * 4096:
            k = BLOCK * max(2, k // (2 * BLOCK))
        return {"op": op, "rows": rows, "n": n, "k": k}
    rows, n = _log(rng, 1, 4096), BLOCK * _log(rng, 2, 448 if op == "swiglu" else 512)
    if op == "norm":
        return {"op": op, "rows": rows, "n": n, "bias": rng.random() < 0.5, "wide": rng.random() < 0.5}
    return {"op": op, "rows": rows, "n": n}


def work(case):
    r, n = case["rows"], case["n"]
    if case["op"] == "product":
        columns, k = n * (2 if case["glu"] else 1), case["k"]
        return {"bytes": columns * k * (1 / 2 + 1 / 32) + r * k * 2 + r * n * (4 if case["wide"] else 2), "flops": 2 * r * columns * k}
    if case["op"] == "product8":
        k = case["k"]
        return {"bytes": n * k * (1 / 2 + 1 / 32) + r * k * (1 + 1 / 32) + r * n * 2, "flops": 2 * r * n * k}
    if case["op"] == "norm":                 # the stream read and written, what joins it, the rows
        return {"bytes": r * n * (8 + (4 if case["wide"] else 2) + 1 + 1 / 32) + 4 * n, "flops": 6 * r * n}
    return {"bytes": r * n * (4 + 1 + 1 / 32), "flops": 6 * r * n}


# ------------------------------------------------------------------ inputs
def _scale_bytes(blocks, largest):
    """Byte of the smallest power of two s with max|block| <= largest * s, largest = 1.5 * 4 or 1.75 * 256."""
    m, e = torch.frexp(blocks.abs().amax(-1))              # max = m 2^e, m in [0.5, 1); 0: m = e = 0
    top_m, top_e = math.frexp(largest)
    e = e.to(torch.int32) - top_e + (m > top_m).to(torch.int32)
    return torch.where(m == 0, torch.zeros_like(e), (e + 127).clamp(0, 254)).to(torch.uint8)


def _weights(n, k, g):
    """(codes [n, k/2], scales [n, k/32]) of a matrix of normal weights, as a file of such weights holds them."""
    w = torch.empty(n, k, device=DEV).normal_(0.0, 0.02, generator=g).view(n, k // BLOCK, BLOCK)
    b = _scale_bytes(w, 6.0)
    w = torch.ldexp(w, 127 - b.to(torch.int32).unsqueeze(-1)).view(n, k)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    code = torch.bucketize(w.abs(), edges).to(torch.uint8) | (w < 0).to(torch.uint8) << 3
    return code[:, 0::2] | code[:, 1::2] << 4, b


def _rows8(r, k, g):
    """(e4m3 [r, k], scales [r, k/32]) of normed rows with some columns larger than the rest."""
    x = torch.empty(r, k, device=DEV).normal_(generator=g) * torch.empty(k, device=DEV).normal_(generator=g).mul_(0.5).exp_()
    b = _scale_bytes(x.view(r, k // BLOCK, BLOCK), 448.0)
    x = torch.ldexp(x.view(r, k // BLOCK, BLOCK), 127 - b.to(torch.int32).unsqueeze(-1)).view(r, k)
    return x.to(torch.float8_e4m3fn), b


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r, n, s = case["rows"], case["n"], {"case": case}
    if case["op"] in ("product", "product8"):
        k = case["k"]
        s["codes"], s["scales"] = _weights(n * (2 if case.get("glu") else 1), k, g)
        if case["op"] == "product":
            x = torch.empty(r, k, device=DEV).normal_(generator=g) * torch.empty(k, device=DEV).normal_(generator=g).mul_(0.5).exp_()
            s["x"] = x.to(torch.bfloat16)
            s["out"] = torch.empty(r, n, device=DEV, dtype=torch.float32 if case["wide"] else torch.bfloat16)
        else:
            s["x"], s["xs"] = _rows8(r, k, g)
            s["out"] = torch.empty(r, n, device=DEV, dtype=torch.bfloat16)
        return s
    s["rows"] = torch.empty(r, n, device=DEV, dtype=torch.float8_e4m3fn)
    s["bytes"] = torch.empty(r, n // BLOCK, device=DEV, dtype=torch.uint8)
    if case["op"] == "norm":
        s["x"] = torch.empty(r, n, device=DEV).normal_(0.0, 2.0, generator=g)
        s["delta"] = torch.empty(r, n, device=DEV).normal_(generator=g).to(torch.float32 if case["wide"] else torch.bfloat16)
        s["bias"] = torch.empty(n, device=DEV).normal_(0.0, 0.1, generator=g) if case["bias"] else None
        s["weight"] = torch.empty(n, device=DEV).normal_(1.0, 0.1, generator=g)
        s["stream"] = torch.empty(r, n, device=DEV)
    else:
        s["gate_up"] = torch.empty(r, 2 * n, device=DEV).normal_(generator=g).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _weights32(codes, scales):
    n, half = codes.shape
    code = torch.stack((codes & 15, codes >> 4), -1).view(n, 2 * half)
    e, m = (code >> 1 & 3).to(torch.int32), (code & 1).to(torch.float32)
    mag = torch.where(e == 0, m * 0.5, torch.ldexp(1.0 + m * 0.5, (e - 1).clamp(min=0)))
    w = torch.where(code >= 8, -mag, mag).view(n, -1, BLOCK)
    return torch.ldexp(w, scales.to(torch.int32).unsqueeze(-1) - 127).view(n, 2 * half)


def _rows32(x, b):
    r, k = x.shape
    return torch.ldexp(x.to(torch.float32).view(r, -1, BLOCK), b.to(torch.int32).unsqueeze(-1) - 127).view(r, k)


def _silu32(g, u):
    return g / (1.0 + torch.exp(-g)) * u


def _packed32(y):
    r, n = y.shape
    y = y.view(r, n // BLOCK, BLOCK)
    b = _scale_bytes(y, 448.0)
    return torch.ldexp(y, 127 - b.to(torch.int32).unsqueeze(-1)).view(r, n).to(torch.float8_e4m3fn), b


def run(s):
    case = s["case"]
    if case["op"] == "product":
        if own:
            from transformer_amd import kernels
            return kernels.gemm_mx4(s["x"], kernels.Mx4(s["codes"], s["scales"]), s["out"], swiglu=case["glu"])
        y = s["x"].to(torch.float32) @ _weights32(s["codes"], s["scales"]).t()
        if case["glu"]:
            y = _silu32(y[:, :case["n"]], y[:, case["n"]:])
        return y.to(s["out"].dtype)
    if case["op"] == "product8":
        if own:
            from transformer_amd import kernels
            return kernels.gemm_mx4(kernels.Mx8(s["x"], s["xs"]), kernels.Mx4(s["codes"], s["scales"]), s["out"])
        return (_rows32(s["x"], s["xs"]) @ _weights32(s["codes"], s["scales"]).t()).to(torch.bfloat16)
    if case["op"] == "norm":
        if own:
            from transformer_amd import kernels
            kernels.add_rmsnorm_mx8(s["x"], s["weight"], EPS, kernels.Mx8(s["rows"], s["bytes"]), s["delta"], s["bias"],
                                    stream=s["stream"])
            return {"stream": s["stream"], "rows": s["rows"], "scales": s["bytes"].view(torch.float8_e8m0fnu)}
        v = s["x"] + s["delta"].to(torch.float32)
        if s["bias"] is not None:
            v = v + s["bias"]
        y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["weight"]
        rows, b = _packed32(y)
        return {"stream": v, "rows": rows, "scales": b.view(torch.float8_e8m0fnu)}
    if own:
        from transformer_amd import kernels
        kernels.swiglu_mx8(s["gate_up"], kernels.Mx8(s["rows"], s["bytes"]))
        return {"rows": s["rows"], "scales": s["bytes"].view(torch.float8_e8m0fnu)}
    gu = s["gate_up"].to(torch.float32)
    rows, b = _packed32(_silu32(gu[:, :case["n"]], gu[:, case["n"]:]))
    return {"rows": rows, "scales": b.view(torch.float8_e8m0fnu)}


# ------------------------------------------------------------------ the definitions, in 64 bits
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _weights64(codes, scales):
    table = torch.tensor([v for v in _E2M1] + [-v for v in _E2M1], dtype=torch.float64, device=codes.device)
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2] = table[(codes % 16).long()]
    w[:, 1::2] = table[(codes // 16).long()]
    return w * torch.exp2(scales.double() - 127.0).repeat_interleave(BLOCK, 1)


def _packed64(y):
    """(e4m3 values of the rows over their scales, scales), both float64."""
    top = y.unflatten(1, (-1, BLOCK)).abs().amax(-1)
    e = torch.ceil(torch.log2(top / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e))   # log2's last bit
    scale = torch.exp2(e.clamp(-127, 127))
    v = y / scale.repeat_interleave(BLOCK, 1)
    _, ve = torch.frexp(v)
    step = torch.exp2((ve - 1).clamp(min=-6).double() - 3.0)
    return torch.round(v / step) * step, scale


def exact(case, seed):
    s = prepare(case, seed)
    n = case["n"]
    if case["op"] in ("product", "product8"):
        x = s["x"].double()
        if case["op"] == "product8":
            x = x * torch.exp2(s["xs"].double() - 127.0).repeat_interleave(BLOCK, 1)
        y = x @ _weights64(s["codes"], s["scales"]).t()
        if case.get("glu"):
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        return y
    if case["op"] == "norm":
        v = s["x"].double() + s["delta"].double() + (0.0 if s["bias"] is None else s["bias"].double())
        rows, scale = _packed64(v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / n + EPS) * s["weight"].double())
        return {"stream": v, "rows": rows, "scales": scale}
    gate, up = s["gate_up"].double().split(n, -1)
    rows, scale = _packed64(gate * torch.sigmoid(gate) * up)
    return {"rows": rows, "scales": scale}
