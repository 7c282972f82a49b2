"""What the 8-bit linear layer's operators are measured on: rows rounded to 8 bits (b200_quantize_i8), the
root-mean-square norm with the residual's addition and an 8-bit result (b200_rms_norm_i8), and the 8-bit
integer product with token and channel scales (b200_gemm_i8).

`run` computes an operator in its plain form, or with `own` set through the framework's entry points."""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"bf16": 13, "f16": 10, "f32": 11}
MOST_ELEMENTS = 8192 * 8192
MOST_MACS = 8192 ** 3


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the attention's output of an 8 x 1024 token batch at width 768, before its projection
        {"name": "quantize_prompt", "op": "quantize", "rows": 8192, "cols": 768, "type": "bf16", "pad": 0},
        # an f32 LM head laid out in 8 bits, one scale per vocabulary entry
        {"name": "quantize_head", "op": "quantize", "rows": 50257, "cols": 768, "type": "f32", "pad": 0},
        # one decoded token at width 768: latency
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 768, "type": "bf16", "wtype": "f32", "residual": True, "pad": 0},
        # a ragged batch of an odd width whose rows start at odd addresses
        {"name": "norm_odd", "op": "norm", "rows": 333, "cols": 1003, "type": "f16", "wtype": "f16", "residual": True, "pad": 2},
        # the 8 x 1024 token batch at width 768
        {"name": "norm_prompt", "op": "norm", "rows": 8192, "cols": 768, "type": "bf16", "wtype": "bf16", "residual": True, "pad": 0},
        # a long prompt of a wide model
        {"name": "norm_wide", "op": "norm", "rows": 8192, "cols": 8192, "type": "bf16", "wtype": "bf16", "residual": True, "pad": 0},
        # one decoded token, width 768 to its queries, keys and values: latency
        {"name": "gemm_token", "op": "gemm", "M": 1, "N": 2304, "K": 768, "type": "bf16", "bias": True, "gelu": False, "pad": 0},
        # 32 sequences decoding together through a wide layer: the weights' bytes
        {"name": "gemm_decode", "op": "gemm", "M": 32, "N": 8192, "K": 4096, "type": "bf16", "bias": False, "gelu": False, "pad": 0},
        # odd in every direction, rows not 16-byte aligned, f32 result
        {"name": "gemm_ragged", "op": "gemm", "M": 211, "N": 1003, "K": 999, "type": "f32", "bias": True, "gelu": False, "pad": 0},
        # a short prompt into a wide hidden layer with its activation
        {"name": "gemm_gelu", "op": "gemm", "M": 1024, "N": 4096, "K": 1024, "type": "f16", "bias": True, "gelu": True, "pad": 0},
        # the 8 x 1024 token batch, width 768 to its queries, keys and values
        {"name": "gemm_prompt", "op": "gemm", "M": 8192, "N": 2304, "K": 768, "type": "bf16", "bias": True, "gelu": False, "pad": 0},
        # the largest product of the framework's sweep
        {"name": "gemm_large", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "type": "bf16", "bias": False, "gelu": False, "pad": 0},
    ]


def _spread(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; half of them round (a multiple of 64), the rest any."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 64:
        n = (n + 32) // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gemm", "gemm"])
    pad = rng.choice([0, 0, 0, 16, 1])
    if op == "gemm":
        m, n, k = _spread(rng, 1, 8192), _spread(rng, 16, 32768), _spread(rng, 16, 16384)
        k = max(16, min(k, MOST_MACS // (m * n)))
        return {"op": "gemm", "M": m, "N": n, "K": k, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.5,
                "gelu": rng.random() < 0.25, "pad": pad}
    rows, cols = _spread(rng, 1, 65536), _spread(rng, 16, 16384)
    rows = max(1, min(rows, MOST_ELEMENTS // cols))
    case = {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "pad": pad}
    if op == "norm":
        case["wtype"] = rng.choice([case["type"], "f32"])
        case["residual"] = rng.random() < 0.75
    return case


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["M"], case["N"], case["K"]
        out = 4 if case["type"] == "f32" else 2
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + m * n * out, "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "quantize":
        return {"bytes": rows * cols * (size + 1) + 4 * rows, "flops": 3 * rows * cols}
    wsize = 4 if case["wtype"] == "f32" else 2
    streams = 3 if case["residual"] else 2  # x, residual, h
    return {"bytes": rows * cols * (streams * size + 1) + 4 * rows + wsize * cols, "flops": 8 * rows * cols}


# ------------------------------------------------------------------------------------------ the inputs
def _rows(rows, cols, pad, dtype):
    """An empty [rows, cols] whose rows lie cols + pad elements apart."""
    return torch.empty(rows, cols + pad, device="cuda", dtype=dtype)[:, :cols]


def _activations(g, rows, cols, dtype, pad):
    """Activations as a transformer has them: a few channels far larger than the rest."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    out = _rows(rows, cols, pad, dtype)
    out.copy_(x)
    return out


def _int8(g, rows, cols, pad, outliers):
    """Rows in 8 bits with a scale each, as quantising normal values gives them."""
    out, scale = _rows(rows, cols, pad, torch.int8), torch.empty(rows, device="cuda")
    step = max(1, (1 << 26) // max(1, cols))
    for at in range(0, rows, step):
        x = torch.randn(min(step, rows - at), cols, device="cuda", generator=g)
        if outliers:
            x[:, ::97] *= 5.0
        top = x.abs().amax(1).clamp_min_(1e-6)
        out[at:at + step] = (x * (127.0 / top)[:, None]).round_().clamp_(-127, 127).to(torch.int8)
        scale[at:at + step] = top / 127.0
    return out, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "gemm":
        m, n, k, pad = case["M"], case["N"], case["K"], case["pad"]
        s["a"], s["a_scale"] = _int8(g, m, k, pad, True)
        s["b"], s["b_scale"] = _int8(g, n, k, pad, False)
        s["b_scale"] *= 1.0 / math.sqrt(k)
        s["bias_values"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        s["c"] = torch.empty(m, n, device="cuda", dtype=TYPES[case["type"]])
        # room for 16-byte aligned copies of both operands: a program keeps one such workspace
        s["scratch"] = torch.empty(m * (k + 16) + n * (k + 16) + 512, device="cuda", dtype=torch.uint8)
        return s
    rows, cols, dtype, pad = case["rows"], case["cols"], TYPES[case["type"]], case["pad"]
    s["x"] = _activations(g, rows, cols, dtype, pad)
    s["q"] = torch.empty(rows, cols, device="cuda", dtype=torch.int8)
    s["scale"] = torch.empty(rows, device="cuda")
    if case["op"] == "norm":
        s["r"] = _activations(g, rows, cols, dtype, pad) if case["residual"] else None
        s["h"] = torch.empty(rows, cols, device="cuda", dtype=dtype) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(TYPES[case["wtype"]])
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _round_rows(t):
    """[rows, cols] f32 to 8 bits: the values and their rows' largest magnitudes.  The division is in 64
    bits, where a quotient next to a border between two values stays on its side."""
    top = t.abs().amax(1)
    q = (t.double() * 127.0 / top.double().clamp_min(1e-300)[:, None]).round().to(torch.int8)
    return q, top


def _plain(s):
    if s["op"] == "gemm":
        c = s["a"].float() @ s["b"].float().t()
        c = c * s["a_scale"][:, None] * s["b_scale"][None, :]
        if s["bias"]:
            c = c + s["bias_values"]
        if s["gelu"]:
            c = 0.5 * c * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (c + 0.044715 * c * c * c)))
        return {"c": c.to(TYPES[s["type"]])}
    x = s["x"].float()
    if s["op"] == "quantize":
        q, top = _round_rows(x)
        return {"q": q, "scale": top / 127.0}
    out = {}
    if s["residual"]:
        out["h"] = (x + s["r"].float()).to(s["x"].dtype)
        x = out["h"].float()
    rstd = torch.rsqrt(x.square().mean(1) + EPS)
    out["q"], top = _round_rows(x * s["w"].float())
    out["scale"] = top / 127.0 * rstd
    return out


# ------------------------------------------------------------------------------------------ the framework's calls
_kernels = None


def _own(s):
    global _kernels
    if _kernels is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "mccl-jax_b200"))
        from pjrt_b200 import kernels
        _kernels = kernels.Kernels()
    k, stream = _kernels, torch.cuda.current_stream().cuda_stream
    if s["op"] == "gemm":
        a, b, c, bias, scratch = s["a"], s["b"], s["c"], s["bias_values"], s["scratch"]
        k.gemm_i8(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), s["a_scale"].data_ptr(), s["b_scale"].data_ptr(),
                  bias.data_ptr() if bias is not None else None, c.data_ptr(), c.stride(0), s["M"], s["N"], s["K"], CODES[s["type"]],
                  1 if s["gelu"] else 0, scratch.data_ptr(), scratch.numel(), stream)
        return {"c": c}
    x, q, scale = s["x"], s["q"], s["scale"]
    if s["op"] == "quantize":
        k.quantize_i8(x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), s["rows"], s["cols"], CODES[s["type"]], stream)
        return {"q": q, "scale": scale}
    r, h = s["r"], s["h"]
    k.rms_norm_i8(x.data_ptr(), x.stride(0), r.data_ptr() if r is not None else None, r.stride(0) if r is not None else 0,
                  s["w"].data_ptr(), h.data_ptr() if h is not None else None, h.stride(0) if h is not None else 0, q.data_ptr(), q.stride(0),
                  scale.data_ptr(), s["rows"], s["cols"], CODES[s["type"]], CODES[s["wtype"]], EPS, stream)
    return {"h": h, "q": q, "scale": scale} if r is not None else {"q": q, "scale": scale}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "gemm":
        c = torch.empty(case["M"], case["N"], device="cuda", dtype=torch.float64)
        b = s["b"].double()
        step = max(1, (1 << 27) // case["K"])
        for at in range(0, case["M"], step):  # the sums of integers below 2^53 are exact
            torch.mm(s["a"][at:at + step].double(), b.t(), out=c[at:at + step])
        c *= s["a_scale"].double()[:, None]
        c *= s["b_scale"].double()
        if case["bias"]:
            c += s["bias_values"].double()
        if case["gelu"]:
            c = c / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (c + 0.044715 * c ** 3)))
        return {"c": c}
    h, out = s["x"].double(), {}
    weight = 1.0
    if case["op"] == "norm":
        if case["residual"]:
            h = h + s["r"].double()
            out["h"] = h
            h = h.to(TYPES[case["type"]]).double()  # the norm reads the sum as it is stored
        weight = s["w"].double()
    t = h * weight
    out["q"] = None
    out["scale"] = t.abs().max(dim=1).values / 127.0
    if case["op"] == "norm":
        out["scale"] = out["scale"] / ((h * h).sum(1) / case["cols"] + EPS).sqrt()
    return out
