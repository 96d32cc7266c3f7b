"""Cases of the 8-bit integer operators of the inference path: what is measured, its plain form and its exact result.

Operators (harp_b200.ops.functional):

  rmsnorm_mod_quant   h = residual + gate*x;  y = rms(h)*w*(1+scale) + shift;  y in 8 bits with a scale for each row
  swiglu_quant        y = silu(g)*u of [g | u];  y in 8 bits with a scale for each row
  quant_rows          x in 8 bits with a scale for each row (activations by token, weights by output channel)
  gemm_s8             (a b^T) in 8-bit integers with a scale for each row of a and of b, plus bias

Rows in 8 bits: s = max(max|y| / 127, smallest normal fp32 number), q = y / s rounded half to even.  A run returns the
values q * s in bf16 beside s, and what else the operator writes.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
TINY = 2.0 ** -126

# DiT-XL/2 at 1024 px: 4096 image + 256 text tokens, batch 4; hidden 1152, SwiGLU width 4608.
# mmdit-2b: hidden 2304, SwiGLU width 6144.


def listed():
    return [
        # the norm between attention and MLP of every DiT-XL/2 block: gated residual, modulation, batch 4 at 1024 px
        {"name": "norm-dit-xl2", "op": "norm", "dtype": "bf16", "batch": 4, "rows": 4352, "cols": 1152,
         "residual": True, "gate": True, "mod": True, "weight": False},
        # an fp32 stream with an odd width and a learned weight, no residual (a text encoder's output, ragged length)
        {"name": "norm-fp32-odd", "op": "norm", "dtype": "fp32", "batch": 1, "rows": 1061, "cols": 1155,
         "residual": False, "gate": False, "mod": False, "weight": True},
        # one token of mmdit-2b's width: latency
        {"name": "norm-one-token", "op": "norm", "dtype": "bf16", "batch": 1, "rows": 1, "cols": 2304,
         "residual": True, "gate": False, "mod": False, "weight": True},
        # the activation between W1|W3 and W2 of a DiT-XL/2 block, batch 4 at 1024 px
        {"name": "swiglu-dit-xl2", "op": "swiglu", "dtype": "bf16", "batch": 4, "rows": 4352, "cols": 4608},
        # the same of a prompt of 77 tokens in fp32, odd width
        {"name": "swiglu-prompt-odd", "op": "swiglu", "dtype": "fp32", "batch": 1, "rows": 77, "cols": 1001},
        # the attention output before its projection, batch 4 at 1024 px
        {"name": "rows-attention-out", "op": "rows", "dtype": "bf16", "batch": 4, "rows": 4352, "cols": 1152},
        # the adaLN input: one conditioning vector for each of 3 samples
        {"name": "rows-conditioning", "op": "rows", "dtype": "fp32", "batch": 1, "rows": 3, "cols": 2304},
        # W1|W3 of a DiT-XL/2 block: the largest product, batch 4 at 1024 px
        {"name": "gemm-w13", "op": "gemm", "out": "bf16", "m": 17408, "n": 9216, "k": 1152, "bias": False},
        # W2 of the same block: narrow output, long sum
        {"name": "gemm-w2", "op": "gemm", "out": "bf16", "m": 17408, "n": 1152, "k": 4608, "bias": True},
        # QKV of a small image with its prompt (288 tokens)
        {"name": "gemm-qkv-small", "op": "gemm", "out": "bf16", "m": 288, "n": 3456, "k": 1152, "bias": True},
        # the adaLN modulation of 4 samples: few rows, the weights are what is read
        {"name": "gemm-adaln", "op": "gemm", "out": "bf16", "m": 4, "n": 6912, "k": 1152, "bias": True},
        # odd sizes in every direction, fp32 output
        {"name": "gemm-odd-fp32", "op": "gemm", "out": "fp32", "m": 1061, "n": 1003, "k": 1155, "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "rows", "gemm"])
    if op == "gemm":
        case = {"op": op, "out": rng.choice(["bf16", "bf16", "fp32"]), "m": _log(rng, 1, 17408), "n": _log(rng, 24, 9216),
                "k": _log(rng, 32, 6144), "bias": rng.random() < 0.5}
        if rng.random() < 0.6:  # the widths of most models are multiples of 64
            case["n"], case["k"] = max(64, case["n"] // 64 * 64), max(64, case["k"] // 64 * 64)
        most = 17408 * 9216 * 1152
        if case["m"] * case["n"] * case["k"] > most:
            case["m"] = max(1, most // (case["n"] * case["k"]))
        return case
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp32"]), "batch": rng.choice([1, 1, 2, 4]),
            "cols": _log(rng, 48, 6144)}
    if rng.random() < 0.6:
        case["cols"] = max(64, case["cols"] // 64 * 64)
    most = 17408 * (4608 if op == "swiglu" else 1152) // (2 if case["dtype"] == "fp32" else 1)
    case["rows"] = _log(rng, 1, max(1, min(17408, most // case["cols"]) // case["batch"]))
    if op == "norm":
        case["residual"] = rng.random() < 0.6
        case["gate"] = case["residual"] and rng.random() < 0.6
        case["mod"] = rng.random() < 0.6
        case["weight"] = rng.random() < 0.5
    return case


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _activations(g, rows, cols, dtype):
    """Rows of different size with a few large channels, as residual streams have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.1 * torch.randn(rows, 1, generator=g, device="cuda"))
    c = torch.exp(0.2 * torch.randn(1, cols, generator=g, device="cuda"))
    c[:, torch.randint(0, cols, (max(1, cols // 512),), generator=g, device="cuda")] *= 3.0
    return (x * c).to(dtype)


def _int8(g, rows, cols):
    """8-bit rows as the quantisers give them: bell-shaped, row stride a multiple of 16 bytes."""
    ld = -(-cols // 16) * 16
    q = torch.empty(rows, ld, dtype=torch.int8, device="cuda")
    q.copy_((torch.randn(rows, ld, generator=g, device="cuda") * 34.0).round_().clamp_(-127, 127))
    return q[:, :cols]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        s = {"op": op, "out": DTYPES[case["out"]], "a": _int8(g, m, k), "b": _int8(g, n, k),
             "sa": torch.rand(m, generator=g, device="cuda") * 0.05 + 0.005,
             "sb": torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-4, "bias": None}
        if case["bias"]:
            s["bias"] = (torch.randn(n, generator=g, device="cuda") * 0.1).to(torch.bfloat16)
        return s
    dt, b, r, d = DTYPES[case["dtype"]], case["batch"], case["rows"], case["cols"]
    if op == "swiglu":
        return {"op": op, "gu": _activations(g, b * r, 2 * d, dt), "cols": d}
    if op == "rows":
        return {"op": op, "x": _activations(g, b * r, d, dt)}
    s = {"op": op, "x": _activations(g, b * r, d, dt), "rows": r, "eps": 1e-6, "residual": None, "gate": None,
         "scale": None, "shift": None, "w": None}
    if case["residual"]:
        s["residual"] = _activations(g, b * r, d, dt)
    # the modulation is one product's output [batch, 6 * cols], as the blocks have it: its parts are strided views
    mod = (torch.randn(b, 6 * d, generator=g, device="cuda") * 0.3).to(dt)
    if case["gate"]:
        s["gate"] = mod[:, 2 * d:3 * d]
    if case["mod"]:
        s["shift"], s["scale"] = mod[:, 3 * d:4 * d], mod[:, 4 * d:5 * d]
    if case["weight"]:
        s["w"] = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
    return s


def _rows8(y):
    s = (y.abs().amax(1) * (1.0 / 127.0)).clamp_min(TINY)
    q = torch.round(y * (1.0 / s)[:, None]).clamp(-127, 127)
    return (q * s[:, None]).to(torch.bfloat16), s


def _plain(s):
    op = s["op"]
    if op == "gemm":
        y = (s["a"].float() @ s["b"].float().t()) * s["sa"][:, None] * s["sb"][None, :]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(s["out"])
    if op == "rows":
        return _rows8(s["x"].float())
    if op == "swiglu":
        d = s["cols"]
        gate, up = s["gu"][:, :d].float(), s["gu"][:, d:].float()
        return _rows8(gate / (1.0 + torch.exp(-gate)) * up)
    x, r = s["x"], s["rows"]
    b, d = x.shape[0] // r, x.shape[1]
    h = x.float().view(b, r, d)
    if s["residual"] is not None:
        if s["gate"] is not None:
            h = h * s["gate"].float()[:, None]
        h = s["residual"].float().view(b, r, d) + h
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"])
    if s["w"] is not None:
        y = y * s["w"].float()
    if s["scale"] is not None:
        y = y * (1.0 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    v, sc = _rows8(y.view(b * r, d))
    return (v, sc, h.view(b * r, d).to(x.dtype)) if s["residual"] is not None else (v, sc)


def _framework(s):
    from harp_b200.ops import functional as Fn

    op = s["op"]
    if op == "gemm":
        return Fn.gemm_s8(s["a"], s["sa"], s["b"], s["sb"], bias=s["bias"], out_dtype=s["out"])
    if op == "rows":
        q, sc = Fn.quant_rows(s["x"])
        return Fn.dequant_rows(q, sc), sc
    if op == "swiglu":
        q, sc = Fn.swiglu_quant(s["gu"], s["cols"])
        return Fn.dequant_rows(q, sc), sc
    q, sc, h = Fn.rmsnorm_mod_quant(s["x"], s["w"], s["scale"], s["shift"], s["rows"], s["eps"],
                                    residual=s["residual"], gate=s["gate"])
    v = Fn.dequant_rows(q, sc)
    return (v, sc, h) if s["residual"] is not None else (v, sc)


def run(state):
    with torch.no_grad():
        return _framework(state) if own else _plain(state)


def work(case):
    """Inputs and outputs once each; of the 8-bit rows both the bytes and the bf16 values that a run returns."""
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        out = 2 if case["out"] == "bf16" else 4
        return {"bytes": m * k + n * k + 4 * (m + n) + (2 * n if case["bias"] else 0) + out * m * n, "flops": 2 * m * n * k}
    e = 2 if case["dtype"] == "bf16" else 4
    rows, d = case["batch"] * case["rows"], case["cols"]
    written = rows * d * 3 + 4 * rows
    if case["op"] == "swiglu":
        return {"bytes": 2 * e * rows * d + written, "flops": 10 * rows * d}
    if case["op"] == "rows":
        return {"bytes": e * rows * d + written, "flops": 5 * rows * d}
    streams = 3 if case["residual"] else 1
    vectors = case["batch"] * (int(case["gate"]) + 2 * int(case["mod"])) + int(case["weight"])
    return {"bytes": e * d * (streams * rows + vectors) + written, "flops": 16 * rows * d}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "gemm":
        y = torch.matmul(s["a"].to(f64), s["b"].to(f64).T)
        y.mul_(s["sa"].to(f64).unsqueeze(1)).mul_(s["sb"].to(f64).unsqueeze(0))
        return y if s["bias"] is None else y.add_(s["bias"].to(f64))
    h = None
    if case["op"] == "rows":
        y = s["x"].to(f64)
    elif case["op"] == "swiglu":
        gate, up = s["gu"].to(f64).split(case["cols"], dim=1)
        y = torch.sigmoid(gate).mul_(gate).mul_(up)
    else:
        of_row = torch.arange(case["batch"], device="cuda").repeat_interleave(case["rows"])
        h = s["x"].to(f64)
        if case["gate"]:
            h = h * s["gate"].to(f64)[of_row]
        if case["residual"]:
            h = h + s["residual"].to(f64)
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + s["eps"])
        if case["weight"]:
            y = y * s["w"].to(f64)
        if case["mod"]:
            y = y + y * s["scale"].to(f64)[of_row] + s["shift"].to(f64)[of_row]
    step = torch.maximum(y.abs().max(dim=1).values / 127, torch.full((), TINY, dtype=f64, device="cuda"))
    values = torch.round(y / step.unsqueeze(1)) * step.unsqueeze(1)
    return (values, step, h) if case.get("residual") else (values, step)
