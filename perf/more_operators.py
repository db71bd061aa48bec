"""The work of the 8-bit integer linears and of the norms between them.

Each case is one pass through one operator:

* ``norm``     the residual stream's update by a block's output, with the norms before and after it,
               a gate and a scale; the result as values or as codes for the next products
* ``quant``    a block's input as 8-bit codes with one scale for each token
* ``qkv``      the three projections of one input: codes of its tokens, integer products, scales
* ``linear``   one such projection
* ``gate_up``  two of them, ``silu(gate) * up``

A code is the nearest to x / scale, ties to even; a token's scale is its largest magnitude / 127, rounded to
32 bits.  Widths are the benchmark's (4096, 1024 and 14336 channels, a head of 128256) and generic ones; 16
sequences are the reference server's slots and 512 tokens its prefill chunk.  Activations are normal with a few
channels many times as large, as a transformer's are; weights are normal, their scales vary by channel.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST = 4096 * 14336 * 4096  # products of the largest case
EPS = 1e-5


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # a token's residual update and the norm of the next block: latency counts
        {"name": "norm_token", "op": "norm", "m": 1, "k": 4096, "dtype": "f32", "stream": "f32", "pre": "rms", "post": "", "gate": False,
         "scale": 1.0, "codes": False},
        # a batch of tokens: norms before and after, in 16 bits over a stream in 32, codes for the next products
        {"name": "norm_batch64_codes", "op": "norm", "m": 64, "k": 4096, "dtype": "bf16", "stream": "f32", "pre": "rms", "post": "rms",
         "gate": False, "scale": 0.5, "codes": True},
        # a prompt of no round width: layer norm, gate and residual scale
        {"name": "norm_prompt", "op": "norm", "m": 4000, "k": 5000, "dtype": "f16", "stream": "f16", "pre": "layer", "post": "", "gate": True,
         "scale": 0.22, "codes": False},
        # the server's slots in front of the down projection
        {"name": "quant_batch16", "op": "quant", "m": 16, "k": 14336, "dtype": "f16"},
        # four prefill chunks there
        {"name": "quant_chunks", "op": "quant", "m": 2048, "k": 14336, "dtype": "bf16"},
        # q, k and v of one token
        {"name": "qkv_token", "op": "qkv", "m": 1, "n": 4096, "kv": 1024, "k": 4096, "dtype": "f32", "bias": False},
        # q, k and v of a prefill chunk, with biases
        {"name": "qkv_chunk", "op": "qkv", "m": 512, "n": 4096, "kv": 1024, "k": 4096, "dtype": "bf16", "bias": True},
        # the head over a small batch of tokens: a long stream of weights
        {"name": "linear_head8", "op": "linear", "m": 8, "n": 128256, "k": 4096, "dtype": "f32", "bias": False},
        # nothing round: rows, channels and width
        {"name": "linear_odd", "op": "linear", "m": 77, "n": 2777, "k": 1999, "dtype": "f16", "bias": True},
        # the down projection of a prompt
        {"name": "linear_prompt", "op": "linear", "m": 4096, "n": 4096, "k": 14336, "dtype": "bf16", "bias": False},
        # gate and up of the server's slots, one token each
        {"name": "gate_up_batch16", "op": "gate_up", "m": 16, "n": 14336, "k": 4096, "dtype": "bf16"},
        # gate and up of four prefill chunks
        {"name": "gate_up_chunks", "op": "gate_up", "m": 2048, "n": 14336, "k": 4096, "dtype": "f32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "norm", "quant", "qkv", "linear", "linear", "linear", "gate_up", "gate_up"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    m = _log_int(rng, 1, 4096)
    if op in ("norm", "quant"):
        k = _log_int(rng, 64, 16384 if op == "norm" else 32768)
        k = k if rng.random() < 0.4 else -(-k // 128) * 128
        m = max(1, min(m, 4000 * 5000 // k))
        if op == "quant":
            return {"op": op, "m": m, "k": k, "dtype": dtype}
        return {"op": op, "m": m, "k": k, "dtype": dtype, "stream": rng.choice((dtype, "f32")), "pre": rng.choice(("rms", "rms", "layer")),
                "post": rng.choice(("", "rms", "layer")), "gate": rng.random() < 0.3, "scale": rng.choice((1.0, 0.5, 0.22)),
                "codes": rng.random() < 0.5}
    k, n = _log_int(rng, 64, 16384), _log_int(rng, 16, 32768)
    if rng.random() < 0.6:
        k, n = -(-k // 128) * 128, -(-n // 64) * 64
    case = {"op": op, "m": m, "n": n, "k": k, "dtype": dtype}
    if op == "qkv":
        case["kv"] = -(-n // rng.choice((1, 4, 8)))
    rows = n + 2 * case["kv"] if op == "qkv" else 2 * n if op == "gate_up" else n
    case["m"] = max(1, min(m, LARGEST // (rows * k)))
    return case if op == "gate_up" else {**case, "bias": rng.random() < 0.4}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _states(g, m: int, k: int, dtype) -> torch.Tensor:
    """Activations [m, k]: normal, a few channels many times as large."""
    x = torch.randn(m, k, generator=g, device="cuda")
    loud = torch.rand(k, generator=g, device="cuda") < 0.02
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _weight(g, n: int, k: int) -> dict:
    """Codes [n, k] and one scale a channel, of normal weights."""
    codes = (torch.randn(n, k, generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
    return {"codes": codes, "scales": (0.6 + 0.8 * torch.rand(n, generator=g, device="cuda")) / (32 * math.sqrt(k))}


def prepare(case, seed) -> dict:
    g, op, dtype, m, k = _gen(seed), case["op"], TYPES[case["dtype"]], case["m"], case["k"]
    s = {"case": case, "x": _states(g, m, k, dtype)}
    if op == "norm":
        s["residual"] = (_states(g, m, k, torch.float32) * 2).to(TYPES[case["stream"]])
        s["gate"] = torch.randn(k, generator=g, device="cuda").to(dtype) if case["gate"] else None
        for name in ("pre", "post"):
            s[name] = None
            if case[name]:
                s[name] = {"weight": 1 + 0.3 * torch.randn(k, generator=g, device="cuda"),
                           "bias": 0.1 * torch.randn(k, generator=g, device="cuda") if case[name] == "layer" else None}
    elif op != "quant":
        ns = {"qkv": (case["n"], case.get("kv"), case.get("kv")), "linear": (case["n"],), "gate_up": (case["n"],) * 2}[op]
        s["weights"] = [_weight(g, n, k) for n in ns]
        s["biases"] = [torch.randn(n, generator=g, device="cuda") if case.get("bias") else None for n in ns]
    if own:  # the framework's handles on these tensors, the weights' rows laid out as it keeps them
        from lightbulb_amd import int8
        if op == "norm":
            s["norms"] = [s[name] and int8.Norm(s[name]["weight"], EPS, bias=s[name]["bias"], kind=case[name]) for name in ("post", "pre")]
        elif op != "quant":
            s["linears"] = [int8.Int8Linear(int8.Int8Weight(w["codes"], w["scales"]), b) for w, b in zip(s["weights"], s["biases"])]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case, op, x = s["case"], s["case"]["op"], s["x"]
    if own:
        from lightbulb_amd import int8
        if op == "norm":
            post, pre = s["norms"]
            r, y = int8.residual_norm(x, s["residual"], post=post, gate=s["gate"], scale=case["scale"], norm=pre, quantize=case["codes"])
            return [r, y.codes, y.scales] if case["codes"] else [r, y]
        if op == "quant":
            t = int8.quantize_tokens(x)
            return [t.codes, t.scales]
        if op == "qkv":
            return int8.int8_linear_group(s["linears"], x)
        if op == "linear":
            return s["linears"][0].forward(x)
        return int8.int8_gate_up_silu(*s["linears"], x)
    if op == "norm":
        return _plain_norm(s)
    codes, scales = _plain_codes(x.float())
    if op == "quant":
        return [codes, scales]
    ys = [_plain_product(codes, scales, w, b) for w, b in zip(s["weights"], s["biases"])]
    if op == "gate_up":
        return (ys[0] / (1 + (-ys[0]).exp()) * ys[1]).to(x.dtype)
    ys = [y.to(x.dtype) for y in ys]
    return ys if op == "qkv" else ys[0]


def _plain_codes(x):
    """Codes and scales of f32 rows; the quotients in 64 bits, where next to a border 32 would not tell."""
    amax = x.abs().amax(-1)
    fine = amax < math.inf
    s = torch.where(amax > 0, (amax.double() / 127).float().clamp(min=2.0 ** -126), 0.0)
    r = torch.where((s > 0)[:, None], x.double() / torch.where(s > 0, s, 1.0).double()[:, None], 0.0)
    return torch.where(fine[:, None], r.round(), 0.0).to(torch.int8), torch.where(fine, s, math.nan)


def _plain_product(codes, scales, w, bias):
    y = codes.float() @ w["codes"].float().t() * scales[:, None] * w["scales"]
    return y if bias is None else y + bias


def _plain_normed(x, norm, kind: str):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * norm["weight"].to(x.dtype)
    return x if norm["bias"] is None else x + norm["bias"]


def _plain_norm(s):
    case = s["case"]
    t = torch.float64 if case["codes"] else torch.float32  # (values next to a code's border)
    u = s["x"].to(t)
    if case["post"]:
        u = _plain_normed(u, s["post"], case["post"])
    if s["gate"] is not None:
        u = u * s["gate"]
    r = s["residual"].to(t) + u * case["scale"]
    y = _plain_normed(r, s["pre"], case["pre"])
    r = r.to(s["residual"].dtype)
    return [r, *_plain_codes(y.float())] if case["codes"] else [r, y.to(s["x"].dtype)]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    x = s["x"].double()
    if op == "norm":
        return _exact_norm(s, x)
    codes, scales = _exact_codes(x)
    if op == "quant":
        return [None, scales]  # (codes are whole numbers)
    tokens = codes * scales[:, None]
    ys = []
    for w, bias in zip(s["weights"], s["biases"]):
        y = tokens @ (w["codes"].double() * w["scales"].double()[:, None]).t()
        ys.append(y if bias is None else y + bias.double())
    if op == "gate_up":
        return torch.sigmoid(ys[0]) * ys[0] * ys[1]
    return ys if op == "qkv" else ys[0]


def _exact_codes(x):
    top = torch.linalg.vector_norm(x, math.inf, dim=-1)
    scales = torch.div(top, 127).float().double()
    return torch.round(torch.div(x, scales[:, None])).nan_to_num(0.0), scales


def _exact_norm(s, x):
    def normed(v, norm, kind):
        mean = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
        spread = torch.sqrt(((v - mean) ** 2).sum(-1, keepdim=True) / v.shape[-1] + EPS)
        out = norm["weight"].double() * (v - mean) / spread
        return out + norm["bias"].double() if norm["bias"] is not None else out

    case = s["case"]
    if s["post"] is not None:
        x = normed(x, s["post"], case["post"])
    if s["gate"] is not None:
        x = s["gate"].double() * x
    r = case["scale"] * x + s["residual"].double()
    y = normed(r, s["pre"], case["pre"])
    return [r, None, _exact_codes(y)[1]] if case["codes"] else [r, y]


# ---------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------
def work(case) -> dict:
    op, m, k, size = case["op"], case["m"], case["k"], TYPES[case["dtype"]].itemsize
    if op == "norm":
        # x and the stream read, the stream and the result written; each norm's weights, the gate
        stream = TYPES[case["stream"]].itemsize
        vectors = sum({"": 0, "rms": 4, "layer": 8}[case[name]] for name in ("pre", "post")) + (size if case["gate"] else 0)
        result = m * (k + 4) if case["codes"] else m * k * size
        return {"bytes": m * k * (size + 2 * stream) + result + vectors * k, "flops": 0}
    if op == "quant":
        return {"bytes": m * k * size + m * (k + 4), "flops": 0}
    rows = case["n"] + 2 * case["kv"] if op == "qkv" else case["n"] * (2 if op == "gate_up" else 1)
    out = case["n"] if op == "gate_up" else rows
    return {"bytes": rows * (k + 4 + (4 if case.get("bias") else 0)) + m * k * size + m * out * size, "flops": 2 * m * rows * k}
