"""Cases of the 8-bit integer (W8A8) linear path: tokens quantised row by row with a scale each, weights with a scale per
output channel, exact integer products.

* ``norm``:   residual add + RMSNorm with an 8-bit output (the input of the qkv / gate_up projections)
* ``swiglu``: SiLU(gate) * up with an 8-bit output (the input of the down projection)
* ``quant``:  plain row quantiser (the input of the attention output projection)
* ``linear``: the integer matrix product with its scales
* ``mlp``:    norm -> gate_up -> SwiGLU -> down, as a decoder layer runs them

Codes are returned as the values they stand for (``code * scale``), together with the scales.
"""
import math

import torch

own = False

FLOOR = 2.0 ** -120          # smallest scale of a row
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode token of the 27B-shaped model (hidden 5120): latency
        {"name": "norm decode 1", "op": "norm", "n": 1, "h": 5120, "delta": True, "f16": False},
        # one prefill chunk of the same model, with the f16 copy that a bf16 / fp8 linear of the layer reads
        {"name": "norm prefill 4096", "op": "norm", "n": 4096, "h": 5120, "delta": True, "f16": True},
        # a three-token speculative verify (intermediate 17408)
        {"name": "swiglu verify 3", "op": "swiglu", "n": 3, "inter": 17408},
        # a prefill chunk of the same
        {"name": "swiglu prefill 4096", "op": "swiglu", "n": 4096, "inter": 17408},
        # sixteen lanes' attention outputs (24 heads x 256) on their way to the output projection
        {"name": "quant lanes 16", "op": "quant", "n": 16, "k": 6144, "type": "f16"},
        # a ragged prompt and an odd width
        {"name": "quant ragged 1237", "op": "quant", "n": 1237, "k": 4111, "type": "bf16"},
        # batch-1 decode through gate_up: streaming weights
        {"name": "linear decode 1", "op": "linear", "n": 1, "m": 34816, "k": 5120, "out": "bf16"},
        # sixteen lanes through the down projection: few output channels, a long sum
        {"name": "linear lanes 16", "op": "linear", "n": 16, "m": 5120, "k": 17408, "out": "bf16"},
        # seven verify columns through the LM head, fp32 logits
        {"name": "linear head 7", "op": "linear", "n": 7, "m": 248320, "k": 5120, "out": "f32"},
        # odd sizes in every direction: a short prompt through a small adapter-like projection
        {"name": "linear odd 203", "op": "linear", "n": 203, "m": 1001, "k": 2063, "out": "f32"},
        # a prefill chunk through gate_up: the tensor cores' rate
        {"name": "linear prefill 4096", "op": "linear", "n": 4096, "m": 34816, "k": 5120, "out": "bf16"},
        # a 333-token prompt through a whole feed-forward block
        {"name": "mlp prompt 333", "op": "mlp", "n": 333, "h": 5120, "inter": 17408},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "quant", "linear", "linear", "mlp"])
    n = _log(rng, 1, 4096)
    if op == "norm":
        return {"op": op, "n": n, "h": _log(rng, 64, 17408), "delta": rng.random() < 0.8, "f16": rng.random() < 0.5}
    if op == "swiglu":
        return {"op": op, "n": n, "inter": _log(rng, 64, 17408)}
    if op == "quant":
        return {"op": op, "n": n, "k": _log(rng, 64, 17408), "type": rng.choice(sorted(TYPES))}
    if op == "linear":
        m, k = _log(rng, 64, 34816), _log(rng, 64, 17408)
        if rng.random() < 0.5:                  # model widths are multiples of 64; the others stay odd
            m, k = -(-m // 64) * 64, min(17408, -(-k // 64) * 64)
        return {"op": op, "n": min(n, 4096 * 34816 * 5120 // (m * k)), "m": m, "k": k, "out": rng.choice(["bf16", "f32"])}
    h = 16 * _log(rng, 8, 320)
    return {"op": op, "n": _log(rng, 1, 2048), "h": h, "inter": 16 * _log(rng, 8, 1088)}


def work(case):
    op, n = case["op"], case["n"]
    if op == "norm":
        h = case["h"]
        each = 2 + (4 if case["delta"] else 0) + 1 + (2 if case["f16"] else 0)
        return {"bytes": n * h * each + 4 * h + 4 * n, "flops": 8 * n * h}
    if op == "swiglu":
        return {"bytes": n * case["inter"] * 5 + 4 * n, "flops": 10 * n * case["inter"]}
    if op == "quant":
        return {"bytes": n * case["k"] * ((4 if case["type"] == "f32" else 2) + 1) + 4 * n, "flops": 4 * n * case["k"]}
    if op == "linear":
        m, k = case["m"], case["k"]
        return {"bytes": n * k + m * k + 4 * (n + m) + n * m * (4 if case["out"] == "f32" else 2), "flops": 2 * n * m * k}
    h, inter = case["h"], case["inter"]
    return {"bytes": 3 * h * inter + 4 * (3 * h + 2 * inter) + n * h * 8, "flops": 6 * n * h * inter}


# ------------------------------------------------------------------ inputs

def _codes(rows, k, g):
    """int8 codes as a quantised Gaussian row gives them, rows 16-byte aligned as the product wants them."""
    t = torch.zeros((rows, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 28) // k)
    for r in range(0, rows, step):
        v = torch.randn((min(step, rows - r), k), generator=g, device="cuda")
        t[r:r + step, :k] = (v * 31.0).round_().clamp_(-127, 127).to(torch.int8)
    return t[:, :k]


def _scales(rows, size, g):
    return (0.5 + torch.rand(rows, generator=g, device="cuda")) * size


def _hidden(n, h, g, dtype=torch.bfloat16):
    """Hidden rows: unit Gaussian channels with a few that run an order of magnitude hotter, rows of different size."""
    x = torch.randn((n, h), generator=g, device="cuda")
    hot = torch.rand(h, generator=g, device="cuda") < 0.01
    row = torch.exp(0.5 * torch.randn((n, 1), generator=g, device="cuda"))
    return (x * torch.where(hot, 10.0, 1.0) * row).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, n = case["op"], case["n"]
    s = {"case": case}
    if op in ("norm", "mlp"):
        h = case["h"]
        s["res"], s["w"] = _hidden(n, h, g), 0.1 * torch.randn(h, generator=g, device="cuda")
        s["delta"] = _hidden(n, h, g) if case.get("delta", True) else None
    if op == "swiglu":
        s["gu"] = _hidden(n, 2 * case["inter"], g)
    if op == "quant":
        s["x"] = _hidden(n, case["k"], g, TYPES[case["type"]])
    if op == "linear":
        m, k = case["m"], case["k"]
        s["codes"], s["row_scale"] = _codes(m, k, g), _scales(m, 1 / (31 * math.sqrt(k)), g)
        s["q"], s["scale"] = _codes(n, k, g), _scales(n, 1 / 31, g)
    if op == "mlp":
        h, inter = case["h"], case["inter"]
        s["gu_codes"], s["gu_scale"] = _codes(2 * inter, h, g), _scales(2 * inter, 1 / (31 * math.sqrt(h)), g)
        s["down_codes"], s["down_scale"] = _codes(h, inter, g), _scales(h, 1 / (31 * math.sqrt(inter)), g)
    return s


# ------------------------------------------------------------------ the framework's calls

def _run_own(s):
    import velogb10_b200.ops.int8 as ops
    from velogb10_b200.models.weights import QLinear
    case = s["case"]
    op, n = case["op"], case["n"]
    if op == "norm":
        f16 = torch.empty((n, case["h"]), dtype=torch.float16, device="cuda") if case["f16"] else None
        act = ops.add_rmsnorm_int8(s["res"], s["delta"], s["w"], EPS, out16=f16)
        return {"res": s["res"], "values": ops.dequantize_act_int8(act), "scale": act.scale, "f16": f16}
    if op == "swiglu":
        act = ops.swiglu_int8(s["gu"])
        return {"values": ops.dequantize_act_int8(act), "scale": act.scale}
    if op == "quant":
        act = ops.quantize_act_int8(s["x"])
        return {"values": ops.dequantize_act_int8(act), "scale": act.scale}
    if op == "linear":
        q = QLinear("int8", case["m"], case["k"], codes=s["codes"], row_scale=s["row_scale"])
        return ops.linear_int8(q, ops.Int8Act(s["q"], s["scale"]), out_f32=case["out"] == "f32")
    h, inter = case["h"], case["inter"]
    gate_up = QLinear("int8", 2 * inter, h, codes=s["gu_codes"], row_scale=s["gu_scale"])
    down = QLinear("int8", h, inter, codes=s["down_codes"], row_scale=s["down_scale"])
    act = ops.add_rmsnorm_int8(s["res"], s["delta"], s["w"], EPS)
    act = ops.swiglu_int8(ops.linear_int8(gate_up, act))
    return {"res": s["res"], "out": ops.linear_int8(down, act)}


# ------------------------------------------------------------------ plain forms (32 bits)

def _plain_quant(y):
    scale = (y.abs().amax(-1) / 127.0).clamp_min(FLOOR)
    return torch.round(y / scale[:, None]), scale


def _plain_norm(s):
    res = s["res"]
    if s["delta"] is not None:
        res.copy_(res.float() + s["delta"].float())
    x = res.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + s["w"])


def _plain_swiglu(gu):
    gate, up = gu.float().chunk(2, -1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_linear(q, scale, codes, row_scale, dtype):
    # a sum of integer products in fp32 is exact up to 2^24 and rounded by less than the output's type after that
    return ((q.float() @ codes.float().t()) * scale[:, None] * row_scale).to(dtype)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op == "norm":
        y = _plain_norm(s)
        q, scale = _plain_quant(y)
        return {"res": s["res"], "values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale,
                "f16": y.clamp(-65504.0, 65504.0).to(torch.float16) if case["f16"] else None}
    if op in ("swiglu", "quant"):
        q, scale = _plain_quant(_plain_swiglu(s["gu"]) if op == "swiglu" else s["x"].float())
        return {"values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale}
    if op == "linear":
        return _plain_linear(s["q"], s["scale"], s["codes"], s["row_scale"], TYPES[case["out"]])
    q, scale = _plain_quant(_plain_norm(s))
    gu = _plain_linear(q, scale, s["gu_codes"], s["gu_scale"], torch.bfloat16)
    q, scale = _plain_quant(_plain_swiglu(gu))
    return {"res": s["res"], "out": _plain_linear(q, scale, s["down_codes"], s["down_scale"], torch.bfloat16)}


# ------------------------------------------------------------------ definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64

    def rows_to_8_bits(y):
        unit = torch.maximum(y.abs().max(dim=1).values / 127, torch.full((), FLOOR, dtype=d, device=y.device))
        return torch.div(y, unit.unsqueeze(1)).round(), unit

    def product(tokens, unit, codes, per_channel):
        # both factors are whole numbers below 2^7: the sum is exact in 64 bits
        total = torch.matmul(tokens.to(d), codes.to(d).transpose(0, 1))
        return total.mul_(unit.to(d).unsqueeze(1)).mul_(per_channel.to(d).unsqueeze(0))

    def normed():
        x = s["res"].to(d)
        if s["delta"] is not None:
            x = (x + s["delta"].to(d)).to(torch.bfloat16).to(d)      # the residual is kept in bf16
        mean = (x * x).sum(dim=1, keepdim=True) / x.shape[1]
        return x, x / torch.sqrt(mean + EPS) * (s["w"].to(d) + 1)

    def gated(gu):
        half = gu.shape[1] // 2
        g, u = gu[:, :half].to(d), gu[:, half:].to(d)
        return g * torch.sigmoid(g) * u

    op = case["op"]
    if op == "linear":
        return product(s["q"], s["scale"], s["codes"], s["row_scale"])
    if op == "mlp":
        x, y = normed()
        gu = product(*rows_to_8_bits(y), s["gu_codes"], s["gu_scale"]).to(torch.bfloat16)   # stored in bf16
        return {"res": x, "out": product(*rows_to_8_bits(gated(gu)), s["down_codes"], s["down_scale"])}
    got = {}
    if op == "norm":
        got["res"], y = normed()
        got["f16"] = y if case["f16"] else None
    else:
        y = gated(s["gu"]) if op == "swiglu" else s["x"].to(d)
    codes, got["scale"] = rows_to_8_bits(y)
    got["values"] = codes * got["scale"].unsqueeze(1)
    return got
