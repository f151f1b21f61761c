"""The microscaled (MX) operators as they are measured: 4-bit quantisation and reading back, the product of two
quantised operands, the product of a gradient with a quantised operand, and a linear layer's training step made of them.

An MX operand is a matrix of narrow-float codes (E4M3, E5M2: a byte each; E2M1: two to a byte, the even column in the low
half) with one power-of-two scale byte for every 32 columns of a row: element = decode(code) * 2 ** (scale - 127).
"""
import math

import torch

own = False

GROUP = 32
E4M3, E5M2, E2M1 = 0, 1, 4
BITS = {E4M3: 8, E5M2: 8, E2M1: 4}
OUT = {"bf16": torch.bfloat16, "f32": torch.float32}
HALVES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of the eight E2M1 codes


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token's activations on their way into a 4-bit layer: latency is all there is
        {"name": "fp4_one_token", "op": "round_trip", "rows": 1, "cols": 4096, "dtype": "bf16", "gap": 0},
        # the weights of a layer, rows of very different size, quantised once per training step
        {"name": "fp4_weights", "op": "round_trip", "rows": 8192, "cols": 8192, "dtype": "bf16", "gap": 0},
        # float32 activations that are a slice of a wider tensor, at odd sizes
        {"name": "fp4_slice_f32", "op": "round_trip", "rows": 1003, "cols": 4128, "dtype": "f32", "gap": 96},
        # 8-bit activations read back to bfloat16, heavy tails and outliers
        {"name": "read_e4m3", "op": "read", "rows": 16384, "cols": 8192, "format": E4M3, "out": "bf16"},
        # one token through a square 4-bit layer: the weights are read once
        {"name": "fp4_product_1_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "a": E2M1, "b": E2M1, "bias": False},
        # a small batch of tokens against a wide 8-bit layer
        {"name": "e4m3_product_24_tokens", "op": "product", "m": 24, "n": 16384, "k": 8192, "a": E4M3, "b": E4M3, "bias": True},
        # odd sizes, the two 8-bit formats mixed
        {"name": "e5m2_product_ragged", "op": "product", "m": 1111, "n": 1003, "k": 2080, "a": E5M2, "b": E4M3, "bias": True},
        # a training batch through an 8-bit layer
        {"name": "e4m3_product_batch", "op": "product", "m": 8192, "n": 4096, "k": 4096, "a": E4M3, "b": E4M3, "bias": True},
        # the largest 4-bit product
        {"name": "fp4_product_large", "op": "product", "m": 8192, "n": 8192, "k": 8192, "a": E2M1, "b": E2M1, "bias": False},
        # gradient of a layer's input, from the layer's 8-bit weights
        {"name": "e4m3_input_gradient", "op": "grad", "m": 8192, "n": 4096, "k": 4096, "format": E4M3, "across": False},
        # gradient of a layer's weights, from the activations kept in 8 bits; an odd number of tokens
        {"name": "e4m3_weight_gradient", "op": "grad", "m": 4096, "n": 8192, "k": 5003, "format": E4M3, "across": True},
        # one training step of a 4-bit layer: both quantisations, the product, the three gradients
        {"name": "fp4_layer_step", "op": "step", "m": 4096, "n": 4096, "k": 4096, "format": E2M1},
    ]


def _spread(rng, lo, hi, by=1):
    """A multiple of `by` between the two, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / by)) * by))


def draw(rng):
    op = rng.choice(["round_trip", "read", "product", "product", "product", "grad", "grad", "step"])
    if op == "round_trip":
        return {"op": op, "rows": _spread(rng, 1, 8192), "cols": _spread(rng, 32, 8192, 32),
                "dtype": rng.choice(["bf16", "bf16", "f32"]), "gap": rng.choice([0, 0, 8, 64, 96])}
    if op == "read":
        return {"op": op, "rows": _spread(rng, 1, 16384), "cols": _spread(rng, 32, 8192, 32),
                "format": rng.choice([E4M3, E5M2, E2M1]), "out": rng.choice(["bf16", "f32"])}
    if op == "product":
        a, b = rng.choice([(E2M1, E2M1), (E2M1, E2M1), (E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2)])
        return {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 16, 8192), "k": _spread(rng, 32, 8192, 32),
                "a": a, "b": b, "bias": rng.random() < 0.5}
    if op == "grad":
        across = rng.random() < 0.5
        t, o, i = _spread(rng, 1, 8192), _spread(rng, 8, 8192, 8), _spread(rng, 32, 4096, 32)
        return {"op": op, "m": o if across else t, "n": i, "k": t if across else o,
                "format": rng.choice([E4M3, E5M2, E2M1]), "across": across}
    return {"op": op, "m": _spread(rng, 1, 4096), "n": _spread(rng, 8, 4096, 8), "k": _spread(rng, 32, 4096, 32),
            "format": rng.choice([E4M3, E2M1])}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols):
    """Normal values with one in a thousand some thirty times as large: what a layer is fed."""
    x = _normal(g, rows, cols)
    return torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 0.001, x * 30.0, x)


def _weights(g, rows, cols):
    """Normal values of scale 0.02 whose rows differ in size by up to a hundred."""
    return 0.02 * _normal(g, rows, cols) * 10.0 ** (2.0 * torch.rand(rows, 1, generator=g, device="cuda") - 1.0)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = dict(case)
    if op == "round_trip":
        t = OUT[case["dtype"]]
        x = (_weights if case["rows"] > 4096 else _activations)(g, case["rows"], case["cols"] + case["gap"]).to(t)
        s["x"] = x[:, :case["cols"]]
    elif op == "read":
        s["codes"], s["scales"] = _quantised(_activations(g, case["rows"], case["cols"]), case["format"])
    elif op == "product":
        s["ac"], s["as"] = _quantised(_activations(g, case["m"], case["k"]), case["a"])
        s["bc"], s["bs"] = _quantised(_weights(g, case["n"], case["k"]), case["b"])
        s["bias_"] = _normal(g, case["n"]).to(torch.bfloat16) if case["bias"] else None
    elif op == "grad":
        shape = (case["k"], case["m"]) if case["across"] else (case["m"], case["k"])
        s["g"] = (1e-3 * _normal(g, *shape)).to(torch.bfloat16)
        make = _activations if case["across"] else _weights
        s["codes"], s["scales"] = _quantised(make(g, case["k"], case["n"]), case["format"])
    else:
        s["x"] = _activations(g, case["m"], case["k"]).to(torch.bfloat16).requires_grad_()
        s["w"] = _weights(g, case["n"], case["k"]).to(torch.bfloat16).requires_grad_()
        s["b"] = _normal(g, case["n"]).to(torch.bfloat16).requires_grad_()
        s["g"] = (1e-3 * _normal(g, case["m"], case["n"])).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _scale_bytes(x, fmt):
    """The byte s of every group: the largest power of two 2 ** (127 - s) that keeps the group's largest value within the
    format's largest; 127 for a group of zeros."""
    top, frac = {E4M3: (8, 1.75), E5M2: (15, 1.75), E2M1: (2, 1.5)}[fmt]
    amax = x.reshape(x.shape[0], -1, GROUP).abs().amax(2)
    m, e = torch.frexp(amax)                      # amax = m * 2 ** e, m in [1/2, 1)
    s = (e - 1) - top + (2 * m > frac).to(e.dtype) + 127
    return torch.where(amax > 0, s.clamp(0, 254), 127)


def _power(field):
    """2 ** (field - 127) from an exponent field in 32 bits, exactly; NaN for 255."""
    field = field.int()
    return torch.where(field == 0, 0x400000, torch.where(field == 255, 0x7FC00000, field << 23)).view(torch.float32)[:, :, None]


def _to_halves(q):
    """Magnitude codes of the E2M1 values nearest to q, ties to the even code."""
    a = q.abs()
    return ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
            + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8))


def _quantised(x, fmt):
    """Codes and scale bytes of a matrix, in 32 bits."""
    x = x.float()
    s = _scale_bytes(x, fmt)
    q = (x.reshape(x.shape[0], -1, GROUP) * _power(254 - s)).reshape(x.shape)
    if fmt == E2M1:
        c = _to_halves(q) | (torch.signbit(q).to(torch.uint8) << 3)
        c = c[:, 0::2] | (c[:, 1::2] << 4)
    else:
        c = q.to(torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2).view(torch.uint8)
    return c, s.to(torch.uint8)


def _values(c, s, fmt):
    """What codes and scale bytes stand for, in 32 bits."""
    if fmt == E2M1:
        n = torch.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)
        table = torch.tensor(HALVES + tuple(-v for v in HALVES), device=c.device)
        v = table[n.int()]
    else:
        v = c.view(torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2).float()
    return (v.reshape(c.shape[0], -1, GROUP) * _power(s)).reshape(v.shape)


def run(s):
    op = s["op"]
    if op == "round_trip":
        x = s["x"]
        if own:
            from mor_b200 import ops
            c, e = ops.quantize_mx_fp4(x, x.shape[0], x.shape[1], GROUP)
            return ops.dequantize_mx(c, e, x.shape[0], x.shape[1], GROUP, E2M1), e
        c, e = _quantised(x, E2M1)
        return _values(c, e, E2M1).to(torch.bfloat16), e
    if op == "read":
        t = OUT[s["out"]]
        if own:
            from mor_b200 import ops
            return ops.dequantize_mx(s["codes"], s["scales"], s["rows"], s["cols"], GROUP, s["format"], t)
        return _values(s["codes"], s["scales"], s["format"]).to(t)
    if op == "product":
        if own:
            from mor_b200 import ops
            return ops.mx_matmul(s["ac"], s["as"], s["bc"], s["bs"], s["m"], s["n"], s["k"], s["a"], s["b"], s["bias_"])
        y = _values(s["ac"], s["as"], s["a"]) @ _values(s["bc"], s["bs"], s["b"]).t()
        return (y if s["bias_"] is None else y + s["bias_"].float()).to(torch.bfloat16)
    if op == "grad":
        if own:
            from mor_b200 import ops
            return ops.mx_matmul_grad(s["g"], s["codes"], s["scales"], s["m"], s["n"], s["k"], s["format"], s["across"])
        g = s["g"].float()
        return ((g.t() if s["across"] else g) @ _values(s["codes"], s["scales"], s["format"])).to(torch.bfloat16)
    if own:
        from mor_b200.nn import mx_linear
        y = mx_linear(s["x"], s["w"], s["b"], s["format"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"]))
    xq = _values(*_quantised(s["x"].detach(), s["format"]), s["format"])
    wq = _values(*_quantised(s["w"].detach(), s["format"]), s["format"])
    g = s["g"].float()
    outs = (xq @ wq.t() + s["b"].detach().float(), g @ wq, g.t() @ xq, g.sum(0))
    return tuple(t.to(torch.bfloat16) for t in outs)


# ------------------------------------------------------------------------------------------------ work
def _operand(rows, cols, fmt):
    return rows * cols * BITS[fmt] / 8 + rows * (cols // GROUP)


def work(case):
    op = case["op"]
    if op == "round_trip":    # the input once, the codes and scales written and read, the values written
        n = case["rows"] * case["cols"]
        width = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * width + 2 * _operand(case["rows"], case["cols"], E2M1) + 2 * n, "flops": 0}
    if op == "read":
        n = case["rows"] * case["cols"]
        return {"bytes": _operand(case["rows"], case["cols"], case["format"]) + n * (2 if case["out"] == "bf16" else 4), "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "product":
        return {"bytes": _operand(m, k, case["a"]) + _operand(n, k, case["b"]) + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "grad":
        return {"bytes": 2 * m * k + _operand(k, n, case["format"]) + 2 * m * n, "flops": 2 * m * n * k}
    f = case["format"]        # x, w, b and the gradient read; y and the three gradients written; the operands kept in between
    return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n + 2 * n) + 2 * (_operand(m, k, f) + _operand(n, k, f)), "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------------------ 64 bits
def _two_to(e):
    """2 ** e for whole e in the normal range of 64 bits, by its bits: a library's power is off in the last one."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(c, s, fmt):
    """Codes taken apart into sign, exponent and mantissa fields."""
    c = c.to(torch.int32)
    if fmt == E2M1:
        c = torch.cat(((c & 15)[:, :, None], (c >> 4)[:, :, None]), 2).flatten(1)
    width, mant, bias = {E4M3: (8, 3, 7), E5M2: (8, 2, 15), E2M1: (4, 1, 1)}[fmt]
    sign = 1.0 - 2.0 * (c >> (width - 1)).double()
    field = (c & ((1 << (width - 1)) - 1)) >> mant
    frac = (c & ((1 << mant) - 1)).double() / (1 << mant)
    v = sign * torch.where(field > 0, 1.0 + frac, frac) * _two_to(field.clamp(min=1) - bias)
    return v * _two_to(s.long() - 127).repeat_interleave(GROUP, dim=1)


def _quantise64(x, fmt):
    """Nearest representable values under each group's scale, by rounding to the spacing of the binade they lie in."""
    limit, mant, lowest = {E4M3: (448.0, 3, -6), E5M2: (57344.0, 2, -14), E2M1: (6.0, 1, 0)}[fmt]
    x = x.double()
    amax = x.abs().unflatten(1, (-1, GROUP)).amax(2)
    safe = torch.where(amax > 0, amax, 1.0)
    up = torch.floor(torch.log2(limit / safe))
    up = torch.where(safe * _two_to(up) > limit, up - 1, up)          # a logarithm next to a whole number
    up = torch.where(safe * _two_to(up + 1) <= limit, up + 1, up)
    up = torch.where(amax > 0, up, 0.0).clamp(-127, 127)
    q = x * _two_to(up).repeat_interleave(GROUP, dim=1)
    _, e = torch.frexp(q.abs())
    step = _two_to((e - 1).clamp(min=lowest) - mant)
    q = torch.round(q / step) * step                                         # ties to even
    return q * _two_to(-up).repeat_interleave(GROUP, dim=1), (127 - up).to(torch.uint8)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "round_trip":
        return _quantise64(s["x"], E2M1)
    if op == "read":
        return _decode64(s["codes"], s["scales"], case["format"])
    if op == "product":
        y = torch.mm(_decode64(s["ac"], s["as"], case["a"]), _decode64(s["bc"], s["bs"], case["b"]).transpose(0, 1))
        return y if s["bias_"] is None else y.add_(s["bias_"].double())
    g = s["g"].double()
    if op == "grad":
        return torch.mm(g.transpose(0, 1) if case["across"] else g, _decode64(s["codes"], s["scales"], case["format"]))
    x, w = _quantise64(s["x"].detach(), case["format"])[0], _quantise64(s["w"].detach(), case["format"])[0]
    return torch.mm(x, w.transpose(0, 1)) + s["b"].detach().double(), torch.mm(g, w), torch.mm(g.transpose(0, 1), x), g.sum(0)
