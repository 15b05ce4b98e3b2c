"""Timed cases of the microscaled operators: rows quantised in blocks of 32 values that share a power-of-two scale, the
norm that writes such rows, the linear layer with 4-bit weights, and the ConvNeXt tail made of them.

A block's scale is 2^e (one byte, e + 127); its elements are e4m3 (8 bits, largest 448) or e2m1 (4 bits, largest 6, two
a byte, the even one in the low half). e is the least for which the block's largest magnitude over 2^e still rounds to the
largest element or below it, were the elements' grid continued: at most 464 for e4m3 (which ties to 448), below 7 for
e2m1. Weights are kept as bytes: codes [rows, K/2] and scales [rows, 16 * ceil(K/512)], of which K/32 are in use.

Every op and what it needs:
  quantize  n, k, fmt, dtype                    mx_quantize, then mx_dequantize: the values that the blocks hold, in bf16
  norm      n, c, kind, residual, dtype         add_norm_mx: the sum, and its norm as e4m3 elements and their scales
  linear    n, k, co, fmt, act, residual, dtype mx_linear: x quantised to fmt, e2m1 weights, bias
  tail      n, c, dtype                         convnext_mlp_mx: LayerNorm, C -> 4C with SiLU, 4C -> C, the residual
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # A weight matrix of the coarsest level's MLP going into 4 bits: the smallest bulk conversion.
        {"name": "quantize_weights", "op": "quantize", "n": 4096, "k": 1024, "fmt": "e2m1", "dtype": "f16"},
        # The features of a 256^3 shell, 256 channels: a whole level's activations.
        {"name": "quantize_rows", "op": "quantize", "n": 390503, "k": 256, "fmt": "e2m1", "dtype": "bf16"},
        # One token's residual sum and norm ahead of its next linear layer: latency alone.
        {"name": "norm_token", "op": "norm", "n": 1, "c": 4096, "kind": "rms", "residual": True, "dtype": "bf16"},
        # A decoder level's rows ahead of the MLP: LayerNorm, no residual.
        {"name": "norm_rows", "op": "norm", "n": 58321, "c": 256, "kind": "layer", "residual": False, "dtype": "f16"},
        # A long prompt's rows: the norm where it is bandwidth.
        {"name": "norm_long", "op": "norm", "n": 32771, "c": 4096, "kind": "rms", "residual": True, "dtype": "bf16"},
        # One token through a square layer: the weights are read once for it.
        {"name": "linear_token", "op": "linear", "n": 1, "k": 4096, "co": 4096, "fmt": "e4m3", "act": "none",
         "residual": False, "dtype": "bf16"},
        # A batch of single tokens through a widening layer: still bound by the weights' bytes.
        {"name": "linear_batch", "op": "linear", "n": 77, "k": 4096, "co": 8192, "fmt": "e4m3", "act": "silu",
         "residual": False, "dtype": "bf16"},
        # A long prompt through a square layer, both operands in 4 bits: the largest product.
        {"name": "linear_long", "op": "linear", "n": 16411, "k": 4096, "co": 4096, "fmt": "e2m1", "act": "none",
         "residual": True, "dtype": "bf16"},
        # The same rows with 8-bit activations, to a width that no tile divides.
        {"name": "linear_mixed", "op": "linear", "n": 8209, "k": 2080, "co": 4128, "fmt": "e4m3", "act": "silu",
         "residual": False, "dtype": "f16"},
        # The ConvNeXt tails of the three levels where the two products carry the time.
        {"name": "tail_1024", "op": "tail", "n": 1803, "c": 1024, "dtype": "f16"},
        {"name": "tail_512", "op": "tail", "n": 11467, "c": 512, "dtype": "bf16"},
        {"name": "tail_256", "op": "tail", "n": 58321, "c": 256, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear", "linear", "tail"])
    dt = rng.choice(["f16", "bf16"])
    if op == "quantize":
        k = 32 * _log(rng, 2, 128)
        return {"op": op, "n": _log(rng, 1, 100_000_000 // k // 2), "k": k, "fmt": rng.choice(["e2m1", "e4m3"]), "dtype": dt}
    if op == "norm":
        c = 32 * _log(rng, 2, 128)
        return {"op": op, "n": _log(rng, 1, min(390000, 130_000_000 // c)), "c": c, "kind": rng.choice(["rms", "layer"]),
                "residual": rng.random() < 0.6, "dtype": dt}
    if op == "linear":
        k, co = 32 * _log(rng, 4, 128), 32 * _log(rng, 4, 256)
        return {"op": op, "n": _log(rng, 1, min(60000, 16000 * 4096 * 4096 // (k * co))), "k": k, "co": co,
                "fmt": rng.choice(["e4m3", "e2m1"]), "act": rng.choice(["none", "silu"]), "residual": rng.random() < 0.5,
                "dtype": dt}
    c = rng.choice([256, 512, 1024, 32 * rng.randint(4, 32)])
    return {"op": op, "n": _log(rng, 1, min(100000, 58000 * 256 * 256 // (c * c) * 4)), "c": c, "dtype": dt}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _features(g, n, c, dt):
    """Activations: channels of unequal spread, a hundredth of them ten times as large."""
    spread = torch.exp(0.5 * _rand(g, c)) * torch.where(torch.rand(c, generator=g, device="cuda") < 0.01, 10.0, 1.0)
    return (_rand(g, n, c) * spread).to(dt)


def _weights(g, co, k):
    """(codes, scales) of a [co, k] layer, as bytes."""
    elements, e = _blocks(_rand(g, co, k) / math.sqrt(k), "e2m1")
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    code = torch.searchsorted(table, elements.abs().contiguous()) + 8 * (elements < 0)
    code = code.view(co, k // 2, 2).to(torch.uint8)
    scales = torch.zeros((co, 16 * -(-k // 512)), dtype=torch.uint8, device="cuda")
    scales[:, :k // 32] = (e + 127).to(torch.uint8)
    return code[:, :, 0] | code[:, :, 1] << 4, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n, op = DTYPES[case["dtype"]], case["n"], case["op"]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _features(g, n, case["k"], dt)
    elif op == "norm":
        c = case["c"]
        s["x"] = _features(g, n, c, dt)
        s["res"] = (3 * _rand(g, n, c) + 0.5).to(dt) if case["residual"] else None
        s["gamma"] = torch.rand(c, generator=g, device="cuda") + 0.5
        s["beta"] = 0.2 * _rand(g, c) if case["kind"] == "layer" else None
    elif op == "linear":
        k, co = case["k"], case["co"]
        s["x"] = _features(g, n, k, dt)
        s["w"] = _weights(g, co, k)
        s["bias"] = 0.1 * _rand(g, co)
        s["res"] = _rand(g, n, co).to(dt) if case["residual"] else None
    else:
        c = case["c"]
        s["h"], s["x"] = (_features(g, n, c, dt) + 1).to(dt), _rand(g, n, c).to(dt)
        s["gamma"], s["beta"] = torch.rand(c, generator=g, device="cuda") + 0.5, 0.2 * _rand(g, c)
        s["w1"], s["b1"] = _weights(g, 4 * c, c), 0.1 * _rand(g, 4 * c)
        s["w2"], s["b2"] = _weights(g, c, 4 * c), 0.1 * _rand(g, c)
    return s


# ---- the plain form: 32 bits -----------------------------------------------------------------------------------


def _blocks(x, fmt):
    """x float32 [n,k] in blocks of 32: (elements float32 [n,k], exponents int32 [n,k/32])."""
    n, k = x.shape
    b = x.view(n, k // 32, 32)
    m, e = torch.frexp(b.abs().amax(2))  # m in [1/2, 1), 0 for a block of zeros
    if fmt == "e4m3":
        e = torch.where(2 * m <= 1.8125, e - 9, e - 8)
    else:
        e = torch.where(2 * m < 1.75, e - 3, e - 2)
    e = torch.where(m == 0, -127, e.clamp(-127, 127))
    v = torch.ldexp(b, -e.unsqueeze(2))
    if fmt == "e4m3":
        q = v.to(torch.float8_e4m3fn).float()
    else:
        a = v.abs()
        q = 0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5)
        q = torch.where(v < 0, -q, q)
    return q.view(n, k), e


def _values(q, e):
    n, k = q.shape
    return torch.ldexp(q.view(n, k // 32, 32), e.unsqueeze(2)).view(n, k)


def _decode(w, k):
    codes, scales = w
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    q = table[torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], k).int()]
    return _values(q, scales[:, :k // 32].int() - 127)


def _norm(t, kind, gamma, beta):
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * gamma
    return y if beta is None else y + beta


def _silu(v):
    return v / (1 + torch.exp(-v))


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return _values(*_blocks(s["x"].float(), case["fmt"])).to(torch.bfloat16)
    if op == "norm":
        t = s["x"] if s["res"] is None else (s["x"].float() + s["res"].float()).to(s["x"].dtype)
        q, e = _blocks(_norm(t.float(), case["kind"], s["gamma"], s["beta"]), "e4m3")
        return {"sum": t, "elements": q.to(torch.float8_e4m3fn),
                "scales": torch.ldexp(torch.ones_like(e, dtype=torch.float32), e).to(torch.float8_e8m0fnu)}
    if op == "linear":
        x = _values(*_blocks(s["x"].float(), case["fmt"]))
        y = x @ _decode(s["w"], case["k"]).T + s["bias"]
        if case["act"] == "silu":
            y = _silu(y)
        return (y if s["res"] is None else y + s["res"].float()).to(s["x"].dtype)
    c = case["c"]
    a = _values(*_blocks(_norm(s["h"].float(), "layer", s["gamma"], s["beta"]), "e4m3"))
    a = _silu(a @ _decode(s["w1"], c).T + s["b1"])
    y = _values(*_blocks(a, "e4m3")) @ _decode(s["w2"], 4 * c).T + s["b2"]
    return (y + s["x"].float()).to(s["x"].dtype)


# ---- the framework's operators ---------------------------------------------------------------------------------


def _own(s):
    import spconv_amd as sp

    case, op = s["case"], s["case"]["op"]
    fmt = sp.MX_E2M1 if case.get("fmt") == "e2m1" else sp.MX_E4M3
    if op == "quantize":
        return sp.mx_dequantize(sp.mx_quantize(s["x"], fmt), torch.bfloat16)
    if op == "norm":
        t, q = sp.add_norm_mx(s["x"], s["res"], s["gamma"], s["beta"], eps=EPS,
                              kind=sp.NORM_LAYER if case["kind"] == "layer" else sp.NORM_RMS)
        # The 8-bit elements and scales as the values that their bytes are.
        return {"sum": t, "elements": q.codes.view(torch.float8_e4m3fn),
                "scales": q.scales[:, :case["c"] // 32].view(torch.float8_e8m0fnu)}
    if op == "linear":
        w = sp.MxTensor(*s["w"], case["k"], sp.MX_E2M1)
        return sp.mx_linear(s["x"], w, s["bias"], residual=s["res"], act=sp.ACT_SILU if case["act"] == "silu" else sp.ACT_NONE,
                            fmt=fmt)
    c = case["c"]
    return sp.convnext_mlp_mx(s["h"], s["x"], s["gamma"], s["beta"], sp.MxTensor(*s["w1"], c, sp.MX_E2M1), s["b1"],
                              sp.MxTensor(*s["w2"], 4 * c, sp.MX_E2M1), s["b2"], eps=EPS)


def run(state):
    if own:
        package = os.path.join(os.getcwd(), "trellis2-cuda_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        return _own(state)
    return _plain(state)


# ---- 64 bits ---------------------------------------------------------------------------------------------------


def _nearest(v, fmt):
    """float64 values to the nearest element, halves to the even one: multiples of the step at each magnitude."""
    least, bits, most = (-6, 3, 448.0) if fmt == "e4m3" else (0, 1, 6.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** least))) - bits)
    return torch.clamp(torch.round(v / step) * step, -most, most)


def _held(x, fmt):
    """(elements, scales per block) of float64 rows."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(2)
    s = torch.exp2(torch.floor(torch.log2(top)) - (8 if fmt == "e4m3" else 2))
    s = torch.where(top > 464 * s, 2 * s, s) if fmt == "e4m3" else torch.where(top >= 7 * s, 2 * s, s)
    return _nearest(b / s[:, :, None], fmt), s


def _held_values(x, fmt):
    q, s = _held(x, fmt)
    return (q * s[:, :, None]).reshape(x.shape)


def _weight64(w, k):
    codes, scales = w
    c = torch.empty((codes.shape[0], k), dtype=torch.long, device=codes.device)
    c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
    expo, man = (c // 2) % 4, (c % 2).double()
    mag = torch.where(expo == 0, 0.5 * man, (1 + 0.5 * man) * torch.exp2(expo.double() - 1))
    s = torch.exp2(scales[:, :k // 32].double() - 127)
    return torch.where(c >= 8, -mag, mag) * s.repeat_interleave(32, 1)


def _norm64(t, kind, gamma, beta):
    mean = t.sum(1, keepdim=True) / t.shape[1] if kind == "layer" else 0.0
    var = (t - mean).square().sum(1, keepdim=True) / t.shape[1]
    y = (t - mean) / torch.sqrt(var + EPS) * gamma.double()
    return y + beta.double() if beta is not None else y


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        return _held_values(s["x"].double(), case["fmt"])
    if op == "norm":
        t = s["x"].double()
        if s["res"] is not None:
            t = (t + s["res"].double()).to(s["x"].dtype).double()  # the sum is held, and normalised, in the inputs' type
        q, scales = _held(_norm64(t, case["kind"], s["gamma"], s["beta"]), "e4m3")
        return {"sum": t, "elements": q.reshape(t.shape), "scales": scales}
    if op == "linear":
        y = torch.mm(_held_values(s["x"].double(), case["fmt"]), _weight64(s["w"], case["k"]).t()) + s["bias"].double()
        y = y * torch.sigmoid(y) if case["act"] == "silu" else y
        return y if s["res"] is None else y + s["res"].double()
    c = case["c"]
    a = _held_values(_norm64(s["h"].double(), "layer", s["gamma"], s["beta"]), "e4m3")
    a = torch.mm(a, _weight64(s["w1"], c).t()) + s["b1"].double()
    a = _held_values(a * torch.sigmoid(a), "e4m3")
    return torch.mm(a, _weight64(s["w2"], 4 * c).t()) + s["b2"].double() + s["x"].double()


def work(case):
    n, op = case["n"], case["op"]
    if op == "quantize":
        return {"bytes": 4 * n * case["k"], "flops": 2 * n * case["k"]}
    if op == "norm":
        c = case["c"]
        return {"bytes": n * c * (6 if case["residual"] else 2) + n * c * 33 // 32 + 4 * c, "flops": 8 * n * c}
    if op == "linear":
        k, co = case["k"], case["co"]
        return {"bytes": 2 * n * k + co * k * 17 // 32 + 4 * co + 2 * n * co * (2 if case["residual"] else 1),
                "flops": 2 * n * k * co}
    c = case["c"]
    return {"bytes": 6 * n * c + 8 * c * c * 17 // 32 + 28 * c, "flops": 16 * n * c * c}
