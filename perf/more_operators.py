"""Timed cases of the linear layers with many weights: products of groups of rows with a weight matrix each, their two
gradients, and low-rank adapters of many requests beside one shared projection.

Rows of one group are consecutive: group g has rows ends[g-1] .. ends[g] - 1 (ends[-1] taken as 0), ends int32 on the
device; groups may be empty, and rows from the last end on belong to none.

Every op and what it needs (y, dy [N,O], x, dx [N,K], w, dw [G,O,K], bias, db [G,O]):
  forward  n, groups, k, o, dtype   group_linear: y[n] = w[g] x[n] + bias[g]; rows of no group stay as they were
  dx       n, groups, k, o, dtype   group_linear_dx: dx[n] = w[g]^T dy[n]
  dw       n, groups, k, o, dtype   group_linear_dw: dw[g] = sum of dy[n] x[n]^T over g's rows, db[g] = sum of dy[n]
  linear   n, adapters, rank, k, o  adapter_linear: y[n] = w x[n] + bias + scale[s] b[s] (a[s] x[n]), s = slots[n]
  add      n, adapters, rank, k, o  adapter_add: y[n] + scale[s] b[s] (a[s] x[n]), beside a projection y made elsewhere
A row whose slot is -1 has no adapter.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST = 16411 * 2048 * 4096  # products of the largest case


def listed():
    return [
        # One token, routed to two of sixteen experts: the smallest call, latency alone.
        {"name": "experts_token", "op": "forward", "n": 2, "groups": 16, "k": 1024, "o": 1024, "skew": 0.0, "spare": 0, "bias": False,
         "dtype": "bf16"},
        # 48 requests' single tokens, eight of 64 experts each: every expert has a few rows, its weights are what counts.
        {"name": "experts_batch", "op": "forward", "n": 384, "groups": 64, "k": 2048, "o": 1416, "skew": 0.3, "spare": 0, "bias": False,
         "dtype": "f16"},
        # Prompts through 64 experts, some 500 rows each.
        {"name": "experts_many", "op": "forward", "n": 32771, "groups": 64, "k": 1024, "o": 2048, "skew": 0.3, "spare": 0, "bias": False,
         "dtype": "f16"},
        # Long prompts through eight wide experts, in a buffer with room behind the last row.
        {"name": "experts_long", "op": "forward", "n": 16411, "groups": 8, "k": 2048, "o": 4096, "skew": 0.2, "spare": 500, "bias": True,
         "dtype": "bf16"},
        # Training: a small batch's gradients in widths that no tile divides, and a long one's.
        {"name": "dx_ragged", "op": "dx", "n": 4099, "groups": 16, "k": 1032, "o": 1416, "skew": 0.4, "spare": 0, "dtype": "f16"},
        {"name": "dx_long", "op": "dx", "n": 16411, "groups": 8, "k": 2048, "o": 4096, "skew": 0.2, "spare": 0, "dtype": "bf16"},
        {"name": "dw_ragged", "op": "dw", "n": 4099, "groups": 16, "k": 1032, "o": 1416, "skew": 0.4, "spare": 0, "bias": False, "out": "f16",
         "dtype": "f16"},
        {"name": "dw_long", "op": "dw", "n": 16411, "groups": 8, "k": 2048, "o": 4096, "skew": 0.2, "spare": 0, "bias": True, "out": "f32",
         "dtype": "bf16"},
        # One token of one request through its adapter and the layer that all share.
        {"name": "adapters_token", "op": "linear", "n": 1, "adapters": 8, "rank": 16, "k": 4096, "o": 4096, "requests": 1, "bias": False,
         "dtype": "bf16"},
        # Prompts of 24 requests.
        {"name": "adapters_prompts", "op": "linear", "n": 8209, "adapters": 16, "rank": 64, "k": 4096, "o": 4096, "requests": 24,
         "bias": True, "dtype": "bf16"},
        # Single tokens of 77 requests, in no order, beside a projection from 4-bit weights.
        {"name": "add_batch", "op": "add", "n": 77, "adapters": 32, "rank": 16, "k": 4096, "o": 4096, "requests": 77, "dtype": "bf16"},
        # Their prompts, in widths that no tile divides.
        {"name": "add_prompts", "op": "add", "n": 8209, "adapters": 32, "rank": 24, "k": 2080, "o": 4128, "requests": 40, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["forward", "forward", "dx", "dw", "linear", "add"])
    dt = rng.choice(["f16", "bf16"])
    k, o = 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512)
    if op in ("linear", "add"):
        n, rank, adapters = _log(rng, 1, min(16000, MOST // (k * o))), 8 * rng.randint(1, 8), _log(rng, 1, 64)
        case = {"op": op, "n": n, "adapters": adapters, "rank": rank, "k": k, "o": o,
                "requests": n if n <= 128 else rng.randint(1, 64), "dtype": dt}
        return {**case, "bias": rng.random() < 0.3} if op == "linear" else case
    groups = _log(rng, 1, max(1, min(128, (1 << 28) // (k * o))))
    case = {"op": op, "n": _log(rng, 1, min(32000, MOST // (k * o))), "groups": groups, "k": k, "o": o,
            "skew": round(rng.uniform(0, 0.4), 2), "spare": rng.choice([0, 0, rng.randint(1, 300)]), "dtype": dt}
    if op != "dx":
        case["bias"] = rng.random() < 0.3
    return {**case, "out": rng.choice(["f32", dt])} if op == "dw" else case


# ---- inputs ----------------------------------------------------------------------------------------------------


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _features(g, n, c, dt):
    """Activations: channels of unequal spread."""
    return (_rand(g, n, c) * torch.exp(0.3 * _rand(g, c))).to(dt)


def _weights(g, dt, count, o, k):
    return (_rand(g, count, o, k) / math.sqrt(k)).to(dt)


def _shares(case):
    """Each group's share of the rows, the largest first."""
    p = (torch.arange(case["groups"], dtype=torch.float64) + 1) ** -case["skew"]
    return p / p.sum()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op, n, k, o = DTYPES[case["dtype"]], case["op"], case["n"], case["k"], case["o"]
    s = {"case": case}
    if op in ("linear", "add"):
        count, rank = case["adapters"], case["rank"]
        s["x"] = _features(g, n, k, dt)
        s["a"], s["b"] = _weights(g, dt, count, rank, k), _weights(g, dt, count, o, rank)
        s["scale"] = torch.rand(count, generator=g, device="cuda") + 0.5
        cuts = torch.randint(0, n, (case["requests"] - 1,), generator=g, device="cuda").sort()[0]
        request = torch.searchsorted(cuts, torch.arange(n, device="cuda"), right=True)
        if case["requests"] == n:
            request = torch.arange(n, device="cuda")
        slot = torch.randint(0, count, (case["requests"],), generator=g, device="cuda")
        slot = torch.where(torch.rand(case["requests"], generator=g, device="cuda") < (0.1 if n > 1 else 0.0), -1, slot)
        s["slots"] = slot[request].int()
        if op == "linear":
            s["w"] = _weights(g, dt, 1, o, k)[0]
            s["bias"] = 0.1 * _rand(g, o) if case["bias"] else None
        else:
            s["y"] = _rand(g, n, o).to(dt)
        return s
    rows, groups = n + case["spare"], case["groups"]
    order = torch.randperm(groups, generator=g, device="cuda")
    group = order[torch.multinomial(_shares(case).cuda(), n, replacement=True, generator=g)]
    length = torch.bincount(group, minlength=groups)
    s["ends"], s["longest"] = length.cumsum(0).int(), int(length.max())
    if op != "dx":
        s["x"] = _features(g, rows, k, dt)
    if op != "forward":
        s["dy"] = _rand(g, rows, o).to(dt)
    if op != "dw":
        s["w"] = _weights(g, dt, groups, o, k)
        s["out"] = torch.full((rows, o if op == "forward" else k), 0.5, dtype=dt, device="cuda")
    s["bias"] = 0.1 * _rand(g, groups, o) if op == "forward" and case["bias"] else None
    return s


# ---- the plain form: 32 bits -----------------------------------------------------------------------------------


def _plain_adapters(s):
    case, x, slots, a, b = s["case"], s["x"].float(), s["slots"].long(), s["a"].float(), s["b"].float()
    n, count = case["n"], case["adapters"]
    y = s["y"].float() if case["op"] == "add" else x @ s["w"].float().T
    if s.get("bias") is not None:
        y = y + s["bias"]
    if n <= count:  # each row's own matrices
        at = slots.clamp_min(0)
        h = torch.bmm(a[at], x.unsqueeze(2)) * torch.where(slots >= 0, s["scale"][at], 0.0).view(n, 1, 1)
        return (y + torch.bmm(b[at], h).squeeze(2)).to(s["x"].dtype)
    h = (x @ a.view(-1, case["k"]).T).view(n, count, case["rank"])  # of every adapter, with those that are not the row's set to zero
    on = torch.where(slots.unsqueeze(1) == torch.arange(count, device=x.device), s["scale"], 0.0)
    return (y + (h * on.unsqueeze(2)).view(n, -1) @ b.transpose(1, 2).reshape(-1, case["o"])).to(s["x"].dtype)


def _plain_groups(s):
    case, ends, most = s["case"], s["ends"], s["longest"]
    n, groups, op = case["n"], case["groups"], case["op"]
    row = torch.arange(n, device=ends.device, dtype=torch.int32)
    g = torch.searchsorted(ends, row, right=True)
    at = g * most + row - torch.cat((ends.new_zeros(1), ends))[g]

    def by_group(t):  # [groups, longest, ...], zeros behind each group's rows
        return t.new_zeros((groups * most, t.shape[1]), dtype=torch.float32).index_copy(0, at, t[:n].float()).view(groups, most, -1)

    if op == "dw":
        dy = by_group(s["dy"])
        dw = torch.bmm(dy.transpose(1, 2).contiguous(), by_group(s["x"])).to(torch.float32 if case["out"] == "f32" else DTYPES[case["out"]])
        return (dw, dy.sum(1).to(dw.dtype)) if case["bias"] else dw
    t = s["x"] if op == "forward" else s["dy"]
    if n <= groups:  # each row's own weights
        w = s["w"][g].float()
        y = torch.bmm(w if op == "forward" else w.transpose(1, 2).contiguous(), t[:n].float().unsqueeze(2)).squeeze(2)
    else:
        w = s["w"].float()
        y = torch.bmm(by_group(t), w.transpose(1, 2).contiguous() if op == "forward" else w).view(groups * most, -1)[at]
    if s["bias"] is not None:
        y = y + s["bias"][g]
    s["out"][:n] = y.to(t.dtype)
    return s["out"]


# ---- the framework's operators ---------------------------------------------------------------------------------


def _own(s):
    import spconv_amd as sp

    op = s["case"]["op"]
    if op == "forward":
        return sp.group_linear(s["x"], s["w"], s["ends"], bias=s["bias"], out=s["out"])
    if op == "dx":
        return sp.group_linear_dx(s["dy"], s["w"], s["ends"], out=s["out"])
    if op == "dw":
        return sp.group_linear_dw(s["dy"], s["x"], s["ends"], out_dtype=torch.float32 if s["case"]["out"] == "f32" else None,
                                  bias=s["case"]["bias"])
    if op == "linear":
        return sp.adapter_linear(s["x"], s["w"], s["a"], s["b"], s["slots"], scale=s["scale"], bias=s["bias"])
    return sp.adapter_add(s["y"], s["x"], s["a"], s["b"], s["slots"], scale=s["scale"])


def run(state):
    if own:
        package = os.path.join(os.getcwd(), "trellis2-cuda_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        return _own(state)
    return _plain_adapters(state) if state["case"]["op"] in ("linear", "add") else _plain_groups(state)


# ---- 64 bits ---------------------------------------------------------------------------------------------------


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("linear", "add"):
        x = s["x"].double()
        y = s["y"].double() if op == "add" else torch.mm(x, s["w"].double().t())
        if s.get("bias") is not None:
            y += s["bias"].double()
        for i in range(case["adapters"]):
            rows = (s["slots"] == i).nonzero().squeeze(1)
            h = torch.mm(x[rows], s["a"][i].double().t())
            y[rows] += torch.mm(h, s["b"][i].double().t()) * s["scale"][i].double()
        return y
    bounds = [0] + s["ends"].tolist()
    if op == "dw":
        dw = torch.zeros((case["groups"], case["o"], case["k"]), dtype=torch.float64, device="cuda")
        db = torch.zeros((case["groups"], case["o"]), dtype=torch.float64, device="cuda")
        for i in range(case["groups"]):
            dy = s["dy"][bounds[i]:bounds[i + 1]].double()
            dw[i] = torch.mm(dy.t(), s["x"][bounds[i]:bounds[i + 1]].double())
            db[i] = dy.sum(0)
        return (dw, db) if case["bias"] else dw
    y = s["out"].double()
    for i in range(case["groups"]):
        rows = slice(bounds[i], bounds[i + 1])
        if op == "dx":
            y[rows] = torch.mm(s["dy"][rows].double(), s["w"][i].double())
        else:
            y[rows] = torch.mm(s["x"][rows].double(), s["w"][i].double().t())
            if s["bias"] is not None:
                y[rows] += s["bias"][i].double()
    return y


def work(case):
    n, k, o, op = case["n"], case["k"], case["o"], case["op"]
    if op in ("linear", "add"):
        rank = case["rank"]
        used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** case["requests"])  # adapters that some request has
        base = 2 * n * o if op == "add" else 2 * k * o + (4 * o if case["bias"] else 0)
        return {"bytes": int(2 * n * (k + o) + base + 2 * used * rank * (k + o) + 4 * n),
                "flops": 2 * n * rank * (k + o) + (0 if op == "add" else 2 * n * k * o)}
    used = float((1 - (1 - _shares(case)) ** n).sum())  # groups that have a row
    if op == "dw":
        size = 4 if case["out"] == "f32" else 2
        return {"bytes": 2 * n * (k + o) + size * case["groups"] * o * (k + (1 if case["bias"] else 0)),
                "flops": 2 * n * k * o + (n * o if case["bias"] else 0)}
    return {"bytes": int(2 * n * (k + o) + 2 * used * k * o + (4 * used * o if case.get("bias") else 0)), "flops": 2 * n * k * o}
