"""What a recurrent language model learns with, as measurable cases: the operators in plain torch and through this package.

A case is a dict of plain values.  ``op`` names the public entry points:

* ``scan``    the gated linear recurrence over prompts (``hip_ops.gated_scan``, ``gated_scan_backward``), dense or packed
* ``step``    one token through it (``hip_ops.gated_scan_step``), the state updated in place
* ``gated``   a feed-forward block's two projections, activation and product (``hip_ops.gated_linear``, ``.._backward``)
* ``linear``  a projection with bias, activation and residual (``hip_ops.fused_linear``, ``.._backward``)
* ``logp``    given tokens' log probabilities, the rows' entropies and best alternatives (``hip_ops.token_log_probs``,
  ``.._backward``)

With ``train`` a pass is the operator and its backward pass, and its outputs are the result and every gradient.  Layer sizes are
those of the ``TESMConfig`` presets (d_model, d_intermediate, states of all heads); the vocabulary is the configuration's.  Packed
prompts lie one behind the other in one row axis; ``tail`` rows follow the last sequence, as in a batch padded to a fixed size, and
hold zeros in every output.
"""
from __future__ import annotations

import math
import random

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 151936


def listed():
    return [
        # one short prompt through a base layer's recurrence: latency
        dict(name="scan_short", op="scan", dtype="bf16", B=1, L=37, C=384, packed=0, tail=0, init=False, train=False),
        # a base layer's recurrence over a full training batch
        dict(name="scan_base", op="scan", dtype="bf16", B=4, L=2048, C=384, packed=0, tail=0, init=False, train=True),
        # ragged sequences continued from earlier ones, float32, a channel count that no vector width divides
        dict(name="scan_packed_f32", op="scan", dtype="f32", B=11, L=1500, C=333, packed=1, tail=3, init=True, train=True),
        # all heads of a large layer on one long sequence: the largest call
        dict(name="scan_long", op="scan", dtype="bf16", B=1, L=32768, C=8192, packed=0, tail=0, init=True, train=True),
        # one token for each of 64 sequences, a large layer
        dict(name="step_large", op="step", dtype="bf16", B=64, C=8192),
        # one token of one sequence through a base layer's feed-forward: the smallest product
        dict(name="gated_one", op="gated", dtype="bf16", M=1, K=768, F=2048, act="silu", train=False),
        # a base layer's feed-forward over a full training batch
        dict(name="gated_base", op="gated", dtype="bf16", M=8192, K=768, F=2048, act="silu", train=True),
        # float32 and odd sizes throughout
        dict(name="gated_odd_f32", op="gated", dtype="f32", M=999, K=515, F=1030, act="gelu", train=True),
        # the projection back into the residual stream over a full training batch
        dict(name="linear_base", op="linear", dtype="bf16", M=8192, K=2048, N=768, act=None, bias=True, residual=True, train=True),
        # a large layer's widest projection over a prompt
        dict(name="linear_large", op="linear", dtype="bf16", M=8192, K=4096, N=16384, act="gelu", bias=True, residual=False,
             train=False),
        # one generated token's log probability and its 20 best alternatives: latency
        dict(name="logp_one", op="logp", dtype="bf16", rows=1, V=VOCAB, top=20, ignored=0.0, banned=0.0, train=False),
        # the loss of a full training batch, padding among it
        dict(name="logp_train", op="logp", dtype="bf16", rows=8192, V=VOCAB, top=0, ignored=0.1, banned=0.0, train=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ones' ranges: any operator, sizes over their logarithm, odd ones among them."""
    op = rng.choice(["scan", "scan", "scan", "step", "gated", "gated", "linear", "linear", "logp", "logp"])
    dtype = "f32" if rng.random() < 0.3 else "bf16"
    train = rng.random() < 0.6
    if op == "scan":
        B = _log(rng, 1, 16)
        C = rng.choice([256, 384, 512, 1536, 8192, _log(rng, 1, 2000), _log(rng, 1, 2000)])
        packed = rng.randint(0, 1)
        return dict(op=op, dtype=dtype, B=B, L=_log(rng, rng.choice([1, 64, 512]), max(600, min(32768 // B, 60000000 // (B * C)))),
                    C=C, packed=packed, tail=rng.randint(0, 9) * packed, init=rng.random() < 0.5, train=train)
    if op == "step":
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 256), C=rng.choice([256, 384, 512, 8192, _log(rng, 1, 4000)]))
    if op in ("gated", "linear"):
        K = rng.choice([256, 512, 768, 1024, 2048, _log(rng, 8, 2500), _log(rng, 8, 2500)])
        N = rng.choice([512, 768, 1536, 2048, 2816, _log(rng, 8, 2500), _log(rng, 8, 2500)])
        M = _log(rng, 1, 16384) if train or rng.random() < 0.5 else _log(rng, 1, 64)
        if op == "gated":
            return dict(op=op, dtype=dtype, M=M, K=K, F=N, act=rng.choice(["silu", "silu", "gelu"]), train=train)
        return dict(op=op, dtype=dtype, M=M, K=K, N=N, act=rng.choice([None, None, "silu", "gelu"]), bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5, train=train)
    V = rng.choice([VOCAB, VOCAB, _log(rng, 500, VOCAB)])
    top = 0 if train or rng.random() < 0.4 else rng.choice([1, 5, 20, 64])
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 512 if top else 3000), V=V, top=top, ignored=rng.choice([0.0, 0.3]),
                banned=rng.choice([0.0, 0.0, 0.3]), train=train)


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    if math.prod(shape) > 1 << 28:  # (in parts: no float32 copy of the largest ones)
        return torch.stack([_randn(g, *shape[1:], dtype=dtype) for _ in range(shape[0])])
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _lengths(case):
    """The lengths of a packed case's sequences: ragged, from a single row up; from the case alone."""
    r = random.Random(case["B"] * 1000003 + case["L"])
    return [1 if i == 1 else r.randint(max(1, case["L"] // 8), case["L"]) for i in range(case["B"])]


def _starts(case):
    at = [0]
    for n in _lengths(case):
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=dict(case))
    if op != "logp":
        dtype = DTYPES[case["dtype"]]
    if op == "scan":
        C = case["C"]
        s["seq_starts"] = None
        lead = (case["B"], case["L"])
        if case["packed"]:
            at = _starts(case)
            s["seq_starts"] = torch.tensor(at, dtype=torch.int32, device="cuda")
            lead = (1, at[-1] + case["tail"])
        # the gates before their activations as a projection leaves them; biases that keep a state for 3 to 400 tokens
        s["value"], s["write"], s["decay"] = (_randn(g, *lead, C, dtype=dtype) for _ in range(3))
        s["bias"] = 1 + 5 * torch.rand(C, generator=g, device="cuda")
        s["h0"] = 0.5 * _randn(g, case["B"], C) if case["init"] else None
        if case["train"]:
            s["grad"] = _randn(g, *lead, C, dtype=dtype)
            s["grad_state"] = _randn(g, case["B"], C) if case["init"] else None
    elif op == "step":
        s["value"], s["write"], s["decay"] = (_randn(g, case["B"], case["C"], dtype=dtype) for _ in range(3))
        s["bias"] = 1 + 5 * torch.rand(case["C"], generator=g, device="cuda")
        s["h"] = 0.5 * _randn(g, case["B"], case["C"])
    elif op in ("gated", "linear"):
        M, K, N = case["M"], case["K"], case["F" if op == "gated" else "N"]
        s["x"] = _randn(g, M, K, dtype=dtype)
        if op == "gated":
            s["wg"], s["wu"] = ((_randn(g, N, K) / math.sqrt(K)).to(dtype) for _ in range(2))
        else:
            s["w"] = (_randn(g, N, K) / math.sqrt(K)).to(dtype)
            s["b"] = (0.3 * _randn(g, N)).to(dtype) if case["bias"] else None
            s["r"] = _randn(g, M, N, dtype=dtype) if case["residual"] else None
        if case["train"]:
            s["grad"] = _randn(g, M, N, dtype=dtype)
    else:
        rows, V = case["rows"], case["V"]
        s["logits"] = torch.empty(rows, V, dtype=DTYPES[case["dtype"]], device="cuda")
        banned = torch.rand(V, generator=g, device="cuda") < case["banned"]
        for i in range(0, rows, 1024):
            part = s["logits"][i:i + 1024]
            part.copy_((2.5 * torch.randn(part.shape, generator=g, device="cuda")).masked_fill_(banned, -math.inf))
        targets = torch.randint(0, V, (rows,), generator=g, device="cuda")
        allowed = torch.nonzero(~banned)[:, 0]
        if allowed.numel():  # no target among the masked tokens
            targets = allowed[targets % allowed.numel()]
        drop = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        s["targets"] = targets.masked_fill_(drop, -100)
        if case["train"]:  # a mean's gradient for the log probabilities, a small bonus for the entropies
            s["grad"] = -torch.rand(rows, generator=g, device="cuda") / rows
            s["grad_entropy"] = 0.01 * torch.rand(rows, generator=g, device="cuda") / rows
    return s


# ------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"scan": _scan, "step": _step, "gated": _gated, "linear": _linear, "logp": _logp}[op](s)
    from tesm_amd import hip_ops
    train = case.get("train", False)
    if op == "scan":
        gates = (s["value"], s["write"], s["decay"], s["bias"])
        how = dict(state=s["h0"], seq_starts=s["seq_starts"])
        if not train:
            return hip_ops.gated_scan(*gates, **how)
        h, state, kept = hip_ops.gated_scan(*gates, keep=True, **how)
        return (h, state) + tuple(hip_ops.gated_scan_backward(s["grad"], *gates, kept=kept, grad_state=s["grad_state"], **how))
    if op == "step":
        return hip_ops.gated_scan_step(s["value"], s["write"], s["decay"], s["bias"], state=s["h"]), s["h"]
    if op == "gated":
        args = (s["x"], s["wg"], s["wu"])
        if not train:
            return hip_ops.gated_linear(*args, act=case["act"])
        h, kept = hip_ops.gated_linear(*args, act=case["act"], keep=True)
        return (h,) + tuple(hip_ops.gated_linear_backward(s["grad"], *args, kept=kept, act=case["act"]))
    if op == "linear":
        how = dict(act=case["act"], residual=s["r"])
        if not train:
            return hip_ops.fused_linear(s["x"], s["w"], s["b"], **how)
        y, kept = hip_ops.fused_linear(s["x"], s["w"], s["b"], keep=True, **how)
        return (y,) + tuple(hip_ops.fused_linear_backward(s["grad"], s["x"], s["w"], s["b"], kept=kept, act=case["act"]))
    if not train:
        return hip_ops.token_log_probs(s["logits"], s["targets"], top=case["top"])
    logp, entropy, _, _, kept = hip_ops.token_log_probs(s["logits"], s["targets"], keep=True)
    return logp, entropy, hip_ops.token_log_probs_backward(s["grad"], s["grad_entropy"], s["logits"], s["targets"], kept=kept)


def _shifted(t, n, fill):
    """Row t - n (n < 0: row t + |n|) in row t's place, ``fill`` where there is none; rows are the second axis."""
    pad = torch.full_like(t[:, :abs(n)], fill)
    return torch.cat([pad, t[:, :-n]] if n > 0 else [t[:, -n:], pad], 1)


def _recur(a, u, sign):
    """h_t = a_t h_(t -/+ 1) + u_t over the second axis, by doubling: after n rounds h_t holds 2^n rows' terms."""
    n = 1
    while n < a.shape[1]:
        u = u + a * _shifted(u, sign * n, 0.0)
        n *= 2
        if n < a.shape[1]:
            a = a * _shifted(a, sign * n // 2, 1.0)
    return u


def _spread(s):
    """Where a packed case's rows lie in a (sequences, longest) batch, and the real rows."""
    case = s["case"]
    at = s["seq_starts"].long()
    rows = torch.arange(_starts(case)[-1], device="cuda")
    seq = torch.searchsorted(at, rows, right=True) - 1
    return rows, seq, rows - at[seq]


def _scan(s):
    case = s["case"]
    dtype, B, C = s["value"].dtype, case["B"], case["C"]
    if case["packed"]:
        rows, seq, place = _spread(s)
        longest = max(_lengths(case))

        def wide(t, fill=0.0):
            out = torch.full((B, longest, C), fill, device="cuda")
            out[seq, place] = t[0, rows].float()
            return out

        def back(t):
            out = torch.zeros(s["value"].shape, dtype=dtype, device="cuda")
            out[0, rows] = t[seq, place].to(dtype)
            return out
        real = wide(torch.ones_like(s["value"]))
    else:
        def wide(t, fill=0.0):
            return t.float()

        def back(t):
            return t.to(dtype)
        real = None
    v, w, f = wide(s["value"]).tanh(), torch.sigmoid(wide(s["write"])), wide(s["decay"]) + s["bias"]
    a, u = torch.sigmoid(f), w * v
    if real is not None:  # behind a sequence's end the state stays
        a, u = a * real + (1 - real), u * real
    if s["h0"] is not None:
        u = torch.cat([u[:, :1] + a[:, :1] * s["h0"][:, None], u[:, 1:]], 1)
    h = _recur(a, u, 1)
    state = h[:, -1].contiguous()
    if not case["train"]:
        return back(h), state
    g = wide(s["grad"])
    if s["grad_state"] is not None:
        g = torch.cat([g[:, :-1], g[:, -1:] + s["grad_state"][:, None]], 1)
    g = _recur(_shifted(a, -1, 0.0), g, -1)
    first = s["h0"][:, None] if s["h0"] is not None else torch.zeros_like(h[:, :1])
    before = torch.cat([first, h[:, :-1]], 1)
    df = g * before * a * torch.sigmoid(-f)
    if real is not None:
        df = df * real
    out = [back(h), state, back(g * w * (1 - v * v)), back(g * v * w * (1 - w)), back(df), df.double().sum((0, 1)).float()]
    return out + [(a[:, 0] * g[:, 0]) if s["h0"] is not None else None]


def _step(s):
    a = torch.sigmoid(s["decay"].float() + s["bias"])
    s["h"].copy_(a * s["h"] + torch.sigmoid(s["write"].float()) * s["value"].float().tanh())
    return s["h"].to(s["value"].dtype), s["h"]


def _act(z, act):
    """The activation and its derivative."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _gated(s):
    case, dtype = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    gate, up = x @ wg.t(), x @ wu.t()
    value, slope = _act(gate, case["act"])
    h = (value * up).to(dtype)
    if not case["train"]:
        return h
    d = s["grad"].float()
    dg, du = d * up * slope, d * value
    return h, (dg @ wg + du @ wu).to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype)


def _linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    value, slope = _act(z, case["act"])
    y = (value if s["r"] is None else value + s["r"].float()).to(dtype)
    if not case["train"]:
        return y
    dz = s["grad"].float() * slope
    db = None if s["b"] is None else dz.double().sum(0).to(dtype)
    return y, (dz @ w).to(dtype), (dz.t() @ x).to(dtype), db


def _ordered(x):
    """32-bit values as whole numbers of the same order."""
    b = (x + 0.0).view(torch.int32).long()
    return torch.where(b < 0, -(b & 0x7fffffff), b)


def _logp(s):
    case, logits = s["case"], s["logits"].float()
    rows, V = logits.shape
    known = s["targets"] != -100
    at = s["targets"].clamp(min=0)[:, None]
    far = logits - logits.amax(-1, keepdim=True)
    e = far.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    logp = torch.where(known, (far.gather(1, at) - lse)[:, 0], 0.0)
    entropy = (lse - (e * far.clamp(min=-1e4)).sum(-1, keepdim=True) / total)[:, 0]
    if case["train"]:
        p = e / total
        g = torch.where(known, s["grad"], 0.0)[:, None]
        d = -p * (g + s["grad_entropy"][:, None] * ((far - lse).clamp(min=-1e4) + entropy[:, None]))
        d.scatter_add_(1, at, g)
        return logp, entropy, d.to(s["logits"].dtype)
    if not case["top"]:
        return logp, entropy, None, None
    place = torch.arange(V, device="cuda")
    best = ((_ordered(logits) << 32) - place).topk(case["top"], -1).values  # equal ones: the lower index first
    tokens = (-best) & 0xffffffff
    return logp, entropy, far.gather(1, tokens) - lse, tokens


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------
def work(case):
    op, size = case["op"], 2 if case["dtype"] == "bf16" else 4
    train = case.get("train", False)
    if op == "step":
        return {"bytes": case["B"] * case["C"] * (4 * size + 8) + 4 * case["C"], "flops": 20 * case["B"] * case["C"]}
    if op == "scan":
        M = sum(_lengths(case)) if case["packed"] else case["B"] * case["L"]
        states = case["B"] * case["C"] * ((4 if train else 2) if case["init"] else 1)
        return {"bytes": case["C"] * (size * M * (8 if train else 4) + (8 if train else 4)) + 4 * states,
                "flops": M * case["C"] * (60 if train else 20)}
    if op == "logp":
        n = case["rows"] * case["V"]
        return {"bytes": size * n * (2 if train else 1) + case["rows"] * (16 + (8 if train else 0) + 12 * case["top"]),
                "flops": n * (14 if train else 6)}
    M, K = case["M"], case["K"]
    if op == "gated":
        N = case["F"]
        return {"bytes": size * (M * K + 2 * N * K + M * N) * (2 if train else 1), "flops": 4 * M * K * N * (3 if train else 1)}
    N = case["N"]
    return {"bytes": size * ((M * K + N * K + M * N + N * case["bias"]) * (2 if train else 1) + M * N * case["residual"]),
            "flops": 2 * M * K * N * (3 if train else 1)}


# ------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "step": _exact_step, "gated": _exact_gated, "linear": _exact_linear, "logp": _exact_logp}[case["op"]](s)


def _half_tanh(x):
    """1 / (1 + e^-x), from the hyperbolic tangent of half the argument."""
    return (1 + torch.tanh(x / 2)) / 2


def _exact_scan(s):
    """Row by row, forwards and backwards; a batch's sequences side by side, packed ones one by one."""
    case = s["case"]
    C, train = case["C"], case["train"]
    shape = s["value"].shape
    if case["packed"]:
        at = _starts(case)
        parts = [(slice(0, 1), slice(at[i], at[i + 1]), slice(i, i + 1)) for i in range(case["B"])]
    else:
        parts = [(slice(None), slice(None), slice(None))]
    hs = torch.zeros(shape, dtype=torch.float64, device="cuda")
    last = torch.zeros(case["B"], C, dtype=torch.float64, device="cuda")
    if train:
        dv, dw, df = (torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(3))
        db, dh0 = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros_like(last)
    for b, t, seq in parts:
        keep = _half_tanh(s["decay"][b, t].double() + s["bias"].double())
        add = _half_tanh(s["write"][b, t].double()) * torch.tanh(s["value"][b, t].double())
        h = s["h0"][seq].double() if s["h0"] is not None else torch.zeros_like(last[seq])
        first, mine = h, hs[b, t]
        for i in range(keep.shape[1]):
            torch.addcmul(add[:, i], keep[:, i], h, out=mine[:, i])
            h = mine[:, i]
        last[seq] = h
        if not train:
            continue
        g = s["grad"][b, t].double()
        if s["grad_state"] is not None:
            g[:, -1] += s["grad_state"][seq].double()
        for i in range(keep.shape[1] - 2, -1, -1):
            g[:, i].addcmul_(keep[:, i + 1], g[:, i + 1])
        dh0[seq] = keep[:, 0] * g[:, 0]
        gate, val = _half_tanh(s["write"][b, t].double()), torch.tanh(s["value"][b, t].double())
        dv[b, t] = g * gate / torch.cosh(s["value"][b, t].double()) ** 2
        dw[b, t] = g * val * gate * _half_tanh(-s["write"][b, t].double())
        del gate, val, add
        slope = keep * _half_tanh(-s["decay"][b, t].double() - s["bias"].double())
        df[b, t] = g * slope * torch.cat([first[:, None], mine[:, :-1]], 1)
        db += df[b, t].sum((0, 1))
    if not train:
        return hs, last
    return [hs, last, dv, dw, df, db, dh0 if s["h0"] is not None else None]


def _exact_step(s):
    keep = _half_tanh(s["decay"].double() + s["bias"].double())
    h = keep * s["h"].double() + _half_tanh(s["write"].double()) * torch.tanh(s["value"].double())
    return h, h


def _exact_act(z, act):
    if act is None:
        return z, 1.0
    if act == "silu":
        p = _half_tanh(z)
        return z * p, p + z * p * _half_tanh(-z)
    p = torch.erfc(-z / math.sqrt(2)) / 2
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _exact_gated(s):
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    gate, up = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    value, slope = _exact_act(gate, s["case"]["act"])
    if not s["case"]["train"]:
        return value * up
    d = s["grad"].double()
    dg, du = d * slope * up, d * value
    return value * up, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.t(), x), torch.mm(du.t(), x)


def _exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.mm(x, w.t())
    if s["b"] is not None:
        z += s["b"].double()
    value, slope = _exact_act(z, s["case"]["act"])
    y = value + s["r"].double() if s["r"] is not None else value
    if not s["case"]["train"]:
        return y
    dz = s["grad"].double() * slope
    return y, torch.mm(dz, w), torch.mm(dz.t(), x), (dz.sum(0) if s["b"] is not None else None)


def _exact_logp(s):
    case = s["case"]
    rows, V = s["logits"].shape
    outs = []
    for i in range(0, rows, 256):
        x, t = s["logits"][i:i + 256].double(), s["targets"][i:i + 256]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        p = lp.exp()
        lp = torch.where(p > 0, lp, lp.clamp(min=-1e6))
        entropy = -(p * lp).sum(-1)
        mine = t >= 0
        token = lp[torch.arange(len(t), device="cuda"), t.clamp(min=0)] * mine
        out = [token, entropy]
        if case["train"]:
            g, ge = s["grad"][i:i + 256].double() * mine, s["grad_entropy"][i:i + 256].double()
            d = -p * g[:, None] - ge[:, None] * p * (lp + entropy[:, None])
            d[torch.arange(len(t), device="cuda"), t.clamp(min=0)] += g
            out.append(d.to(torch.float32) if rows * V > 1 << 28 else d)  # (24 bits of a result that is held in 8)
        elif case["top"]:
            out.append(lp.sort(-1, descending=True).values[:, :case["top"]])
        outs.append(out)
    done = [torch.cat(c) for c in zip(*outs)]
    if case["train"]:
        return done
    return done + [None, None] if not case["top"] else done + [None]
