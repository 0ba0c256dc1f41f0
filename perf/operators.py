"""Recurrent states from a prompt to a beam search, as measurable cases: the operators in plain torch and through this package.

A case is a dict of plain values.  ``op`` names the public entry points:

* ``conv``     the short causal convolution over prompts (``hip_ops.causal_conv``), dense or packed
* ``scan``     the selective state space scan over prompts (``hip_ops.selective_scan``), dense or packed
* ``step``     one token through both (``hip_ops.selective_scan_step``), the scan's state updated in place
* ``select``   a beam search's choice over beams and vocabulary (``hip_ops.beam_select``)
* ``reorder``  the inference caches of all layers moved to their new beams (``hip_ops.reorder_rows``)

Layer sizes are those of the ``TESMConfig`` presets with an inner width of twice d_model, heads of 64 channels and 128 states;
the vocabulary is the configuration's.  Packed prompts lie one behind the other in one row axis; ``tail`` rows follow the last
sequence, as in a batch padded to a fixed size, and stay as they are.
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
        # the convolution of a base layer over a full batch of prompts
        dict(name="conv_base", op="conv", dtype="bf16", B=4, L=2048, C=1792, W=4, packed=0, tail=0, init=False),
        # ragged prompts continued from earlier ones, float32, a channel count that no vector width divides
        dict(name="conv_packed_f32", op="conv", dtype="f32", B=9, L=2600, C=1153, W=3, packed=1, tail=5, init=True),
        # one short prompt, a base layer: latency
        dict(name="scan_short", op="scan", dtype="bf16", B=1, L=37, H=24, P=64, G=1, N=128, packed=0, tail=0, init=False, gate=True),
        # a base layer over a full batch of prompts
        dict(name="scan_base", op="scan", dtype="bf16", B=4, L=2048, H=24, P=64, G=1, N=128, packed=0, tail=0, init=False, gate=True),
        # ragged prompts continued from earlier ones, float32, odd head and state sizes
        dict(name="scan_packed_f32", op="scan", dtype="f32", B=11, L=1500, H=10, P=40, G=2, N=56, packed=1, tail=3, init=True, gate=True),
        # a large layer on one long prompt: the largest call
        dict(name="scan_long", op="scan", dtype="bf16", B=1, L=32768, H=128, P=64, G=8, N=128, packed=0, tail=0, init=True, gate=True),
        # one token of one sequence, a base layer: the smallest call, launch bound
        dict(name="step_one", op="step", dtype="bf16", B=1, H=24, P=64, G=1, N=128, W=4),
        # one token for each of 64 sequences, a large layer
        dict(name="step_large", op="step", dtype="bf16", B=64, H=128, P=64, G=8, N=128, W=4),
        # four beams of one request: latency
        dict(name="select_one", op="select", dtype="bf16", B=1, K=4, V=VOCAB, n=4, finished=False, banned=0.0, first=False),
        # eight beams of 64 requests, some of them finished
        dict(name="select_large", op="select", dtype="bf16", B=64, K=8, V=VOCAB, n=8, finished=True, banned=0.0, first=False),
        # the caches of the tiny() model, four beams of one request
        dict(name="reorder_tiny", op="reorder", kind="ring", layers=12, B=1, K=4, D=384, W=16, R=96),
        # the caches of the medium() model, eight beams of 16 requests
        dict(name="reorder_medium", op="reorder", kind="ring", layers=32, B=16, K=8, D=512, W=32, R=80),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ones' ranges: any operator, sizes over their logarithm, odd ones among them."""
    op = rng.choice(["conv", "scan", "scan", "scan", "step", "step", "select", "select", "reorder"])
    dtype = "f32" if rng.random() < 0.3 else "bf16"
    packed = rng.randint(0, 1)
    if op == "conv":
        B = _log(rng, 1, 16)
        C = rng.choice([1792, 2304, 10240, _log(rng, 8, 4096), _log(rng, 8, 4096)])
        return dict(op=op, dtype=dtype, B=B, L=_log(rng, 1, 32768 // B), C=C, W=rng.choice([2, 3, 4, 4, 4, 6]), packed=packed,
                    tail=rng.randint(0, 9) * packed, init=rng.random() < 0.5)
    if op == "scan":
        B = _log(rng, 1, 16)
        G = rng.choice([1, 1, 2, 4, 8])
        H = G * _log(rng, 1, 64 // G)
        P = rng.choice([64, 64, 64, 32, 128, rng.randint(8, 96)])
        N = rng.choice([128, 128, 64, 16, 256, rng.randint(5, 200)])
        most = int(4e9 / (H * P * N * B))  # a third of the largest listed one's states
        return dict(op=op, dtype=dtype, B=B, L=_log(rng, rng.choice([1, 64, 64]), max(65, min(16384 // B, most))), H=H, P=P, G=G, N=N, packed=packed,
                    tail=rng.randint(0, 9) * packed, init=rng.random() < 0.5, gate=rng.random() < 0.7)
    if op == "step":
        G = rng.choice([1, 1, 2, 8])
        H = G * _log(rng, 1, 128 // G)
        P = rng.choice([64, 64, 128, rng.randint(8, 96)])
        N = rng.choice([128, 128, 64, 16, 256, rng.randint(5, 200)])
        B = _log(rng, 1, max(1, min(128, int(6.7e7 / (H * P * N)))))
        return dict(op=op, dtype=dtype, B=B, H=H, P=P, G=G, N=N, W=rng.choice([2, 4, 4]))
    if op == "select":
        K = rng.choice([1, 2, 3, 4, 5, 8, 16])
        first = rng.random() < 0.2
        V = rng.choice([VOCAB, VOCAB, _log(rng, 500, VOCAB)])
        return dict(op=op, dtype=dtype, B=_log(rng, 1, max(1, (256 if dtype == "f32" else 512) // K)), K=K, V=V,
                    n=K * rng.choice([1, 1, 2]), finished=not first and rng.random() < 0.5,
                    banned=rng.choice([0.0, 0.0, 0.3]), first=first)
    kind = rng.choice(["ring", "ring", "scan"])
    K = rng.choice([2, 3, 4, 5, 8])
    layers = _log(rng, 2, 32)
    B = _log(rng, 1, max(1, 128 // K))
    if kind == "scan":
        layers = min(layers, max(2, 800 // (B * K)))
        return dict(op=op, kind=kind, layers=layers, B=B, K=K, H=_log(rng, 1, 24), P=64, N=128, C=_log(rng, 100, 1792), W=4)
    return dict(op=op, kind=kind, layers=layers, B=B, K=K, D=rng.choice([256, 384, 512, rng.randint(3, 500)]),
                W=rng.choice([1, 16, 32]), R=rng.choice([32, 64, 80, 96]))


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float64 if dtype == torch.float64 else torch.float32).to(dtype)


def _lengths(case):
    """The lengths of a packed case's sequences: ragged, from a single row up, ``B * L / 2`` rows or so in all; from the case alone."""
    r = random.Random(case["B"] * 1000003 + case["L"])
    return [1 if i == 1 else r.randint(max(1, case["L"] // 8), case["L"]) for i in range(case["B"])]


def _starts(case):
    at = [0]
    for n in _lengths(case):
        at.append(at[-1] + n)
    return at


def _layer_params(g, H):
    """Step sizes between 1e-3 and 1e-1 (their inverse softplus is the bias), decay rates 1 .. 16, a skip around 1."""
    size = torch.exp(torch.rand(H, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    return dict(A=-(1 + 15 * torch.rand(H, generator=g, device="cuda")), dt_bias=size + torch.log(-torch.expm1(-size)),
                D=1 + 0.2 * _randn(g, H))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=dict(case))
    if op in ("conv", "scan"):
        dtype = DTYPES[case["dtype"]]
        if case["packed"]:
            at = _starts(case)
            s["seq_starts"] = torch.tensor(at, dtype=torch.int32, device="cuda")
            lead = (1, at[-1] + case["tail"])
        else:
            s["seq_starts"] = None
            lead = (case["B"], case["L"])
    if op == "conv":
        C, W = case["C"], case["W"]
        s["x"] = _randn(g, *lead, C, dtype=dtype)
        s["weight"] = (_randn(g, C, W) / math.sqrt(W)).to(dtype)
        s["bias"] = (0.1 * _randn(g, C)).to(dtype)
        s["state"] = _randn(g, case["B"], W - 1, C, dtype=dtype) if case["init"] else None
        s["out"] = torch.zeros(*lead, C, dtype=dtype, device="cuda")
    elif op == "scan":
        H, P, G, N = case["H"], case["P"], case["G"], case["N"]
        # x, B and C as the convolution leaves them: slices of one row
        row = F.silu(_randn(g, *lead, H * P + 2 * G * N)).to(dtype)
        s["x"] = row[..., :H * P].unflatten(-1, (H, P))
        s["B"] = row[..., H * P:H * P + G * N].unflatten(-1, (G, N))
        s["C"] = row[..., H * P + G * N:].unflatten(-1, (G, N))
        s["dt"] = _randn(g, *lead, H, dtype=dtype)
        s["z"] = _randn(g, *lead, H, P, dtype=dtype) if case["gate"] else None
        s.update(_layer_params(g, H))
        s["h0"] = 0.3 * _randn(g, case["B"], H, P, N) if case["init"] else None
        s["out"] = torch.zeros(*lead, H, P, dtype=dtype, device="cuda")
    elif op == "step":
        dtype = DTYPES[case["dtype"]]
        B, H, P, G, N, W = (case[k] for k in ("B", "H", "P", "G", "N", "W"))
        C = H * P + 2 * G * N
        s["row"] = _randn(g, B, C, dtype=dtype)
        s["weight"] = (_randn(g, C, W) / math.sqrt(W)).to(dtype)
        s["bias"] = (0.1 * _randn(g, C)).to(dtype)
        s["conv_state"] = _randn(g, B, W - 1, C, dtype=dtype)
        s["dt"] = _randn(g, B, H, dtype=dtype)
        s["z"] = _randn(g, B, H, P, dtype=dtype)
        s.update(_layer_params(g, H))
        s["h"] = 0.3 * _randn(g, B, H, P, N)
    elif op == "select":
        dtype = DTYPES[case["dtype"]]
        B, K, V = case["B"], case["K"], case["V"]
        logits = 2.5 * _randn(g, B, K, V)
        if case["banned"]:
            logits.masked_fill_(torch.rand(V, generator=g, device="cuda") < case["banned"], -math.inf)
        s["logits"] = logits.to(dtype)
        s["scores"] = -4 * torch.rand(B, K, generator=g, device="cuda") - 10
        if case["first"]:  # the first token: all beams are the same, only beam 0 counts
            s["logits"] = s["logits"][:, :1].expand(B, K, V).contiguous()
            s["scores"][:, 1:] = -math.inf
        s["finished"] = torch.rand(B, K, generator=g, device="cuda") < 0.25 if case["finished"] else None
    else:
        n, rows, K = case["layers"], case["B"] * case["K"], case["K"]
        if case["kind"] == "ring":
            s["all"] = [_randn(g, n, rows, case["D"], dtype=torch.float64), _randn(g, n, rows, case["W"], case["R"]),
                        _randn(g, n, rows, case["W"], case["D"])]
        else:
            s["all"] = [_randn(g, n, rows, case["H"], case["P"], case["N"]),
                        _randn(g, n, rows, case["W"] - 1, case["C"], dtype=torch.bfloat16)]
        s["caches"] = [t[i] for t in s["all"] for i in range(n)]
        s["parents"] = torch.randint(0, K, (case["B"], K), generator=g, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from tesm_amd import hip_ops
        if op == "conv":
            return hip_ops.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], seq_starts=s["seq_starts"], out=s["out"])
        if op == "scan":
            return hip_ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                          state=s["h0"], seq_starts=s["seq_starts"], out=s["out"])
        if op == "step":
            y, conv_state = hip_ops.selective_scan_step(s["row"], s["dt"], s["A"], s["h"], s["weight"], s["bias"], s["conv_state"],
                                                        n_groups=case["G"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
            return y, s["h"], conv_state
        if op == "select":
            return hip_ops.beam_select(s["logits"], s["scores"], case["n"], finished=s["finished"], pad_token=0)[:3]
        hip_ops.reorder_rows(s["caches"], s["parents"])
        return s["all"]
    return {"conv": _conv, "scan": _scan, "step": _step, "select": _select, "reorder": _reorder}[op](s)


def _positions(s, B, L, M):
    """For every row of the flattened row axis: its sequence and its place in it; (rows, sequences, places) of the real rows."""
    rows = torch.arange(M, device="cuda")
    if s["seq_starts"] is None:
        return rows, rows // L, rows % L
    at = s["seq_starts"].long()
    rows = rows[:_starts(s["case"])[-1]]
    seq = torch.searchsorted(at, rows, right=True) - 1
    return rows, seq, rows - at[seq]


def _conv(s):
    case, x = s["case"], s["x"]
    B, C, W = case["B"], case["C"], case["W"]
    flat = x.reshape(-1, C)
    M = flat.shape[0]
    before = s["state"] if s["state"] is not None else torch.zeros(B, W - 1, C, dtype=x.dtype, device="cuda")
    rows, seq, place = _positions(s, B, case["L"], M)
    table = torch.cat([flat, before.reshape(-1, C)])
    back = torch.arange(W, device="cuda") - (W - 1)
    src = place[:, None] + back
    src = torch.where(src >= 0, rows[:, None] + back, M + seq[:, None] * (W - 1) + (W - 1) + src)
    y = (table[src].float() * s["weight"].float().t()).sum(1) + s["bias"].float()
    s["out"].view(-1, C)[:rows.numel()] = F.silu(y).to(x.dtype)
    # the last W - 1 inputs of every sequence
    n = torch.bincount(seq, minlength=B)
    end = torch.cumsum(n, 0)
    left = n[:, None] - (W - 1) + torch.arange(W - 1, device="cuda")
    last = torch.where(left >= 0, (end - n)[:, None] + left, M + torch.arange(B, device="cuda")[:, None] * (W - 1) + (W - 1) + left)
    return s["out"], table[last]


def _scan(s, Q=64):
    """In chunks of Q rows: inside a chunk every earlier row's product, weighted by the decay between the two; across chunks the
    states at the chunk's ends, weighted by the decay of the chunks between."""
    case, x = s["case"], s["x"]
    S, H, P, G, N = case["B"], case["H"], case["P"], case["G"], case["N"]
    M = x.shape[0] * x.shape[1]
    rows, seq, place = _positions(s, S, case["L"], M)
    longest = max(_lengths(case)) if case["packed"] else case["L"]
    nc = -(-longest // Q)
    to = seq * (nc * Q) + place

    def spread(t, *tail):
        """(S, nc, Q, ...) in 32 bits, zero where a sequence has no row."""
        wide = torch.zeros(S * nc * Q, *tail, device="cuda")
        wide[to] = t.reshape(M, *tail)[rows].float()
        return wide.view(S, nc, Q, *tail)

    dt = torch.zeros(S * nc * Q, H, device="cuda")
    dt[to] = F.softplus(s["dt"].reshape(M, H)[rows].float() + s["dt_bias"])
    dt = dt.view(S, nc, Q, H)
    X, Bm, Cm = spread(x, H, P).transpose(2, 3), spread(s["B"], G, N).transpose(2, 3), spread(s["C"], G, N).transpose(2, 3)
    heads = torch.arange(H, device="cuda") // (H // G)
    cum = (dt.double() * s["A"].double()).cumsum(2).transpose(2, 3)  # (S, nc, H, Q)
    total = cum[..., -1]
    dt = dt.transpose(2, 3)
    earlier = torch.ones(Q, Q, dtype=torch.bool, device="cuda").tril()
    decay = (cum[..., :, None] - cum[..., None, :]).masked_fill(~earlier, -math.inf).exp().float()
    y = ((Cm @ Bm.transpose(-1, -2))[:, :, heads] * decay * dt[..., None, :]) @ X
    # the chunks' own states (S, nc, H, P, N), then every chunk's state on entry
    w = (total[..., None] - cum).exp().float() * dt
    ends = (X * w[..., None]).transpose(-1, -2) @ Bm[:, :, heads]
    upto = total.cumsum(1)  # (S, nc, H)
    since = torch.cat([torch.zeros_like(upto[:, :1]), upto], 1)  # decay before chunk c
    between = since.transpose(1, 2)[..., :, None] - upto.transpose(1, 2)[..., None, :]  # entry of chunk c from the end of chunk e
    between = between.masked_fill(~torch.ones(nc + 1, nc, dtype=torch.bool, device="cuda").tril(-1), -math.inf).exp().float()
    entry = (between @ ends.permute(0, 2, 1, 3, 4).reshape(S, H, nc, P * N)).view(S, H, nc + 1, P, N)
    if s["h0"] is not None:
        entry = entry + since.transpose(1, 2).exp().float()[..., None, None] * s["h0"][:, :, None]
    y = y + (Cm[:, :, heads] * cum.exp().float()[..., None]) @ entry[:, :, :nc].permute(0, 2, 1, 4, 3)
    y = y.transpose(2, 3).reshape(-1, H, P)[to] + s["D"][:, None] * x.reshape(M, H, P)[rows].float()
    if s["z"] is not None:
        y = y * F.silu(s["z"].reshape(M, H, P)[rows].float())
    s["out"].view(M, H, P)[:rows.numel()] = y.to(x.dtype)
    return s["out"], entry[:, :, nc].contiguous()


def _step(s):
    case = s["case"]
    B, H, P, G, N = (case[k] for k in ("B", "H", "P", "G", "N"))
    window = torch.cat([s["conv_state"], s["row"][:, None]], 1)
    row = F.silu((window.float() * s["weight"].float().t()).sum(1) + s["bias"].float())
    x, b, c = row.split([H * P, G * N, G * N], dim=-1)
    x = x.view(B, H, P)
    b, c = (t.view(B, G, N).repeat_interleave(H // G, 1) for t in (b, c))
    dt = F.softplus(s["dt"].float() + s["dt_bias"])
    s["h"].copy_((dt * s["A"]).exp()[..., None, None] * s["h"] + (dt[..., None] * x)[..., None] * b[:, :, None])
    y = (s["h"] @ c[..., None])[..., 0] + s["D"][:, None] * x
    return (y * F.silu(s["z"].float())).to(s["row"].dtype), s["h"], window[:, 1:].contiguous()


def _candidates(s):
    """(B, K * V) in 64 bits: what a token's choice is worth.  A finished beam has one candidate, padding at its own score."""
    logits, scores = s["logits"].double(), s["scores"].double()[..., None]
    worth = scores + (logits - torch.logsumexp(logits, -1, keepdim=True))
    worth = torch.where(worth.isnan(), -math.inf, worth)
    if s["finished"] is not None:
        pad = torch.arange(logits.shape[-1], device="cuda") == 0
        worth = torch.where(s["finished"][..., None], torch.where(pad, scores, -math.inf), worth)
    return worth.flatten(1)


def _select(s):
    n, V = s["case"]["n"], s["case"]["V"]
    worth = _candidates(s)
    low = worth.topk(n, -1).values[:, -1:]
    place = torch.arange(worth.shape[1], device="cuda")
    # those above the lowest chosen value, and of those equal to it the first: ties go to the lower index
    above = torch.where(worth > low, place, worth.shape[1]).topk(n, -1, largest=False, sorted=True).values
    equal = torch.where(worth == low, place, worth.shape[1]).topk(n, -1, largest=False, sorted=True).values
    both = torch.cat([above, equal], -1)
    value = torch.where(both < worth.shape[1], worth.gather(1, both.clamp(max=worth.shape[1] - 1)), -math.inf)
    # real ones before places left open, then by value; the sort is stable
    order = torch.argsort(both >= worth.shape[1], dim=-1, stable=True)
    both, value = both.gather(1, order), value.gather(1, order)
    order = torch.argsort(value, dim=-1, descending=True, stable=True)[:, :n]
    both, value = both.gather(1, order), value.gather(1, order)
    return value.float(), both // V, both % V


def _reorder(s):
    B, K = s["parents"].shape
    rows = (s["parents"] + K * torch.arange(B, device="cuda")[:, None]).flatten()
    for t in s["all"]:
        t.copy_(t[:, rows])
    return s["all"]


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "reorder":
        rows = case["layers"] * case["B"] * case["K"]
        if case["kind"] == "ring":
            each = 8 * case["D"] + 4 * case["W"] * (case["R"] + case["D"])
        else:
            each = 4 * case["H"] * case["P"] * case["N"] + 2 * (case["W"] - 1) * case["C"]
        return {"bytes": 2 * rows * each, "flops": 0}
    size = 2 if case["dtype"] == "bf16" else 4
    if op == "select":
        count = case["B"] * case["K"] * case["V"]
        return {"bytes": size * count + 20 * case["B"] * case["n"], "flops": 4 * count}
    if op == "step":
        B, H, P, G, N, W = (case[k] for k in ("B", "H", "P", "G", "N", "W"))
        C = H * P + 2 * G * N
        return {"bytes": 8 * B * H * P * N + size * (2 * B * (W - 1) * C + C * (W + 1) + B * (C + 2 * H * P + H)),
                "flops": 5 * B * H * P * N + 2 * B * C * W}
    M = sum(_lengths(case)) if case["packed"] else case["B"] * case["L"]
    if op == "conv":
        return {"bytes": size * case["C"] * (2 * M + case["W"] + 1 + case["B"] * (case["W"] - 1) * (1 + case["init"])),
                "flops": M * case["C"] * (2 * case["W"] + 4)}
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    return {"bytes": size * M * (H * P * (2 + case["gate"]) + 2 * G * N + H) + 4 * case["B"] * H * P * N * (1 + case["init"]),
            "flops": 5 * M * H * P * N}


# ------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, row by row
# ------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "reorder":
        K, parents = case["K"], s["parents"].tolist()
        rows = [b * K + p for b in range(case["B"]) for p in parents[b]]
        return [torch.stack([t[:, r] for r in rows], 1) for t in s["all"]]
    if op == "select":
        logits, scores = s["logits"].double(), s["scores"].double()
        top = logits.amax(-1, keepdim=True)
        prob = (logits - top).exp()
        worth = scores[..., None] + (logits - top) - prob.sum(-1, keepdim=True).log()
        worth[worth.isnan()] = -math.inf
        if s["finished"] is not None:
            worth[s["finished"]] = -math.inf
            worth[..., 0] = torch.where(s["finished"], scores, worth[..., 0])
        return worth.flatten(1).sort(-1, descending=True).values[:, :case["n"]], None, None
    if op == "step":
        H, P, G, N, W = (case[k] for k in ("H", "P", "G", "N", "W"))
        acc = s["bias"].double() + s["row"].double() * s["weight"][:, W - 1].double()
        for j in range(W - 1):
            acc = acc + s["conv_state"][:, j].double() * s["weight"][:, j].double()
        row = acc / (1 + (-acc).exp())
        x, b, c = row[:, :H * P].unflatten(1, (H, P)), row[:, H * P:H * P + G * N].unflatten(1, (G, N)), row[:, H * P + G * N:].unflatten(1, (G, N))
        y, h = _exact_row(s, s["h"].double(), x, s["dt"].double(), b, c, s["z"].double())
        return y, h, torch.stack([*(s["conv_state"][:, j].double() for j in range(1, W - 1)), s["row"].double()], 1)
    packed = case["packed"]
    at = _starts(case) if packed else [i * case["L"] for i in range(case["B"] + 1)]
    flat = {k: s[k].flatten(0, 1).double() for k in (("x",) if op == "conv" else ("x", "dt", "B", "C", "z")) if s[k] is not None}
    out = s["out"].flatten(0, 1).double()
    first = torch.tensor(at[:-1], device="cuda")
    longest = max(b - a for a, b in zip(at, at[1:]))
    # sequences in falling length, so that those that still run are the first ones
    order = sorted(range(case["B"]), key=lambda i: at[i] - at[i + 1])
    first = first[torch.tensor(order, device="cuda")]
    running = [sum(at[i + 1] - at[i] > t for i in order) for t in range(longest)]
    if op == "conv":
        C, W = case["C"], case["W"]
        hist = (s["state"].double() if s["state"] is not None else torch.zeros(case["B"], W - 1, C, dtype=torch.float64, device="cuda"))
        final = []
        for i in range(case["B"]):
            rows = torch.cat([hist[i], flat["x"][at[i]:at[i + 1]]])
            acc = s["bias"].double().expand(at[i + 1] - at[i], C)
            for j in range(W):
                acc = acc + rows[j:j + at[i + 1] - at[i]] * s["weight"][:, j].double()
            out[at[i]:at[i + 1]] = acc / (1 + (-acc).exp())
            final.append(rows[rows.shape[0] - (W - 1):])
        return out.view(s["out"].shape), torch.stack(final)
    h = torch.zeros(case["B"], case["H"], case["P"], case["N"], dtype=torch.float64, device="cuda")
    if s["h0"] is not None:
        h = s["h0"].double()[torch.tensor(order, device="cuda")]
    for t, k in enumerate(running):
        at_t = first[:k] + t
        y, h[:k] = _exact_row(s, h[:k], flat["x"][at_t], flat["dt"][at_t], flat["B"][at_t], flat["C"][at_t],
                              flat["z"][at_t] if "z" in flat else None)
        out[at_t] = y
    back = torch.empty_like(h)
    back[torch.tensor(order, device="cuda")] = h
    return out.view(s["out"].shape), back


def _exact_row(s, h, x, dt, b, c, z):
    each = s["A"].numel() // b.shape[1]
    raw = dt + s["dt_bias"].double()
    size = torch.where(raw > 0, raw, 0) + torch.log1p((-raw.abs()).exp())
    h = h * (size * s["A"].double()).exp()[..., None, None] + ((size[..., None] * x)[..., None]
                                                               * b.repeat_interleave(each, 1)[:, :, None])
    y = (h * c.repeat_interleave(each, 1)[:, :, None]).sum(-1) + s["D"].double()[:, None] * x
    return (y if z is None else y * z / (1 + (-z).exp())), h
