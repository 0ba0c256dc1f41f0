"""The operators that learn in 64 bits on the CPU, with the error each value may have (test infrastructure).

A rounding to a type is off by at most half a step, HALF[type] of the value; U is float32's.  Errors are bounds carried
through the same formulas on absolute values, so that no tolerance is picked by hand.
"""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
TINY = 1e-36  # (results below float32's normal numbers may come out as 0)


def sigmoid(x):
    return torch.sigmoid(x)


def within(got, want, tol, what):
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
    bad = ~(((got - want).abs() <= tol + TINY) | (got.isnan() & want.isnan()))
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound; the first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()} +- {tol[bad][0].item()}")


def scan_ref(value, write, decay, bias, state, starts, grad=None, grad_state=None):
    """Row by row.  Returns a dict of (value, error bound) pairs: h, last and, with ``grad``, the gradients.

    A gate is off by at most 6 U of itself (rounded exponent up to 16: 4 U, exponential, sum, reciprocal 1 U each), u_t by 8 U
    (tanh's difference) and each step or composition of the recurrence rounds twice: 16 U of the terms' mass per row covers them.
    """
    dtype = value.dtype
    v, w, f = value.double(), write.double(), decay.double()
    if bias is not None:
        f = f + bias.double()
    B, L, C = v.shape
    seqs = [(b, 0, L, b) for b in range(B)] if starts is None else [(0, starts[i], starts[i + 1], i) for i in range(len(starts) - 1)]
    a, q, sw, tv = sigmoid(f), sigmoid(-f), sigmoid(w), torch.tanh(v)
    u = sw * tv
    h, eh = torch.zeros_like(v), torch.zeros_like(v)
    before, eb, mass_b = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(v)
    last, el = torch.zeros(len(seqs), C, dtype=torch.float64), torch.zeros(len(seqs), C, dtype=torch.float64)
    for b, lo, hi, s in seqs:
        x = state[s].double() if state is not None else torch.zeros(C, dtype=torch.float64)
        m, e = x.abs(), torch.zeros_like(x)
        for t in range(lo, hi):
            before[b, t], eb[b, t], mass_b[b, t] = x, e, m
            m = a[b, t] * m + u[b, t].abs()
            x = a[b, t] * x + u[b, t]
            e = a[b, t] * e + 16 * U * (m + sw[b, t])
            h[b, t], eh[b, t] = x, e
        last[s], el[s] = x, e
    out = dict(h=(h, eh + HALF[dtype] * h.abs()), last=(last, el + U * last.abs()))
    if grad is None:
        return out
    d = grad.double()
    g, eg, mg = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(v)
    dh0, e0 = torch.zeros_like(last), torch.zeros_like(last)
    for b, lo, hi, s in seqs:
        c = grad_state[s].double() if grad_state is not None else torch.zeros(C, dtype=torch.float64)
        m, e = c.abs(), torch.zeros_like(c)
        for t in range(hi - 1, lo - 1, -1):
            c, m = c + d[b, t], m + d[b, t].abs()
            e = e + 4 * U * m
            g[b, t], eg[b, t], mg[b, t] = c, e, m
            c, m, e = a[b, t] * c, a[b, t] * m, a[b, t] * e + 16 * U * a[b, t] * m
        dh0[s], e0[s] = c, e + U * c.abs()
    sech = 1 / torch.cosh(v) ** 2

    def product(factor, more=0.0):
        val = g * factor
        return val, eg * factor.abs() + 24 * U * mg * factor.abs() + more

    dv, ev = product(sw * sech)
    dw, ew = product(u * sigmoid(-w), 8 * U * mg * sw * sigmoid(-w))
    df, ef = product(before * a * q, mg * (eb + 24 * U * mass_b) * a * q)
    out.update(dv=(dv, ev + HALF[dtype] * dv.abs()), dw=(dw, ew + HALF[dtype] * dw.abs()), dd=(df, ef + HALF[dtype] * df.abs()),
               db=(df.sum((0, 1)), ef.sum((0, 1)) + (64 + B * L / 128) * U * df.abs().sum((0, 1))), ds=(dh0, e0))
    return out


def act_ref(z, act):
    """The activation, its derivative, and bounds on both derivatives' size (the second's: 0.5 and 0.8)."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "silu":
        p = sigmoid(z)
        return z * p, p + z * p * sigmoid(-z)
    p = 0.5 * torch.erfc(-z / math.sqrt(2))
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def product_ref(x, w, K):
    """x w^T and the bound of its float32 sum: K additions, and for float32 operands the parts left out."""
    return x @ w.t(), (K + 16) * U * (x.abs() @ w.abs().t())


def dense_ref(x, w, up, bias, residual, act, grad=None):
    """(value, bound) pairs: y and, with ``grad``, dx, dw, du, db.  Slopes of the activations are at most 1.13, their second
    derivatives at most 0.8; an activation is off by 24 U of its argument besides."""
    dtype = x.dtype
    half = HALF[dtype]
    xd, wd = x.double(), w.double()
    M, K = xd.shape
    N = wd.shape[0]
    z, ez = product_ref(xd, wd, K)
    if bias is not None:
        z = z + bias.double()
        ez = ez + U * z.abs()
    val, slope = act_ref(z, act)
    ea = 1.13 * ez + (24 * U * z.abs() if act else 0)
    if up is not None:
        p, ep = product_ref(xd, up.double(), K)
        y = val * p
        ey = ea * p.abs() + (val.abs() + ea) * ep + 2 * U * y.abs()
    else:
        y, ey = val, ea
        if residual is not None:
            y = y + residual.double()
            ey = ey + 2 * U * (val.abs() + residual.double().abs())
    out = dict(y=(y, ey + half * y.abs()))
    if grad is None:
        return out
    d = grad.double()
    # kept products are rounded, to the type or, a pair's, to 16 bits behind the point; and so is the gradient in front of the products
    # (float32: 2^-24, three parts)
    keep = 2.0 ** -16 if up is not None and dtype == torch.bfloat16 else half
    kz = ez + keep * z.abs() if act else torch.zeros_like(z)
    eslope = 0.8 * kz + (24 * U * (1 + z.abs()) if act else 0)
    if up is not None:
        kp = ep + keep * p.abs()
        dz = d * p * slope
        edz = d.abs() * ((p.abs() + kp) * eslope + kp * slope.abs()) + (half + 4 * U) * dz.abs()
        dp = d * val
        edp = d.abs() * (1.13 * kz + 24 * U * z.abs()) + (half + 4 * U) * dp.abs()
    else:
        dz = d * slope
        edz = d.abs() * eslope + ((half + 4 * U) * dz.abs() if act else 0)

    def back(g, eg, m):
        val, e = g @ m, eg @ m.abs() + (g.shape[1] + 32) * U * ((g.abs() + eg) @ m.abs())
        return val, e

    dx, ex = back(dz, edz, wd)
    dw, ew = back(dz.t(), edz.t(), xd)
    if up is not None:
        more, em = back(dp, edp, up.double())
        dx, ex = dx + more, ex + em + 2 * U * (dx.abs() + more.abs())
        du, eu = back(dp.t(), edp.t(), xd)
        out["du"] = (du, eu + half * du.abs())
    if bias is not None:
        db = dz.sum(0)
        out["db"] = (db, (d.abs() * eslope).sum(0) + (M + 16) * U * dz.abs().sum(0) + half * db.abs())
    out["dx"] = (dx, ex + half * dx.abs())
    out["dw"] = (dw, ew + half * dw.abs())
    return out


def logp_ref(logits, targets, top, ignore=-100, grad=None, grad_entropy=None):
    """(value, bound) pairs logp, entropy, top and, with gradients, dx; top_tokens as they have to be.

    A sum is made by 64 lanes of one to four waves, so a lane adds at most V / 64 terms, each off by 4 U; the sum's relative error is
    the error of its logarithm.  p is off by that and by 8 U (1 + |x - lse|).
    """
    x = logits.double()
    V = x.shape[-1]
    es = (V / 64 + 64) * U
    far = x - x.amax(-1, keepdim=True)  # (a row of the type's lowest values would swallow its sum's logarithm)
    lp = far - far.exp().sum(-1, keepdim=True).log()
    lse = torch.zeros_like(lp[..., :1])
    p = lp.exp()
    safe = torch.where(p > 0, lp, 0.0)
    entropy = -(p * safe).sum(-1)
    spread = (p * safe.abs()).sum(-1)
    known = targets != ignore
    at = torch.where(known, targets, 0)[..., None]
    t = torch.where(known, lp.gather(-1, at)[..., 0], 0.0)
    out = dict(logp=(t, es + 2 * U * torch.where(t.isinf(), 0.0, t.abs())), entropy=(entropy, 4 * es * (1 + spread)))
    if top:
        key = torch.where(x.isnan(), -math.inf, x)
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :top]
        out["tokens"] = order
        best = lp.gather(-1, order)
        out["top"] = (best, es + 2 * U * torch.where(best.isinf(), 0.0, best.abs()))
    if grad is not None or grad_entropy is not None:
        g = torch.where(known, grad.double(), 0.0)[..., None] if grad is not None else torch.zeros_like(lse)
        e = grad_entropy.double()[..., None] if grad_entropy is not None else torch.zeros_like(lse)
        d = -p * (g + e * (safe + entropy[..., None]))
        ed = p * (g.abs() + e.abs() * (safe.abs() + spread[..., None])) * (2 * es + 16 * U * (1 + safe.abs()))
        ed = ed + 4 * es * p * e.abs() * (1 + spread[..., None])
        d.scatter_add_(-1, at, g)
        out["dx"] = (d, ed + HALF[logits.dtype] * d.abs() + U * d.abs())
    return out
