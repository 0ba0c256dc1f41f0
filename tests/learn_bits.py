"""How many bits the values between an operator's steps have to hold (test infrastructure): bounds for results that are rounded to
their type once, at the end, with everything in front of that held in 16 bits or more."""
import math

import torch

from learn_refs import HALF, dense_ref

BITS = 2.0 ** -16  # half a step of 16 bits


def dense_bounds(c, act):
    """``dense_ref`` of a case whose gradients in front of the products, and whose kept values, hold 16 bits."""
    dtype, half = c["x"].dtype, HALF[c["x"].dtype]
    HALF[dtype] = min(half, BITS)
    try:
        r = dense_ref(c["x"], c["w"], c["up"], c["bias"], c["residual"], act, c["grad"])
    finally:
        HALF[dtype] = half
    return {k: (v, e + half * v.abs()) for k, (v, e) in r.items()}


def share_beyond(got, want, tol):
    return ((got.double() - want).abs() > tol).double().mean().item()


def rounded(t, dtype=torch.bfloat16):
    return t.to(dtype).double()


def f32_bound(K):
    """How far a float32 product of K random terms per result may be off in norm, relative to its own norm.

    A sum is made of at most K / 4 additions (a matrix instruction takes at least 4 terms at once), each off by at most half a step,
    2^-24, of the sum so far.  Signs are random: the sums so far are not above the result in norm, and the roundings add up as their
    squares do, 2^-24 sqrt(K / 4).  8 half steps more are for the last rounding and for parts of operands below 2^-24 of them.
    """
    return (math.sqrt(K / 4) + 8) * 2.0 ** -24


def off_in_norm(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return ((got - want).norm() / want.norm()).item()
