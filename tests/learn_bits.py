"""How many bits the values between an operator's steps have to hold (test infrastructure): bounds for results that are rounded to
their type once, at the end, with everything in front of that held in 16 bits or more."""
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
