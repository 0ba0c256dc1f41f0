"""The bounds of ``learn_bits`` tell a form that holds fewer bits from one that does not: 64-bit forms with a rounding planted in them."""
import math

import pytest
import torch

from learn_bits import dense_bounds, f32_bound, off_in_norm, rounded, share_beyond
from learn_refs import act_ref

BF = torch.bfloat16
SIZES = [(40, 31, 70), (70, 40, 26), (130, 72, 136)]


def dense_case(seed, M, K, N, dtype, pair=False):
    g = torch.Generator().manual_seed(seed)
    x, w, up, bias, grad = (torch.randn(s, generator=g) for s in ((M, K), (N, K), (N, K), (N,), (M, N)))
    k = math.sqrt(K)
    return dict(x=x.to(dtype), w=(w / k).to(dtype), up=(up / k).to(dtype) if pair else None, bias=None if pair else bias.to(dtype),
                residual=None, grad=grad.to(dtype))


def gradients(c, act, front=lambda t: t, kept=lambda t: t):
    """dx, dw (and du or db), with ``front`` applied to the gradients in front of the products, ``kept`` to the values kept."""
    x, w, d = (c[k].double() for k in ("x", "w", "grad"))
    if c["up"] is not None:
        up = c["up"].double()
        val, slope = act_ref(kept(x @ w.t()), act)
        dg, du = front(d * kept(x @ up.t()) * slope), front(d * val)
        out = dict(dx=dg @ w + du @ up, dw=dg.t() @ x, du=du.t() @ x)
    else:
        _, slope = act_ref(kept(x @ w.t() + c["bias"].double()), act)
        dz = d * slope
        out = dict(dx=front(dz) @ w, dw=front(dz).t() @ x, db=dz.sum(0))
    return {k: v.to(BF) for k, v in out.items()}


def worst(c, act, **kw):
    r, got = dense_bounds(c, act), gradients(c, act, **kw)
    return {k: share_beyond(v, *r[k]) for k, v in got.items()}


@pytest.mark.parametrize("pair,act", [(True, "silu"), (True, "gelu"), (False, "silu"), (False, "gelu")])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_a_gradient_rounded_in_front_of_the_products_is_seen(pair, act, M, K, N):
    c = dense_case(M + K, M, K, N, BF, pair)
    assert not any(worst(c, act).values())
    two = lambda t: rounded(t) + rounded(t - rounded(t))
    assert not any(worst(c, act, front=two).values())
    one = worst(c, act, front=rounded)
    assert one["dx"] and one["dw"]


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_a_kept_value_rounded_to_its_type_is_seen(pair, M, K, N):
    c = dense_case(M + N, M, K, N, BF, pair)
    off = worst(c, "gelu", kept=rounded)
    assert off["dx"] and off["dw"]  # (one value beyond its bound is enough)


def parts(x):
    """float32 values as three of bfloat16."""
    x0 = rounded(x)
    x1 = rounded(x - x0)
    return x0, x1, rounded(x - x0 - x1)


ORDER = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]


@pytest.mark.parametrize("M,K,N", [(70, 104, 72), (100, 70, 50), (300, 1030, 200), (64, 2100, 80)])
def test_a_part_left_out_of_a_float32_product_is_seen(M, K, N):
    """The six products of parts are within the bound, any five of them are not."""
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=g).double(), torch.randn(N, K, generator=g).double()
    xs, ws = parts(x), parts(w)
    terms = {o: xs[o[0]] @ ws[o[1]].t() for o in ORDER}
    assert off_in_norm(sum(terms.values()), x @ w.t()) < 2.0 ** -24
    for left_out in ORDER:
        assert off_in_norm(sum(v for o, v in terms.items() if o != left_out), x @ w.t()) > f32_bound(K), left_out
