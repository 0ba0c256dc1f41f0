"""Every kernel that calls of the operators that learn choose by their sizes, against the 64-bit forms; each test asserts, through the
launch log, that the instantiations it is about ran."""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from learn_bits import dense_bounds, f32_bound, off_in_norm
from learn_refs import logp_ref, scan_ref, within
from tesm_amd import hip_ops
from test_gpu_learn import BOTH, _dev, dense_case, logp_case

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


# ---------------------------------------------------------------------------
# products: kind (0 pair, 1 projection, 2 gradient, 3 gradient's split runs), type, parts, operands that lie down, waves, tiles per wave,
# values of k per tile, stages
# ---------------------------------------------------------------------------
TILES = {
    (BF, True): dict(large="4,2,2,2,64,2", mid="2,2,2,1,64,2", small="2,2,2,1,64,4", tiny="2,2,1,1,64,3"),
    (BF, False): dict(large="2,4,4,2,64,2", mid="2,2,2,2,64,2", small="2,2,2,2,64,4", tiny="2,2,1,1,64,4"),
    (F32, True): dict(large="4,2,1,2,32,2", mid="2,2,2,1,32,3", small="2,2,1,1,32,4", tiny="2,2,1,1,32,2"),
    (F32, False): dict(large="4,2,2,2,32,2", mid="2,4,2,1,32,3", small="2,2,1,1,32,6", tiny="2,2,1,1,32,3"),
}


def product_name(dtype, what, pair, tiles):
    split = tiles.endswith(" split")
    kind = (0 if pair else 1) if what == "y" else 3 if split else 2
    shape = TILES[dtype, pair and what == "y"][tiles.split()[0]]
    result = 0 if dtype == F32 or split else 1
    lie = {"y": "false,false", "dx": "false,true", "dw": "true,true"}[what]
    return f"product_kernel<{kind},{result},{3 if dtype == F32 else 1},{lie},{shape}>"


@pytest.mark.parametrize("dtype,pair,M,K,N,y,dx,dw", [
    (BF, False, 200, 200, 200, "tiny", "tiny", "tiny"),
    (BF, False, 200, 200, 8200, "small", "tiny split", "small"),
    (BF, False, 1300, 200, 3000, "mid", "tiny split", "tiny"),
    (BF, False, 1300, 200, 6200, "large", "small split", "tiny"),
    (BF, False, 1300, 3000, 200, "tiny", "mid", "tiny"),
    (BF, False, 1300, 6200, 200, "tiny", "large", "tiny"),
    (BF, True, 65, 200, 520, "tiny", "tiny split", "tiny"),
    (BF, True, 130, 8200, 3000, "tiny", "large split", "mid"),
    (BF, True, 200, 1300, 3000, "tiny", "small split", "large"),
    (BF, True, 200, 8200, 200, "tiny", "small", "mid"),
    (BF, True, 2000, 200, 2100, "large", "small split", "small split"),
    (BF, True, 2000, 200, 8200, "mid", "small split", "large split"),
    (BF, True, 2100, 200, 1040, "mid", "small split", "small split"),
    (BF, True, 6200, 130, 3000, "large", "mid split", "mid split"),
    (BF, True, 8200, 200, 65, "small", "small", "tiny split"),
    (F32, False, 200, 200, 200, "small", "small", "small"),
    (F32, False, 260, 333, 4100, "tiny", "tiny split", "tiny"),
    (F32, False, 2000, 200, 2100, "large", "tiny split", "mid split"),
    (F32, False, 8200, 520, 200, "mid", "large", "tiny split"),
    (F32, True, 200, 8200, 200, "small", "mid", "large"),
    (F32, True, 260, 200, 6200, "tiny", "small split", "mid"),
    (F32, True, 777, 200, 333, "small", "small split", "small split"),
    (F32, True, 2100, 200, 1040, "large", "mid split", "mid split"),
    (F32, True, 4100, 65, 4100, "large", "large split", "large split"),
    (F32, True, 4100, 200, 200, "mid", "tiny", "tiny split"),
])
def test_products_of_every_tile(dtype, pair, M, K, N, y, dx, dw):
    """All 48 of them, 16 for bfloat16 and 16 for float32 results and 16 for split runs, over several tiles of the contraction and a rest."""
    c = {k: _dev(v) for k, v in dense_case(M + K + N, M, K, N, dtype, pair=pair, bias=not pair).items()}
    act = "silu" if pair else "gelu"
    with hip_ops.launch_log() as log:
        if pair:
            got, kept = hip_ops.gated_linear(c["x"], c["w"], c["up"], act=act, keep=True)
            grads = hip_ops.gated_linear_backward(c["grad"], c["x"], c["w"], c["up"], kept=kept, act=act)
        else:
            got, kept = hip_ops.fused_linear(c["x"], c["w"], c["bias"], act=act, keep=True)
            grads = hip_ops.fused_linear_backward(c["grad"], c["x"], c["w"], c["bias"], kept=kept, act=act)
    ran = [k for k in log.kernels if k.startswith("product_kernel")]
    assert ran == [product_name(dtype, what, pair, tiles) for what, tiles in (("y", y), ("dx", dx), ("dw", dw))]
    r = dense_bounds(c, act)
    within(got, *r["y"], "y")
    for a, name in zip(grads, ("dx", "dw", "du" if pair else "db")):
        within(a, *r[name], name)


@pytest.mark.parametrize("dtype", BOTH)
def test_projection_onto_a_vocabulary(dtype):
    """The largest product of a language model's step, its result's gradient and the weight's."""
    M, K, N = 100, 72, 151936
    c = {k: _dev(v) for k, v in dense_case(3, M, K, N, dtype).items()}
    y = hip_ops.fused_linear(c["x"], c["w"])
    dx, dw, _ = hip_ops.fused_linear_backward(c["grad"], c["x"], c["w"])
    r = dense_bounds(c, None)
    for a, name in ((y, "y"), (dx, "dx"), (dw, "dw")):
        within(a, *r[name], name)
    if dtype == F32:  # (the bound of a sum of 151936 terms is a wide one)
        assert off_in_norm(dx, c["grad"].double() @ c["w"].double()) <= f32_bound(N)
    # few rows of it: a generated token
    y = hip_ops.fused_linear(c["x"][:3], c["w"])
    within(y, *(v[:3] for v in r["y"]), "y")


# ---------------------------------------------------------------------------
# recurrence: two channels per lane from 1024 tiles of 128 on, 128 rows per tile forward above 256 MiB in long sequences
# ---------------------------------------------------------------------------
def scan_on_device(seed, B, L, C, dtype, starts=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    S = B if starts is None else len(starts) - 1
    rand = lambda *s, t=dtype: torch.randn(s, generator=g, device=DEV).to(t)
    c = {k: rand(B, L, C) for k in ("value", "write", "decay", "grad")}
    c.update(bias=1 + 5 * torch.rand(C, generator=g, device=DEV), state=0.5 * rand(S, C, t=F32), grad_state=rand(S, C, t=F32), starts=starts)
    return c


def check_channels(c, channels, names):
    """Some channels of a large case (what a channel holds depends on no other); returns all results."""
    args = [c[k] for k in ("value", "write", "decay", "bias")]
    how = dict(state=c["state"], seq_starts=None if c["starts"] is None else torch.tensor(c["starts"], dtype=torch.int32, device=DEV))
    with hip_ops.launch_log() as log:
        h, last, kept = hip_ops.gated_scan(*args, keep=True, **how)
        grads = hip_ops.gated_scan_backward(c["grad"], *args, kept=kept, grad_state=c["grad_state"], **how)
    assert [k for k in log.kernels if k.startswith(("recur_fwd", "recur_bwd"))] == names
    at = torch.tensor(channels, device=DEV)
    some = {k: c[k][..., at].cpu() for k in ("value", "write", "decay", "grad", "bias", "state", "grad_state")}
    r = scan_ref(some["value"], some["write"], some["decay"], some["bias"], some["state"], c["starts"], some["grad"], some["grad_state"])
    for a, name in zip((h, last, *grads), ("h", "last", "dv", "dw", "dd", "db", "ds")):
        within(a[..., at], *r[name], name)
    return h, grads


PACKED = [5, 70, 70, 4001, 4129, 12345, 16990]  # (an empty one, one of 128 rows, starts that are no multiples of a tile's rows)


def test_scan_of_two_channels_per_lane():
    C = 1030
    check_channels(scan_on_device(1, 8, 1000, C, BF), [0, 1, 63, 64, 127, 128, 129, 766, 1023, 1024, C - 2, C - 1],
                   ["recur_fwd_kernel<1,2,8>", "recur_bwd_kernel<1,2>"])


def test_scan_of_two_channels_per_lane_packed():
    C, starts = 520, PACKED
    h, grads = check_channels(scan_on_device(2, 1, 17003, C, BF, starts), [0, 1, 127, 128, 258, 383, 512, C - 1],
                              ["recur_fwd_kernel<1,2,8>", "recur_bwd_kernel<1,2>"])
    for t in (h, *grads[:3]):
        assert not t[:, :starts[0]].any() and not t[:, starts[-1]:].any()


def test_scan_of_tall_tiles():
    C = 2048
    check_channels(scan_on_device(3, 3, 5600, C, BF), [0, 1, 127, 128, 1000, 1025, C - 2, C - 1],
                   ["recur_fwd_kernel<1,2,16>", "recur_bwd_kernel<1,2>"])


@pytest.mark.parametrize("starts", [PACKED, [0, 128, 192, 256, 16900, 17003]])
def test_scan_of_tall_tiles_packed(starts):
    """Carries that tiles of 128 rows leave are those that tiles of 64 rows read, whatever row a sequence begins on."""
    C = 2048
    h, grads = check_channels(scan_on_device(4, 1, 17003, C, BF, starts), [0, 1, 127, 128, 1000, 1025, C - 2, C - 1],
                              ["recur_fwd_kernel<1,2,16>", "recur_bwd_kernel<1,2>"])
    for t in (h, *grads[:3]):
        assert not t[:, :starts[0]].any() and not t[:, starts[-1]:].any()


def test_scan_of_large_calls_of_short_sequences():
    C = 4096
    check_channels(scan_on_device(6, 50, 192, C, BF), [0, 1, 127, 128, 2000, C - 1], ["recur_fwd_kernel<1,2,8>", "recur_bwd_kernel<1,2>"])


def test_scan_of_tall_tiles_at_any_pitch():
    C = 2046
    check_channels(scan_on_device(7, 1, 17003, C, BF), [0, 1, 127, 128, 1000, C - 1], ["recur_fwd_kernel<1,2,16>", "recur_bwd_kernel<1,2>"])


@pytest.mark.parametrize("B,L,starts", [(4, 4200, None), (1, 17003, PACKED)])
def test_scan_of_large_float32_calls(B, L, starts):
    C = 1024
    check_channels(scan_on_device(5, B, L, C, F32, starts), [0, 1, 63, 64, 500, C - 2, C - 1],
                   ["recur_fwd_kernel<0,1,8>", "recur_bwd_kernel<0,1>"])


# ---------------------------------------------------------------------------
# log probabilities of rows in more than 64 parts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,V", [(F32, 300001), (BF, 600001)])
@pytest.mark.parametrize("top", [0, 20])
def test_logp_of_rows_in_many_parts(dtype, V, top):
    """Joined 64 at a time; the row's largest logits lie in the last parts."""
    x, t, g, e = logp_case(V, 1, V, dtype)
    t[0] = V - 3
    x[0, -2000:] += 4
    r = logp_ref(x, t, top, -100, g, e)
    with hip_ops.launch_log() as log:
        logp, entropy, best, tokens, kept = hip_ops.token_log_probs(_dev(x), _dev(t), top=top, keep=True)
    code, lists = 0 if dtype == F32 else 1, "true" if top else "false"
    assert log.kernels == [f"logp_row_kernel<{code},{lists}>", f"logp_join_kernel<{code},{lists}>"]
    d = hip_ops.token_log_probs_backward(_dev(g), _dev(e), _dev(x), _dev(t), kept=kept)
    for got, name in ((logp, "logp"), (entropy, "entropy"), (d, "dx")) + (((best, "top"),) if top else ()):
        within(got, *r[name], name)
    if top:
        assert torch.equal(tokens.cpu(), r["tokens"])
