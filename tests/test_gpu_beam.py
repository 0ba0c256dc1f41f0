"""Beam selection and the reordering of states against plain torch, and a beam search over the model and over a
selective scan layer."""
import pytest
import torch

from hip_helpers import DEV, need_gpu
from tesm_amd import TESMConfig, TESMLMHeadModel, hip_ops

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()
    with torch.no_grad():
        yield


def offers(logits, scores, finished=None, pad=0):
    """(B, K * V) in 64 bits on the host."""
    logits, scores = logits.cpu().double(), scores.cpu().double()
    norm = torch.logsumexp(torch.nan_to_num(logits, nan=-INF, posinf=INF, neginf=-INF), -1, keepdim=True)
    worth = scores[..., None] + (logits - norm)  # the difference first: a score is lost next to the lowest value of a type
    worth[worth.isnan()] = -INF
    worth[~scores.isfinite()] = -INF
    if finished is not None:
        for b, k in finished.cpu().nonzero().tolist():
            worth[b, k] = -INF
            worth[b, k, pad] = scores[b, k] if scores[b, k].isfinite() else -INF
    return worth.flatten(1)


def select_ref(logits, scores, n, finished=None, pad=0, eos=None):
    V = logits.shape[-1]
    worth = offers(logits, scores, finished, pad)
    value, at = torch.sort(worth, dim=-1, descending=True, stable=True)
    value, at = value[:, :n], at[:, :n]
    done = torch.zeros_like(at, dtype=torch.bool)
    if finished is not None:
        done |= finished.cpu().bool().gather(1, at // V)
    if eos is not None:
        done |= at % V == eos
    return value, at // V, at % V, done


def check_select(logits, scores, n, finished=None, pad=0, eos=None):
    got = hip_ops.beam_select(logits.to(DEV), scores.to(DEV), n, finished=finished.to(DEV) if finished is not None else None,
                              pad_token=pad, eos_token=eos)
    want = select_ref(logits, scores, n, finished, pad, eos)
    assert torch.equal(got[1].cpu(), want[1]), "parents"
    assert torch.equal(got[2].cpu(), want[2]), "tokens"
    if finished is not None or eos is not None:
        assert torch.equal(got[3].cpu(), want[3])
    else:
        assert got[3] is None
    # a float32 rounding of the score, and the logsumexp: its sum's relative error, at most (V / 1024 + 64) 2^-24
    tol = 2.0 ** -24 * (want[0].abs() + logits.shape[-1] / 1024 + 64)
    off = (got[0].cpu().double() - want[0]).abs()
    assert bool(((off <= tol) | (got[0].cpu().double() == want[0])).all()), float(off.nan_to_num().max())
    return got


def _case(seed, B, K, V, dtype, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(B, K, V, generator=g)).to(dtype), -4 * torch.rand(B, K, generator=g) - 1, g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 4, 50, 4), (3, 5, 1000, 10), (2, 8, 4097, 8), (1, 4, 151936, 4),
                                     (2, 16, 20011, 32), (1, 64, 300, 64), (1, 2, 32, 64), (9, 3, 8192, 3), (40, 8, 2049, 8)])
def test_select(dtype, B, K, V, n):
    logits, scores, _ = _case(B + K + V + n, B, K, V, dtype)
    check_select(logits, scores, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", ["equal", "rising", "falling", "two values", "steps"])
@pytest.mark.parametrize("V", [64, 5000, 40000])
def test_select_ties_and_sorted_rows(dtype, order, V):
    """Equal logits are taken from the lowest beam and index on; rows in order are the worst ones for a running list."""
    K, n = 3, 8
    v = torch.arange(V, dtype=torch.float32)
    row = {"equal": torch.zeros(V), "rising": v * (100 / V), "falling": -v * (100 / V), "two values": (v % 97 == 5).float(),
           "steps": torch.floor(v / 1000)}[order]
    logits = row.expand(2, K, V).contiguous().to(dtype)
    scores = torch.tensor([[0.0, 0.0, 0.0], [-1.0, -0.5, -1.0]])
    check_select(logits, scores, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_infinities_and_nans(dtype):
    logits, scores, g = _case(3, 8, 4, 3000, dtype)
    logits[0].masked_fill_(torch.rand(3000, generator=g) < 0.9, -INF)
    logits[1, 2] = -INF                          # a beam without any token
    logits[2] = -INF                             # a request without any
    logits[3, 1, ::3] = float("nan")
    logits[4, 0, 17] = INF                       # that beam has no offers
    logits[5, :, 5:] = -INF                      # fewer finite offers than asked for
    logits[6] = torch.finfo(dtype).min           # the lowest value everywhere: an ordinary, even row
    scores[7, 1:] = -INF                         # the first token: one beam counts
    scores[3, 3] = float("nan")
    check_select(logits, scores, 24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [0, 5, 99])
def test_select_finished_beams(dtype, pad):
    logits, scores, g = _case(11 + pad, 6, 4, 100, dtype)
    finished = torch.rand(6, 4, generator=g) < 0.5
    finished[0], finished[1] = True, False
    scores[2, 0] = -INF
    finished[2, 0] = True
    scores[3] *= 0.01                            # finished beams that win
    check_select(logits, scores, 8, finished, pad, eos=7)
    check_select(logits, scores, 8, finished, pad)
    check_select(logits, scores, 3, None, 0, eos=int(logits[0].float().max(0).values.argmax()))
    got = hip_ops.beam_select(logits[:1].to(DEV), scores[:1].to(DEV), 6, finished=finished[:1].to(torch.uint8).to(DEV), pad_token=pad)
    assert got[2][0, :4].tolist() == [pad] * 4   # four offers above -infinity, then the lowest of the rest
    assert got[0][0, 4:].tolist() == [-INF, -INF]


def test_select_of_unaligned_row_slices():
    wide = torch.randn(2, 3, 1030, generator=torch.Generator().manual_seed(2)).bfloat16()
    scores = -torch.rand(2, 3, generator=torch.Generator().manual_seed(3))
    for lo, hi in ((0, 1030), (1, 1025), (7, 1030), (8, 1000)):
        got = hip_ops.beam_select(wide.to(DEV)[..., lo:hi], scores.to(DEV), 5)
        want = select_ref(wide[..., lo:hi], scores, 5)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])


def test_select_captured_and_replayed():
    sets = [_case(20 + i, 2, 4, 30000, torch.bfloat16)[:2] for i in range(2)]
    sets = [(a.to(DEV), b.to(DEV)) for a, b in sets]
    want = [hip_ops.beam_select(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, capture_error_mode="relaxed"):
            outs.append(hip_ops.beam_select(*s))
        graphs.append(gr)
    for _ in range(3):
        for i in (1, 0):
            for o in outs[i][:3]:
                o.zero_()
            graphs[i].replay()
            hip_ops.beam_select(*sets[1 - i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i][:3], want[i][:3]))


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------
def _tensors(g, rows):
    return [torch.randn(rows, 33, generator=g, dtype=torch.float64), torch.randn(rows, 4, 16, generator=g),
            torch.randn(rows, 5, 7, generator=g).bfloat16(), torch.randint(0, 200, (rows, 3), generator=g, dtype=torch.uint8),
            torch.randint(0, 2, (rows,), generator=g).bool(), torch.randn(rows, 3000, generator=g), torch.zeros(rows, 0),
            torch.randint(0, 9, (rows, 11), generator=g)]


@pytest.mark.parametrize("B,K", [(1, 1), (1, 2), (3, 4), (2, 5), (4, 8), (2, 16), (1, 17), (2, 32), (1, 64)])
def test_reorder(B, K):
    g = torch.Generator().manual_seed(B * 100 + K)
    host = _tensors(g, B * K)
    wide = torch.randn(B * K, 50, generator=g)
    for kind in ("random", "same", "identity", "reverse", "first"):
        parents = {"random": torch.randint(0, K, (B, K), generator=g), "same": torch.full((B, K), K - 1),
                   "identity": torch.arange(K).expand(B, K), "reverse": torch.arange(K - 1, -1, -1).expand(B, K),
                   "first": torch.zeros(B, K, dtype=torch.int64)}[kind].contiguous()
        rows = (parents + K * torch.arange(B)[:, None]).flatten()
        dev = [t.to(DEV) for t in host]
        part = wide.to(DEV)
        hip_ops.reorder_rows(dev + [part[:, 3:40]], parents.to(DEV))
        for t, d in zip(host, dev):
            assert torch.equal(d.cpu(), t[rows]), (kind, t.dtype, t.shape)
        want = wide.clone()
        want[:, 3:40] = wide[rows, 3:40]
        assert torch.equal(part.cpu(), want)


def test_reorder_of_many_tensors_and_none():
    g = torch.Generator().manual_seed(4)
    host = [torch.randn(6, 8 + i, generator=g) for i in range(200)]
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]])
    dev = [t.to(DEV) for t in host]
    hip_ops.reorder_rows(dev, parents.to(DEV))
    rows = torch.tensor([2, 0, 0, 4, 4, 5])
    assert all(torch.equal(d.cpu(), t[rows]) for d, t in zip(dev, host))
    hip_ops.reorder_rows([], parents.to(DEV))
    hip_ops.reorder_rows([torch.zeros(0, 4, device=DEV)], torch.zeros(0, 3, dtype=torch.int64, device=DEV))


def test_reorder_reports_bad_parents():
    """A parent outside the beams leaves its row as it is; the status word says so."""
    hip_ops.device_status()
    t = torch.arange(24, dtype=torch.float32, device=DEV).view(8, 3)
    hip_ops.reorder_rows([t], torch.tensor([[0, 4, 1, -1], [3, 3, 1 << 40, 0]], device=DEV))
    assert t[:, 0].div(3).tolist() == [0, 1, 1, 3, 7, 7, 6, 4]
    assert hip_ops.device_status() == 2
    assert hip_ops.device_status() == 0
    hip_ops.reorder_rows([t], torch.tensor([[0]] * 7 + [[1]], device=DEV))
    assert t[:, 0].div(3).tolist() == [0, 1, 1, 3, 7, 7, 6, 4] and hip_ops.device_status() == 2


def test_reorder_captured_and_replayed_on_another_stream():
    """Parents are read when the graph runs; an eager call on another stream moves other tensors at the same time."""
    g = torch.Generator().manual_seed(11)
    host = _tensors(g, 12)
    first, dev, other = [t.to(DEV) for t in host], [t.to(DEV) for t in host], [t.to(DEV) for t in host]
    parents = torch.zeros(3, 4, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, capture_error_mode="relaxed"):
        hip_ops.reorder_rows(dev, parents)
    for step in range(3):
        p = torch.randint(0, 4, (3, 4), generator=g)
        rows = (p + 4 * torch.arange(3)[:, None]).flatten()
        for d, f in zip(dev, first):
            d.copy_(f)
        parents.copy_(p)
        side.wait_stream(torch.cuda.current_stream())
        gr.replay()
        with torch.cuda.stream(side):
            hip_ops.reorder_rows(other, parents)
        torch.cuda.synchronize()
        assert all(torch.equal(d.cpu(), t[rows]) for d, t in zip(dev, host)), step
        host2 = [t[rows] for t in host] if step == 0 else [t[rows] for t in host2]
        assert all(torch.equal(d.cpu(), t) for d, t in zip(other, host2)), step


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def _model(dtype, **kw):
    cfg = TESMConfig(**dict(dict(d_model=64, n_layer=2, d_intermediate=128, vocab_size=300, max_seq_len=48, d_state=32,
                                 ent_rank=8, entanglement_window=8, entanglement_threshold=0.05, decay_init_bias=1.0,
                                 initializer_range=0.2), **kw))
    torch.manual_seed(5)
    return TESMLMHeadModel(cfg).to(DEV).to(dtype).eval()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, dict(use_mimo=True, n_heads=2), dict(entanglement_window=0)])
def test_model_beam_search(dtype, kw):
    """The method against the same decode steps with plain torch selection and index_select'ed caches."""
    m = _model(dtype, **kw)
    B, K, T, eos = 2, 3, 10, 17
    ids = torch.randint(0, 300, (B, 9), generator=torch.Generator().manual_seed(1)).to(DEV)
    tokens, scores = m.beam_search(ids, K, T, eos_token=eos, pad_token=2)
    caches = m.allocate_inference_cache(B, 32)
    logits = m(ids, inference_params={"state_cache": caches}, logits_to_keep=1)[0].logits
    s, _, tok, done = (t.to(DEV) for t in select_ref(logits, torch.zeros(B, 1), K, None, 2, eos))
    for c in caches.values():
        for k in ("state", "ent_k_cache", "ent_v_cache"):
            c[k] = c[k].repeat_interleave(K, 0)
    hist = tok[..., None]
    while hist.shape[-1] < T and not bool(done.all()):
        logits = m(tok.view(-1, 1), inference_params={"state_cache": caches})[0].logits.view(B, K, -1)
        s, par, tok, done = (t.to(DEV) for t in select_ref(logits, s.float(), K, done, 2, eos))
        rows = (par + K * torch.arange(B, device=DEV)[:, None]).flatten()
        for c in caches.values():
            for k in ("state", "ent_k_cache", "ent_v_cache"):
                c[k] = c[k].index_select(0, rows)
        hist = torch.cat([hist.gather(1, par[..., None].expand_as(hist)), tok[..., None]], -1)
    assert torch.equal(tokens, hist)
    # every step's score is rounded to float32 and carries its logsumexp's error (300 tokens)
    assert float((scores.double() - s.double()).abs().max()) <= T * 2.0 ** -24 * (float(s.abs().max()) + 65)


def test_model_beam_search_ends_when_all_beams_do():
    m = _model(torch.float32)
    ids = torch.randint(0, 300, (1, 5), generator=torch.Generator().manual_seed(1)).to(DEV)
    first = m.beam_search(ids, 1, 1)[0]
    tokens, scores = m.beam_search(ids, 1, 20, eos_token=int(first[0, 0, 0]))
    assert tokens.shape == (1, 1, 1) and bool(scores.isfinite().all())
    tokens, _ = m.beam_search(ids, 2, 44)  # 5 + 44 - 1 = 48 positions
    assert tokens.shape == (1, 2, 44)
    with pytest.raises(ValueError, match="max_seq_len"):
        m.beam_search(ids, 2, 45)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_layer_beam_search(dtype):
    """Prompt convolution and scan, then tokens through the step, the choice and the reordered states, against the same
    search with plain torch states in 64 bits; the choices must agree wherever no two offers are near."""
    g = torch.Generator().manual_seed(8)
    B, L, H, P, G, N, W, K, V, T = 2, 40, 4, 32, 2, 32, 4, 4, 200, 6
    width = H * P + 2 * G * N
    embed = (torch.randn(V, width, generator=g) * 1.0).to(dtype).to(DEV)
    head = torch.randn(H * P, V, generator=g).to(DEV) / 4
    dtw = torch.randn(V, H, generator=g).to(dtype).to(DEV)
    w, wb = (torch.randn(width, W, generator=g) / 2).to(dtype).to(DEV), torch.zeros(width, dtype=dtype, device=DEV)
    A, D = -(0.3 + torch.rand(H, generator=g)).to(DEV), torch.ones(H, device=DEV)
    ids = torch.randint(0, V, (B, L), generator=g).to(DEV)

    row, cs = hip_ops.causal_conv(embed[ids], w, wb)
    x, b, c = row.split([H * P, G * N, G * N], -1)
    y, h = hip_ops.selective_scan(x.unflatten(-1, (H, P)), dtw[ids], A, b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N)), D=D)
    # the reference starts from the same states: the prompt has its own tests
    h64, c64 = h.double().repeat_interleave(K, 0), cs.double().repeat_interleave(K, 0)
    scores, _, tok, _ = hip_ops.beam_select((y[:, -1].flatten(1).float() @ head)[:, None], torch.zeros(B, 1, device=DEV), K)
    h, cs, s64, tok64 = h.repeat_interleave(K, 0), cs.repeat_interleave(K, 0), scores.double(), tok
    for _ in range(T):
        y, cs = hip_ops.selective_scan_step(embed[tok.view(-1)], dtw[tok.view(-1)], A, h, w, wb, cs, n_groups=G, D=D,
                                            out=torch.empty(B * K, H, P, dtype=dtype, device=DEV))
        logits = (y.flatten(1).float() @ head).view(B, K, V)
        scores, par, tok, _ = hip_ops.beam_select(logits, scores)
        hip_ops.reorder_rows([h, cs], par)
        # 64 bits, the chosen parents and tokens taken over so that the two stay together
        win = torch.cat([c64, embed[tok64.view(-1)].double()[:, None]], 1)
        v = _silu64((win * w.double().t()).sum(1))
        x6, b6, c6 = v.split([H * P, G * N, G * N], 1)
        x6 = x6.view(B * K, H, P)
        b6, c6 = (t.reshape(B * K, G, N).repeat_interleave(H // G, 1) for t in (b6, c6))
        d = torch.nn.functional.softplus(dtw[tok64.view(-1)].double())
        h64 = (d * A.double()).exp()[..., None, None] * h64 + (d[..., None] * x6)[..., None] * b6[:, :, None]
        y6 = (h64 * c6[:, :, None]).sum(-1) + x6
        # y's rounding to the layer type reaches a logit through the head: half a step of each term, float32 sums beside it
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        near = float((y6.flatten(1).abs() @ head.double().abs()).max()) * (half + 2.0 ** -24 * (H * P + N + 64))
        worth = offers((y6.flatten(1) @ head.double()).view(B, K, V), s64)
        chosen = (par * V + tok).cpu()
        best = worth.sort(-1, descending=True).values[:, :K]
        assert float((worth.gather(1, chosen) - best).abs().max()) <= 4 * near
        s64, tok64 = scores.double(), tok
        rows = (par + K * torch.arange(B, device=DEV)[:, None]).flatten()
        h64, c64 = h64[rows], win[:, 1:][rows]
        assert torch.equal(cs.double(), c64)
        assert float((h.double() - h64).abs().max()) <= 2.0 ** -24 * 4096 * float(h64.abs().max())


def _silu64(v):
    return v / (1 + torch.exp(-v))
