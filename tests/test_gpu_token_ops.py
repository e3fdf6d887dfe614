"""Token operators (ops/token_ops.py) on the GPU against their definitions in 64 bits (token_oracle)."""
import math

import pytest
import torch

from . import token_oracle as O
from serann.ops import token_ops as TO

pytestmark = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGN = -100


def _logits(R, V, dtype, seed, spread=2.5, peak=12.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * spread
    at = torch.randint(0, V, (R, 1), generator=g)
    x.scatter_add_(1, at, torch.rand(R, 1, generator=g) * peak)
    return x.to(DTYPES[dtype]), at[:, 0], g


def _close(a, b, tol, what):
    a, b = a.detach().cpu().double(), b.double()
    assert a.shape == b.shape, (what, a.shape, b.shape)
    assert torch.equal(a.isnan(), b.isnan()), (what, "NaN")
    fin = b.isfinite()
    assert torch.equal(a[~fin & ~b.isnan()], b[~fin & ~b.isnan()]), (what, "infinite")
    assert torch.isfinite(a[fin]).all(), (what, "finite")
    tol = tol if isinstance(tol, torch.Tensor) else torch.full_like(b, tol)
    over = ((a - b).abs() - tol.expand_as(b))[fin]
    assert not len(over) or float(over.max()) <= 0, (what, float((a - b).abs()[fin].max()), float(over.max()))


def _same(a, b):
    """Bitwise equal, NaN with NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0, 1e30, -1e30), b.nan_to_num(0, 1e30, -1e30))


def _score_tols(x, ref, T):
    """Bounds of logprob and entropy.  logprob = (x_t - m) / T - ln(sum): three roundings of the first term, one logarithm (2
    ulp), the sum's relative error; for a row sure of one token ln(1 + S) is relative to S, which the first bound covers.
    Entropy = ln(sum) - ln2 W / sum: W's terms e (d) carry the errors of e and of d, so twice the sum's bound on the average
    |d| <= log2(V) + 2 bits."""
    eps = O.sum_error(x, T)
    V = x.shape[-1]
    bits = math.log2(max(V, 2)) + 2
    lp = eps + 6 * O.U * ref.get("logprob", ref["entropy"]).abs().nan_to_num(0, 0, 0)
    h = (1 + 2 * 0.7 * bits) * eps + 6 * O.U * ref["entropy"].abs().nan_to_num()
    return lp, h


def _first(t, tile):
    """The first of ``tile`` copies of the rows, after a look that all of them came out the same."""
    if t is None or tile == 1:
        return t
    t = t.reshape((tile, -1) + t.shape[1:])
    assert _same(t.float(), t[:1].float().expand_as(t))
    return t[0]


def _check_score(x, y, T, k, grad=True, seed=0, tile=1):
    """``tile``: the rows are given that many times over (launch shapes that only many rows take)."""
    R, V = x.shape[0], x.shape[-1]
    g = torch.Generator().manual_seed(seed + 99)
    gl, gh = torch.randn(R, generator=g), torch.randn(R, generator=g)
    ref = O.score(x, y, T, k, IGN, gl if grad else None, gh if grad else None)
    xd = x.repeat(tile, 1).cuda().requires_grad_(grad)
    yd = None if y is None else y.repeat(tile).cuda()
    r = full = TO.token_logprobs(xd, yd, temperature=T, top_k=k, ignore_index=IGN)
    r = TO.TokenLogprobs(*(_first(v, tile) for v in r))
    tl, th = _score_tols(x, ref, T)
    if y is not None:
        _close(r.logprob, ref["logprob"], tl, "logprob")
    _close(r.entropy, ref["entropy"], th, "entropy")
    if k:
        assert torch.equal(r.top_ids.cpu(), ref["top_ids"])
        tt = O.sum_error(x, T) + 6 * O.U * ref["top_logprobs"].abs().nan_to_num(0, 0, 0)
        _close(r.top_logprobs, ref["top_logprobs"], tt, "top_logprobs")
    if grad:
        outs, gs = [full.entropy], [gh.repeat(tile).cuda()]
        if y is not None:
            outs.append(full.logprob)
            gs.append(gl.repeat(tile).cuda())
        dx, = torch.autograd.grad(outs, [xd], gs)
        dx = _first(dx, tile)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        # q carries the sum's error and its exponent's (|log2 q| U, three roundings); log q + H carries both bounds
        lq, _ = O.log_q(x, T)
        q = lq.exp()
        lq = torch.where(q > 0, lq, 0.0)
        eps = O.sum_error(x, T) + 4 * O.U * (2 + 1.45 * lq.abs())
        hh = ref["entropy"].abs().nan_to_num()[:, None]
        a = gl.abs().double()[:, None] + gh.abs().double()[:, None] * (lq.abs() + hh)
        b = gh.abs().double()[:, None] * (th[:, None] + O.sum_error(x, T) + 6 * O.U * (lq.abs() + hh))
        tol = (q * (a * (eps + 8 * O.U) + b) + 4 * O.U * gl.abs().double()[:, None]) / T
        tol = tol.nan_to_num() + O.half_ulp(ref["grad"].nan_to_num(), x.dtype) * (1 + 1e-6)
        _close(dx, ref["grad"], tol, "grad")
    return r


# every launch shape: lane groups (V <= 512), one-wave rows, 256-thread rows, rows cut into segments; odd sizes around each
SIZES = [1, 2, 3, 7, 8, 9, 40, 63, 64, 65, 127, 129, 255, 257, 511, 512, 513, 1000, 1025, 2047, 2049, 4095, 4097, 8193, 16385,
         32000, 32769, 50001, 65537]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", SIZES)
def test_score_sizes(V, dtype):
    R = 9 if V > 600 else 70
    x, at, g = _logits(R, V, dtype, V)
    y = torch.where(torch.rand(R, generator=g) < 0.5, at, torch.randint(0, V, (R,), generator=g))
    y[1] = IGN
    _check_score(x, y, 1.0 if V % 2 else 0.7, min(V, 5))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V,k", [(40, 40), (130, 128), (512, 65), (600, 128), (1500, 64), (4000, 128), (9000, 128), (20000, 33),
                                 (70001, 128), (100003, 1), (1000000, 128), (999999, 20)])
def test_score_top_k(V, k, dtype):
    x, at, _ = _logits(5, V, dtype, k)
    _check_score(x, at, 2.0, k, grad=False)


MANY_KINDS = {
    "normal": lambda V, g: torch.randn(6, V, generator=g) * 2.5,
    "ascending": lambda V, g: (torch.arange(V) / V * 8).expand(6, V).clone(),
    "one_block": lambda V, g: torch.randn(6, V, generator=g) + torch.where((torch.arange(V) // 16) % 9 == 0, 9.0, 0.0),
    "few_values": lambda V, g: torch.randint(0, 5, (6, V), generator=g).float(),
    "heavy_tail": lambda V, g: torch.randn(6, V, generator=g) / torch.rand(6, V, generator=g).clamp_min(1e-3) - 20,
    "few_left": lambda V, g: torch.where(torch.rand(6, V, generator=g) < 0.05, torch.randn(6, V, generator=g), -math.inf),
    "half_left": lambda V, g: torch.where(torch.arange(V) < V // 2, torch.randn(6, V, generator=g), -math.inf),
    "lowest": lambda V, g: torch.where(torch.rand(6, V, generator=g) < 0.5, torch.randn(6, V, generator=g), -65504.0),
}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(MANY_KINDS))
def test_score_many_alternatives(kind, dtype):
    """Sorted short rows, counted bounds of rows on one wave, lists longer than a wave: the same ranking, whatever the values."""
    for V, ks in ((33, (17, 33)), (64, (16, 64)), (100, (20, 21, 100)), (129, (24, 25, 128)), (256, (25, 128)), (257, (1, 13, 128)),
                  (300, (12, 24, 64)), (512, (13, 25, 128)), (700, (24, 25, 90)), (1030, (48, 128)), (2500, (31, 128)),
                  (4091, (64, 128)), (6000, (100,))):
        g = torch.Generator().manual_seed(V)
        x = MANY_KINDS[kind](V, g).to(DTYPES[dtype])
        if kind == "normal":
            x[2, V // 3] = math.nan
        y = x.float().nan_to_num(0.0).argmax(-1)
        for k in ks:
            print(kind, dtype, V, k, flush=True)
            _check_score(x, y, 1.3, k, grad=False)


@pytest.mark.parametrize("V", [40, 700, 5000, 40000])
@pytest.mark.parametrize("kind", ["constant", "two_values", "ascending", "zeros_signed", "mostly_masked"])
def test_score_ties_go_to_the_lowest_index(V, kind):
    R, k = 3, 20
    i = torch.arange(V).float()
    row = {"constant": torch.full((V,), 1.5), "two_values": (i % 2), "ascending": i / V * 8,
           "zeros_signed": torch.where(i % 3 == 0, -0.0, 0.0),
           "mostly_masked": torch.where(i >= V - 7, i / V, -math.inf)}[kind]
    x = row.expand(R, V).contiguous().to(torch.bfloat16)
    _check_score(x, torch.tensor([0, V - 1, V // 2]), 1.0, k)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("second", [1.5, 0.0, -0.0, -2.0, -1000.0])
def test_score_ties_below_the_maximum(second, dtype):
    """A few elements at the top, very many or some hundreds equal ones next: what the lists do not hold is found by counting."""
    for V in (300, 700, 1030, 4091, 5000, 33333, 140001):
        for tied in (V // 2, min(V // 2, 650)):
            g = torch.Generator().manual_seed(V + tied)
            x = torch.randn(3, V, generator=g).abs().neg() * 8 + second - 4
            at = torch.rand(3, V, generator=g).argsort(-1)
            x.scatter_(1, at[:, :tied], second)
            x.scatter_(1, at[:, tied:tied + 5], torch.arange(5.0).expand(3, 5) + 4)
            x[2, at[2, -9:]] = -math.inf
            print(V, tied, second, dtype, flush=True)
            _check_score(x.to(DTYPES[dtype]), at[:, 0], 1.0, 20, grad=False)
            _check_score(x.to(DTYPES[dtype]), at[:, 0], 1.0, 100, grad=False)


@pytest.mark.parametrize("V,k", [(200000, 128), (600000, 100), (600000, 3)])
def test_score_segments_that_share_or_lack_the_top(V, k):
    """Long rows in which the alternatives of all segments lie across each other, in which most segments are ruled out, in
    which one segment holds them all, and in which fewer than k tokens are left."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(5, V, generator=g)
    i = torch.arange(V)
    x[0] = -(i % 5000).float() / 512            # the same values in every segment, many of them equal
    x[1, 20000:] = -math.inf
    x[2, 70000:70200] += 30
    x[3] = -math.inf
    x[3, ::V // 40] = torch.randn(len(x[3, ::V // 40]), generator=g)
    _check_score(x, torch.zeros(5, dtype=torch.int64), 1.0, k, grad=False)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [40, 300, 3000, 40000])
def test_score_rows_that_are_masked_or_not_numbers(V, dtype):
    x, at, _ = _logits(10, V, dtype, 3)
    low = torch.finfo(DTYPES[dtype]).min
    x[0] = -math.inf                      # nothing left
    x[1] = low                            # the type's lowest value everywhere: a uniform row
    x[2, 1:] = low
    x[3, : V - 1] = -math.inf             # one token left
    x[4, 5] = math.nan
    x[5, 7] = math.inf
    x[6] = math.nan                       # an ignored row is not read
    x[7, V // 2:] = -math.inf
    x[8] = x[8].float().add(1000).to(x.dtype)
    at[6] = IGN
    at[9] = V                             # outside the vocabulary
    _check_score(x, at, 1.0, 6)


def test_score_of_a_sure_row_keeps_its_digits():
    """ln(1 + S) with S ~ 1e-6: the log-probability of the favoured token is exact to the sum's relative error, not to 6e-8
    absolute."""
    for V in (40, 600, 9000, 70000):
        x = torch.zeros(2, V)
        x[:, 3] = 13.0 + math.log(V)
        lq, _ = O.log_q(x, 1.0)
        r = TO.token_logprobs(x.cuda(), torch.tensor([3, 3]).cuda())
        rel = (r.logprob.cpu().double() / lq[:, 3] - 1).abs().max()
        assert float(rel) <= O.sum_error(x, 1.0) + 16 * O.U * (13 + math.log(V)), (V, float(rel))


def test_score_without_targets_and_without_rows():
    x, _, _ = _logits(4, 100, "fp32", 1)
    r = _check_score(x, None, 1.0, 3)
    assert r.logprob is None
    r = TO.token_logprobs(torch.empty(0, 7, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 2)
    x = torch.empty(3, 0, 9, device="cuda", requires_grad=True)
    r = TO.token_logprobs(x, torch.empty(3, 0, dtype=torch.int32, device="cuda"))
    assert torch.autograd.grad(r.logprob.sum(), x)[0].shape == x.shape


@pytest.mark.parametrize("V", [40, 601, 33001])
@pytest.mark.parametrize("view", ["shifted", "columns", "transposed", "expanded", "strided_vocab", "four_dims", "offset"])
def test_score_reads_strided_logits_in_place(V, view):
    g = torch.Generator().manual_seed(V)
    if view == "shifted":
        base, cut = torch.randn(3, 6, V, generator=g), (lambda t: t[:, :-1])
    elif view == "columns":
        base, cut = torch.randn(3, 5, V + 3, generator=g), (lambda t: t[..., 1:V + 1])
    elif view == "transposed":
        base, cut = torch.randn(5, 3, V, generator=g), (lambda t: t.transpose(0, 1))
    elif view == "expanded":
        base, cut = torch.randn(1, 5, V, generator=g), (lambda t: t.expand(3, 5, V))
    elif view == "strided_vocab":
        base, cut = torch.randn(3, 5, 2 * V, generator=g), (lambda t: t[..., ::2])
    elif view == "four_dims":
        base, cut = torch.randn(2, 3, 4, V, generator=g), (lambda t: t.permute(2, 0, 1, 3)[:, :, :2])
    else:
        base, cut = torch.randn(1 + 15 * V, generator=g), (lambda t: t[1:].view(3, 5, V))
    base = (base * 3).to(torch.bfloat16)
    x = cut(base)
    lead = x.shape[:-1]
    y_all = torch.randint(0, V, tuple(lead[:-1]) + (lead[-1] + 1,), generator=g)
    y = y_all[..., 1:]
    flat = x.reshape(-1, V)
    gl, gh = torch.randn(lead, generator=g), torch.randn(lead, generator=g)
    ref = O.score(flat, y.reshape(-1), 1.0, 4, IGN, gl.reshape(-1), gh.reshape(-1))
    bd = base.cuda().requires_grad_(True)
    xd = cut(bd)
    r = TO.token_logprobs(xd, y_all.cuda()[..., 1:], top_k=4)
    tl, th = _score_tols(flat, ref, 1.0)
    _close(r.logprob.reshape(-1), ref["logprob"], tl, "logprob")
    assert torch.equal(r.top_ids.reshape(-1, 4).cpu(), ref["top_ids"])
    # the gradient of a view reaches its base: of the contiguous copy it must be the same values
    db, = torch.autograd.grad([r.logprob, r.entropy], [bd], [gl.cuda(), gh.cuda()])
    xc = x.contiguous().cuda().requires_grad_(True)
    rc = TO.token_logprobs(xc, y.contiguous().cuda())
    dc, = torch.autograd.grad([rc.logprob, rc.entropy], [xc], [gl.cuda(), gh.cuda()])
    b2 = base.cuda().requires_grad_(True)
    want, = torch.autograd.grad(cut(b2), b2, dc)
    assert torch.equal(db, want)
    assert torch.equal(r.logprob, rc.logprob) and torch.equal(r.entropy, rc.entropy)


def test_score_int32_targets_and_broadcast_upstream_gradients():
    x, at, _ = _logits(33, 77, "fp32", 5)
    xd = x.cuda().requires_grad_(True)
    a = TO.token_logprobs(xd, at.cuda())
    b = TO.token_logprobs(xd, at.cuda().int())
    assert torch.equal(a.logprob, b.logprob)
    d1, = torch.autograd.grad(a.logprob.sum(), xd)          # an expanded gradient of ones
    d2, = torch.autograd.grad(b.logprob, xd, torch.ones(33, device="cuda"))
    assert torch.equal(d1, d2)


def test_score_gradient_against_differences():
    """Central differences of the fp32 outputs: |f(x + h) - f(x - h)| / 2h with h = 2^-4; truncation h^2 / 6 |f'''| with third
    derivatives of a softmax below 1 for the log-probability and 4 for the entropy of these rows, rounding 2 tol / 2h."""
    x, at, g = _logits(4, 50, "fp32", 8, spread=1.0, peak=1.0)
    h = 2.0 ** -4
    xd = x.cuda().requires_grad_(True)
    r = TO.token_logprobs(xd, at.cuda())
    dx, = torch.autograd.grad((r.logprob + r.entropy).sum(), xd)
    tol = h * h / 6 * 5 + 2 * (O.sum_error(x, 1.0) * 10) / (2 * h)
    for v in (0, 7, 49):
        e = torch.zeros(50)
        e[v] = h
        up, dn = (TO.token_logprobs((x + s * e).cuda(), at.cuda()) for s in (1, -1))
        num = ((up.logprob + up.entropy) - (dn.logprob + dn.entropy)) / (2 * h)
        assert float((num - dx[:, v]).abs().max()) <= tol


@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_score_is_bitwise_reproducible(V):
    x, at, _ = _logits(64, V, "bf16", 4)
    x, at = x.cuda(), at.cuda()
    a = TO.token_logprobs(x, at, top_k=9)
    for _ in range(3):
        b = TO.token_logprobs(x, at, top_k=9)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- distillation ------------------------------------------------------------------------------------------------------
def _teacher(x, K, T, g, truncated=False):
    t = torch.log_softmax((x.float() + torch.randn(x.shape, generator=g)) / T, -1)
    lp, ids = t.topk(min(K, x.shape[-1]), -1)
    if K > x.shape[-1]:
        ids = torch.cat([ids, torch.full((x.shape[0], K - x.shape[-1]), -1)], -1)
        lp = torch.cat([lp, torch.zeros(x.shape[0], K - lp.shape[-1])], -1)
    if truncated:
        ids = torch.where(lp.exp().cumsum(-1) - lp.exp() < 0.8, ids, -1)
    return ids, lp


def _check_distill(x, ids, t, T, tail, w, tile=1, floor=0.0):
    """``floor``: what a gradient may be off by where exponentials underflow."""
    R, V = x.shape
    loss, dx = O.distill(x, ids, t, T, tail, w)
    lq, none = O.log_q(x, T)
    q = lq.exp()
    eps = O.sum_error(x, T)
    wv = torch.ones(R).double() if w is None else w.double()
    there = (ids >= 0) & (ids < V)
    P = 1.0 if tail == "drop" else torch.where(there, t.double(), -math.inf).exp().sum(-1).clamp_min(1.0).nan_to_num(1, 1, 1)
    # d loss / d ln(sum) = sum of all p; the bucket's q_0 carries the same bound once more.  The result is rounded once.
    tl = wv.abs() * T * T * P * 2 * eps + O.U * 2 * loss.abs().nan_to_num(0, 0, 0)
    # gradient: q as in the score's backward pass, A q - p rounds three times
    lq0 = torch.where(q > 0, lq, 0.0)
    e = eps + 4 * O.U * (2 + 1.45 * lq0.abs())
    p = torch.zeros(R, V).double().scatter_add_(1, torch.where(there, ids, 0).long(),
                                                torch.where(there, t.double(), -math.inf).exp()).nan_to_num(0, 0, 0)
    if tail == "drop":
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    # B = A - p0 / q0 carries q0's error: where the rest of the student is small, (p0 / q0) q_v times the bound
    big = (dx.abs() / (wv.abs()[:, None] * T).clamp_min(1e-300)).nan_to_num(0, 0, 0)
    tg = wv.abs()[:, None] * T * ((q * 2 + big) * (2 * e + 8 * O.U) + 6 * O.U * p)
    tg = tg.nan_to_num() + O.half_ulp(dx.nan_to_num(), x.dtype) * (1 + 1e-6) + floor
    xd = x.repeat(tile, 1).cuda().requires_grad_(True)
    i, tt, wd = ids.repeat(tile, 1).cuda(), t.repeat(tile, 1).cuda(), None if w is None else w.repeat(tile).cuda()
    got = TO.topk_distill_loss(xd, i, tt, temperature=T, tail=tail, weight=wd)
    _close(_first(got, tile), loss, tl, "loss")
    ones = torch.ones(R * tile, device="cuda")
    d1, = torch.autograd.grad(got, xd, ones)
    _close(_first(d1, tile), dx, tg, "autograd gradient")
    l2, d2 = TO.topk_distill_grad(xd, i, tt, temperature=T, tail=tail, weight=wd)
    _close(_first(l2, tile), loss, tl, "loss (one pass)")
    _close(_first(d2, tile), dx, tg, "gradient (one pass)")
    assert not l2.requires_grad and not d2.requires_grad
    out = torch.full_like(xd, 3.0)
    l3, d3 = TO.topk_distill_grad(xd, i, tt, temperature=T, tail=tail, weight=wd, out=out)
    assert d3.data_ptr() == out.data_ptr() and _same(d3, d2) and _same(l3, l2)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 40, 64, 65, 129, 257, 512, 513, 1025, 2049, 4097, 8193, 32000, 65537, 70001, 131080])
def test_distill_sizes(V, dtype, tail):
    R = 5 if V > 600 else 37
    x, _, g = _logits(R, V, dtype, V)
    T = 2.0 if V % 2 else 1.0
    ids, t = _teacher(x, min(V, 8), T, g, truncated=V % 3 == 0)
    w = torch.rand(R, generator=g) + 0.5
    w[2] = 0
    _check_distill(x, ids, t, T, tail, w)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("V,K", [(40, 1), (40, 40), (40, 64), (300, 256), (700, 256), (5000, 100), (40000, 256), (80000, 65)])
def test_distill_list_lengths(V, K, tail):
    x, _, g = _logits(3, V, "bf16", K)
    ids, t = _teacher(x, K, 1.0, g)
    _check_distill(x, ids, t, 1.0, tail, None)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("V", [40, 900, 9000, 70001])
def test_distill_odd_entries(V, tail):
    """Ids that repeat, that are absent, that lie behind the vocabulary, entries of no mass, a row without any."""
    x, _, g = _logits(6, V, "fp32", 11)
    ids = torch.randint(0, V, (6, 12), generator=g)
    t = torch.log_softmax(torch.randn(6, 20, generator=g), -1)[:, :12].contiguous()
    ids[0, 1:4] = ids[0, 0]
    ids[0, 7] = ids[0, 6]
    ids[1, ::2] = -1
    ids[2, 3:] = V + torch.arange(9) * (1 << 33)
    t[3, 2:5] = -math.inf
    ids[4] = -1
    ids[5] = ids[5, 0]
    _check_distill(x, ids, t, 1.5, tail, None)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("V", [40, 900, 9000])
def test_distill_masked_students(V, tail):
    x, _, g = _logits(7, V, "bf16", 12)
    ids, t = _teacher(x, 6, 1.0, g)
    low = torch.finfo(torch.bfloat16).min
    x[0] = -math.inf                                    # a student with nothing left: infinite loss, no gradient
    x[1, ids[1, 0]] = -math.inf                         # it rules out the teacher's best token
    x[2] = torch.where(torch.zeros(V, dtype=torch.bool).scatter_(0, ids[2], True), x[2], low)      # no mass outside the list
    x[3, V - 3:] = -math.inf
    x[4] = math.nan
    x[5] = low
    x[6, 9] = math.inf
    w = torch.ones(7)
    w[4] = 0                                            # a row of weight 0 is not read
    _check_distill(x, ids, t, 1.0, tail, w)


def test_distill_strided_logits_and_teacher_types():
    x, _, g = _logits(12, 900, "bf16", 13)
    ids, t = _teacher(x, 7, 1.0, g)
    base = torch.zeros(3, 5, 904, dtype=torch.bfloat16)
    base[:, 1:, 2:902] = x.view(3, 4, 900)
    xd = base.cuda()[:, 1:, 2:902]
    want_l, want_d = TO.topk_distill_grad(x.cuda(), ids.cuda(), t.cuda())
    l, d = TO.topk_distill_grad(xd, ids.view(3, 4, 7).cuda(), t.view(3, 4, 7).cuda())
    assert torch.equal(l.view(-1), want_l) and torch.equal(d.view(12, 900), want_d)
    l, d = TO.topk_distill_grad(xd, ids.int().view(3, 4, 7).cuda(), t.view(3, 4, 7).cuda())
    assert torch.equal(l.view(-1), want_l) and torch.equal(d.view(12, 900), want_d)
    a = TO.topk_distill_loss(xd, ids.view(3, 4, 7).cuda(), t.bfloat16().view(3, 4, 7).cuda())
    b = TO.topk_distill_loss(x.cuda(), ids.cuda(), t.bfloat16().float().cuda())
    assert torch.equal(a.view(-1), b)


def test_distill_gradient_against_differences():
    """Central differences, h = 2^-4: third derivatives of the loss below 2 T^2 / T^3 here."""
    x, _, g = _logits(3, 60, "fp32", 14, spread=1.0, peak=1.0)
    ids, t = _teacher(x, 5, 1.0, g)
    h = 2.0 ** -4
    for tail in ("drop", "bucket"):
        _, dx = TO.topk_distill_grad(x.cuda(), ids.cuda(), t.cuda(), tail=tail)
        tol = h * h / 6 * 2 + 2 * 4 * O.sum_error(x, 1.0) / (2 * h)
        for v in (int(ids[0, 0]), int(ids[1, 3]), 1, 59):
            e = torch.zeros(60)
            e[v] = h
            up, dn = (TO.topk_distill_loss((x + s * e).cuda(), ids.cuda(), t.cuda(), tail=tail) for s in (1, -1))
            assert float(((up - dn) / (2 * h) - dx[:, v]).abs().max()) <= tol


# ---- many short rows (a row a lane) --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 12, 31, 33, 40, 63, 64])
def test_many_short_rows(V, dtype):
    R, tile = 52, 1600                    # 68,800 rows and more
    x, at, g = _logits(R, V, dtype, V)
    at[1] = IGN
    if V > 6:
        x[2] = -math.inf
        x[3] = torch.finfo(DTYPES[dtype]).min
        x[4, 2:] = -math.inf
        x[5, 3] = math.nan
        x[6, 3] = math.inf
        x[7] = 0.5
        x[8, ::2], x[8, 1::2] = 0.0, -0.0
        at[9] = V
    _check_score(x, at, 0.7, min(V, 9), tile=tile)
    _check_score(x, None, 1.0, V, grad=False, tile=tile)
    x = x[9:]
    ids, t = _teacher(x, min(V, 8), 2.0, g, truncated=V == 33)
    w = torch.rand(R - 9, generator=g) + 0.5
    w[2] = 0
    x[2] = math.nan
    for tail in ("drop", "bucket"):
        _check_distill(x, ids, t, 2.0, tail, w, tile=tile)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_many_short_rows_with_odd_entries(tail):
    V, tile = 40, 2200
    x, _, g = _logits(31, V, "fp32", 11)
    ids = torch.randint(0, V, (31, 12), generator=g)
    t = torch.log_softmax(torch.randn(31, 20, generator=g), -1)[:, :12].contiguous()
    ids[0, 1:4] = ids[0, 0]
    ids[1, ::2] = -1
    ids[2, 3:] = V + torch.arange(9) * (1 << 33)
    t[3, 2:5] = -math.inf
    ids[4] = -1
    ids[5] = ids[5, 0]
    x[6] = -math.inf
    x[7, ids[7, 0]] = -math.inf
    x[8] = torch.where(torch.zeros(V, dtype=torch.bool).scatter_(0, ids[8], True), x[8], -math.inf)
    x[9, 4] = math.inf
    _check_distill(x, ids, t, 1.5, tail, None, tile=tile)


# ---- together, streams, graphs --------------------------------------------------------------------------------------------
def test_teacher_to_student():
    """A teacher's top tokens go straight into the student's loss; ignored positions carry no entries."""
    g = torch.Generator().manual_seed(20)
    teacher = (torch.randn(4, 9, 1500, generator=g) * 3).to(torch.bfloat16)
    student = (teacher.float() + torch.randn(4, 9, 1500, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, 1500, (4, 9), generator=g)
    y[0, :3] = IGN
    r = TO.token_logprobs(teacher.cuda(), y.cuda(), temperature=2.0, top_k=10)
    loss, dx = TO.topk_distill_grad(student.cuda(), r.top_ids, r.top_logprobs, temperature=2.0)
    want, dwant = O.distill(student.view(36, -1), r.top_ids.cpu().view(36, 10), r.top_logprobs.cpu().view(36, 10), 2.0, "drop",
                            None)
    assert float(loss[0, :3].abs().max()) == 0 and float(dx[0, :3].float().abs().max()) == 0
    _close(loss.view(-1), want, 4 * 2 * O.sum_error(student, 2.0) + 2 * O.U * want, "loss")


def test_another_stream_than_the_inputs():
    x, at, g = _logits(64, 9000, "fp32", 21)
    ids, t = _teacher(x, 9, 1.0, g)
    xd, at, ids, t = x.cuda(), at.cuda(), ids.cuda(), t.cuda()
    want, wl = TO.token_logprobs(xd, at, top_k=5), TO.topk_distill_grad(xd, ids, t, tail="bucket")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, gl = TO.token_logprobs(xd, at, top_k=5), TO.topk_distill_grad(xd, ids, t, tail="bucket")
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(gl, wl))


@pytest.mark.parametrize("V", [40, 9000, 70001])
def test_captured_and_replayed(V):
    """A captured call reads its inputs anew on every replay, with eager work between the replays; two graphs do not share
    workspace that matters."""
    x, at, g = _logits(6, V, "bf16", 22)
    ids, t = _teacher(x, 6, 1.0, g)
    static = x.cuda()
    at, ids, t = at.cuda(), ids.cuda(), t.cuda()
    other = torch.flip(static, [0])

    def call(z):
        return tuple(TO.token_logprobs(z, at, top_k=5)) + TO.topk_distill_grad(z, ids, t, tail="bucket")

    call(static)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(static)
        graphs.append((gr, out))
    for src in (x.cuda(), other, x.cuda()):
        static.copy_(src)
        want = [v.clone() for v in call(src)]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def _both_backward(x, y, ids, t, w):
    r = TO.token_logprobs(x, y)
    a, = torch.autograd.grad([r.logprob, r.entropy], [x], [torch.ones_like(r.logprob), torch.ones_like(r.entropy)])
    loss = TO.topk_distill_loss(x, ids, t, tail="bucket", weight=w)
    b, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    return a, b


@pytest.mark.parametrize("V", [40, 3000, 70001])
def test_saved_tensors_may_come_back_elsewhere(V):
    """Saved-tensor hooks: what the backward pass reads lies at another address, with other strides, than in the forward."""
    base, at, g = _logits(12, V + 4, "bf16", 25)
    base = base.view(3, 4, V + 4)
    ids, t = _teacher(base.view(12, -1)[:, :V], 5, 1.0, g)
    ids, t, w = ids.view(3, 4, 5).cuda(), t.view(3, 4, 5).cuda(), torch.rand(3, 4, generator=g).cuda()
    y = torch.randint(0, V, (3, 5), generator=g).cuda()[:, 1:]
    leaf = base.cuda().requires_grad_(True)
    want = _both_backward(leaf[..., 2:V + 2], y, ids, t, w)
    with torch.autograd.graph.save_on_cpu():
        got = _both_backward(leaf[..., 2:V + 2], y, ids, t, w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("V", [40, 9000])
def test_backward_passes_captured_into_a_graph(V):
    x, at, g = _logits(8, V, "bf16", 26)
    ids, t = _teacher(x, 5, 1.0, g)
    w = torch.rand(8, generator=g).cuda()
    y, ids, t = at.cuda(), ids.cuda(), t.cuda()
    static = x.cuda()

    def call():
        return _both_backward(static.detach().requires_grad_(True), y, ids, t, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    for src in (x.cuda(), torch.flip(x, [0]).cuda(), x.cuda()):
        static.copy_(src)
        want = [v.clone() for v in call()]
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_differentiated_once():
    x, at, _ = _logits(4, 50, "fp32", 27)
    xd = x.cuda().requires_grad_(True)
    r = TO.token_logprobs(xd, at.cuda())
    d, = torch.autograd.grad(r.logprob.sum(), xd, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    loss = TO.topk_distill_loss(xd, at[:, None].cuda(), torch.zeros(4, 1, device="cuda"))
    d, = torch.autograd.grad(loss.sum(), xd, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_only_one_of_the_outputs_is_differentiated():
    x, at, g = _logits(6, 700, "fp32", 28)
    gl = torch.randn(6, generator=g)
    xd = x.cuda().requires_grad_(True)
    r = TO.token_logprobs(xd, at.cuda(), top_k=3)
    assert not r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    both, = torch.autograd.grad([r.logprob, r.entropy], [xd], [gl.cuda(), torch.zeros(6, device="cuda")], retain_graph=True)
    one, = torch.autograd.grad(r.logprob, xd, gl.cuda(), retain_graph=True)
    assert torch.equal(both, one)
    both, = torch.autograd.grad([r.logprob, r.entropy], [xd], [torch.zeros(6, device="cuda"), gl.cuda()], retain_graph=True)
    one, = torch.autograd.grad(r.entropy, xd, gl.cuda())
    assert torch.equal(both, one)


def test_two_threads_at_once():
    import threading
    x, at, g = _logits(40, 20000, "bf16", 29)
    ids, t = _teacher(x, 7, 1.0, g)
    x, at, ids, t = x.cuda(), at.cuda(), ids.cuda(), t.cuda()
    want = tuple(TO.token_logprobs(x, at, top_k=6)) + TO.topk_distill_grad(x, ids, t)
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = tuple(TO.token_logprobs(x, at, top_k=6)) + TO.topk_distill_grad(x, ids, t)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_far_offsets_in_a_large_tensor():
    """Rows behind 2^32 bytes and 2^31 elements of one tensor."""
    V = 70000
    R = (1 << 31) // V + 8
    big = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    x, at, g = _logits(4, V, "bf16", 23)
    big[-4:] = x.cuda()
    y = torch.full((R,), IGN, dtype=torch.int64)
    y[-4:] = at
    r = TO.token_logprobs(big, y.cuda(), top_k=3)
    want = TO.token_logprobs(x.cuda(), at.cuda(), top_k=3)
    # few rows are cut differently from many: equal up to the sums' bounds, ids exactly
    assert torch.equal(r.top_ids[-4:], want.top_ids)
    assert float((r.logprob[-4:] - want.logprob).abs().max()) <= 2 * O.sum_error(x, 1.0) + 12 * O.U * 40
    w = torch.zeros(R)
    w[-4:] = 1
    ids = torch.zeros(R, 2, dtype=torch.int64)
    ids[-4:, 0], ids[-4:, 1] = at, (at + 1) % V
    t = torch.full((R, 2), math.log(0.5))
    loss, dx = TO.topk_distill_grad(big, ids.cuda(), t.cuda(), weight=w.cuda())
    l4, d4 = TO.topk_distill_grad(x.cuda(), ids[-4:].cuda(), t[-4:].cuda())
    assert float((loss[-4:] - l4).abs().max()) <= 2 * O.sum_error(x, 1.0) + 4 * O.U * float(l4.max())
    assert float(dx[:-4].abs().amax()) == 0
    assert float((dx[-4:].float() - d4.float()).abs().max()) <= 2 ** -7


# ---- rows of large finite values --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,values,T", [
    ("fp32", (1e10, -1e10, 1e12, -1e12, 1e20, -1e20, 1e30, -1e30), 1.0),
    ("fp32", (1e10, -1e10, 1e12, -1e12, 1e20, -1e20, 1e30, -1e30), 0.7),
    ("fp32", (3e9, -3e9, 1e9, -1e9, 2.1e9, -2.1e9, 1e20, -1e20), 0.8),
    ("bf16", (1e10, -1e10, 1e12, -1e12, 1e20, -1e20, 1e30, -1e30), 1.0),
    ("bf16", (1e9, -1e9, 1.4e9, -1.4e9, 1e20, -1e20, 1e30, -1e30), 0.8),
    ("fp16", (65504.0, -65504.0, 60000.0, -60000.0, 30000.0, -30000.0, 777.0, -777.0), 1e-4)])
@pytest.mark.parametrize("V,tile", [(40, 1), (40, 4100), (100, 1), (300, 1), (700, 1), (5000, 1), (70001, 1), (140001, 1)])
def test_rows_of_large_finite_values(V, tile, dtype, values, T):
    """A row filled with one large value is uniform, one with a larger element is sure of it, whatever rounding m c takes."""
    x = torch.tensor(values).to(DTYPES[dtype])[:, None].repeat(2, V)
    n = len(values)
    at = torch.arange(2 * n) % V
    step = x[n:, 0].double() * (1 + 2.0 ** (-7 if dtype == "bf16" else -10 if dtype == "fp16" else -20))
    up = torch.maximum(step, (2 - step / x[n:, 0].double()) * x[n:, 0].double()).to(x.dtype)      # towards plus infinity
    if dtype == "fp16":
        x[n], up[0] = 60000.0, 65504.0
    assert (up > x[n:, 0]).all() and up.isfinite().all()
    x[n:, V // 2] = up
    _check_score(x, at, T, min(V, 6), tile=tile)
    ids = torch.stack([at, (at + 1) % V, torch.full_like(at, V // 2)], 1)
    t = torch.log_softmax(torch.randn(2 * n, 5, generator=torch.Generator().manual_seed(V)), -1)[:, :3].contiguous()
    ids[:, 2] = torch.where(ids[:, :2].eq(V // 2).any(-1), -1, ids[:, 2])
    for tail in ("drop", "bucket"):
        _check_distill(x, ids, t, T, tail, None, tile=tile)


# ---- a student sure of the listed tokens -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V,tile", [(4, 1), (40, 1), (40, 6600), (63, 6600), (100, 1), (300, 1), (500, 1), (700, 1), (5000, 1),
                                    (33000, 1), (70001, 1), (140001, 1)])
def test_bucket_of_a_student_sure_of_its_list(V, tile, dtype):
    """The mass outside the list keeps its logarithm however far below the row's maximum it lies (in z = x / T).

    Some elements lie hundreds of octaves below the others outside the list: exponentials below 2^-126 come out as 0, so with
    w <= 1.5 and A, |B| <= 1 a gradient may be off by 1.5 T 2^-126 (0 for 1e-44 was seen)."""
    g = torch.Generator().manual_seed(V)
    K = min(3, V - 1)
    gaps = torch.tensor([0.0, 30.0, 43.0, 46.0, 80.0, 88.0, 95.0, 104.0, 110.0, 300.0])
    for T in (1.0, 0.05):
        x = torch.randn(10, V, generator=g)
        ids = torch.rand(10, V, generator=g).argsort(-1)[:, :K].contiguous()
        high = (gaps * T)[:, None] + torch.rand(10, K, generator=g) * T + 5
        x.scatter_(1, ids, high)
        x = x.clamp_min(-3)
        if V > 8:
            x[8, ids[8, 0]] = -2.0                    # a listed token among the others
            x[9] = torch.where(torch.zeros(V, dtype=torch.bool).scatter_(0, ids[9], True), x[9],
                               torch.where(torch.arange(V) < V // 2, -math.inf, x[9]))
            x[6] = torch.where(torch.zeros(V, dtype=torch.bool).scatter_(0, ids[6], True), x[6], x[6].sub(
                100 * T * (torch.arange(V) * 8 // V).float()))
        t = (torch.log_softmax(torch.randn(10, K, generator=g), -1) + math.log(0.9)).contiguous()
        w = torch.rand(10, generator=g) + 0.5
        print(V, tile, dtype, T, flush=True)
        _check_distill(x.to(DTYPES[dtype]), ids, t, T, "bucket", w, tile=tile, floor=1.5 * T * 2.0 ** -126)


def test_bucket_gradient_of_a_sure_student_against_differences():
    """The loss of [200, 0, 0, 0] with the list {0: 0.9} falls when an unlisted logit rises, by p_0 / 3 = 1 / 30 each.  Linear in
    the logits there but for the softmax of three: third derivative below p_0; rounding 2 tol / 2h with tol 2 ulp of 20."""
    x, ids, t = torch.tensor([[200.0, 0.0, 0.0, 0.0]]), torch.tensor([[0]]), torch.tensor([[math.log(0.9)]])
    h = 2.0 ** -3
    loss, dx = TO.topk_distill_grad(x.cuda(), ids.cuda(), t.cuda(), tail="bucket")
    assert abs(float(loss) - 19.565) < 1e-2
    for v in range(4):
        e = torch.zeros(1, 4)
        e[0, v] = h
        up, dn = (TO.topk_distill_loss((x + s * e).cuda(), ids.cuda(), t.cuda(), tail="bucket") for s in (1, -1))
        assert abs(float((up - dn) / (2 * h) - dx[0, v])) <= h * h / 6 * 0.1 + 2 * 40 * 2.0 ** -23 / (2 * h)


@pytest.mark.parametrize("V,tile", [(40, 1), (40, 33000), (300, 1), (700, 1), (70001, 1), (140001, 1)])
def test_bucket_at_its_end_and_of_rows_that_are_not_numbers(V, tile):
    """The CPU's rules: less than exp(-745) outside the list is ruled out, NaN anywhere is NaN, no entries compare the whole rows."""
    x = torch.full((9, V), -3.0)
    ids = torch.zeros(9, 2, dtype=torch.int64)
    ids[:, 1] = V - 1
    x[:, 0] = torch.tensor([700.0, 730.0, 760.0, 5000.0, 1e6, 3e38, 20.0, 20.0, 20.0])
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6, V // 2] = math.nan
    x[7, 0] = math.nan                                  # a listed one
    x[8, 0] = math.inf
    t = torch.tensor([[0.6, 0.3]]).log().repeat(9, 1)
    for i in (ids, torch.full_like(ids, -1)):
        want, dwant = TO.topk_distill_grad(x, i, t, tail="bucket")
        xd = x.repeat(tile, 1).cuda().requires_grad_(True)
        a = i.repeat(tile, 1).cuda(), t.repeat(tile, 1).cuda()
        loss, dx = TO.topk_distill_grad(xd, *a, tail="bucket")
        auto = TO.topk_distill_loss(xd, *a, tail="bucket")
        dauto, = torch.autograd.grad(auto, xd, torch.ones_like(auto))
        for l, d in ((_first(loss, tile), _first(dx, tile)), (_first(auto.detach(), tile), _first(dauto, tile))):
            l, d = l.cpu(), d.cpu()
            assert torch.equal(l.isnan(), want.isnan()) and torch.equal(d.isnan(), dwant.isnan())
            tol = 2 * O.sum_error(x, 1.0) + 4 * O.U * want.abs()
            assert ((l - want).abs() <= tol)[~want.isnan()].all()
            assert ((d - dwant).abs() <= 8 * O.sum_error(x, 1.0))[~dwant.isnan()].all()


# ---- ids that repeat ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("V,tile", [(5, 1), (40, 1), (40, 8300), (100, 1), (300, 1), (700, 1), (5000, 1), (70001, 1), (140001, 1)])
def test_a_token_listed_in_parts_counts_as_one(V, tile, tail):
    """Entries of one id add up before the logarithm: a list with tokens in two or three parts is the merged list."""
    g = torch.Generator().manual_seed(V + 1)
    x = torch.randn(8, V, generator=g) * 2
    tok = torch.rand(8, V, generator=g).argsort(-1)[:, :3]
    p = torch.softmax(torch.randn(8, 3, generator=g), -1) * 0.8
    x[0, tok[0, 0]] += 30                               # sure of the token that is listed in parts
    whole_ids = torch.cat([tok, torch.full((8, 4), -1)], 1)
    whole = torch.cat([p, torch.zeros(8, 4)], 1).log()
    parts_ids = torch.cat([tok, tok[:, :1], tok[:, 1:2], tok[:, :1], torch.full((8, 1), V)], 1)
    parts = torch.cat([p * torch.tensor([0.5, 0.25, 1.0]), p[:, :1] * 0.25, p[:, 1:2] * 0.75, p[:, :1] * 0.25,
                       torch.ones(8, 1)], 1).log()
    _check_distill(x, whole_ids, whole, 1.0, tail, None, tile=tile)
    _check_distill(x, parts_ids, parts, 1.0, tail, None, tile=tile)
    want, dwant = O.distill(x, whole_ids, whole, 1.0, tail, None)
    loss, dx = TO.topk_distill_grad(x.cuda(), parts_ids.cuda(), parts.cuda(), tail=tail)
    # the parts' logarithms are rounded once each: |ln p| U of their p, in p ln p and in sums of p
    tol = 2 * O.sum_error(x, 1.0) + 2 * O.U * want.abs() + 12 * O.U * (1 + parts[:, :6].abs().amax(-1).double())
    _close(loss, want, tol, "loss")
    assert float((dx.cpu().double() - dwant).abs().max()) <= 4 * O.sum_error(x, 1.0) + 40 * O.U


# ---- calls that are refused on a GPU, and calls in unusual modes --------------------------------------------------------------
def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    x, at, g = _logits(4, 50, "fp32", 30)
    x, ids, t = x.cuda(), at[:, None].cuda(), torch.zeros(4, 1).cuda()
    w = torch.ones(4).cuda()
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda: TO.token_logprobs(d, at.cuda()), lambda: TO.topk_distill_loss(d, ids, t),
                  lambda: TO.topk_distill_loss(x, ids, fwd.make_dual(t, torch.ones_like(t))),
                  lambda: TO.topk_distill_loss(x, ids, t, weight=fwd.make_dual(w, torch.ones_like(w))),
                  lambda: TO.token_logprobs(d.clone().requires_grad_(True))):
            with pytest.raises(RuntimeError):
                f()
        a = TO.token_logprobs(x, at.cuda())
        _, dx = TO.topk_distill_grad(d, ids, t)             # detached: the values alone
        assert fwd.unpack_dual(dx).tangent is None
    assert all(torch.equal(p, q) for p, q in zip(a[:2], TO.token_logprobs(x, at.cuda())[:2]))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda z: TO.token_logprobs(z, at.cuda()).logprob, (x,), (torch.ones_like(x),))


def test_inference_mode():
    x, at, g = _logits(6, 90, "fp32", 31)
    ids, t = _teacher(x, 5, 1.0, g)
    want = tuple(TO.token_logprobs(x.cuda(), at.cuda(), top_k=3)) + TO.topk_distill_grad(x.cuda(), ids.cuda(), t.cuda())
    with torch.inference_mode():
        xd = x.cuda()
        got = tuple(TO.token_logprobs(xd, at.cuda(), top_k=3)) + TO.topk_distill_grad(xd, ids.cuda(), t.cuda(),
                                                                                     out=torch.empty_like(xd))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ignore_index_beyond_the_targets_type():
    x, _, _ = _logits(4, 30, "fp32", 32)
    y = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
    a, b = TO.token_logprobs(x.cuda(), y, ignore_index=1 << 40), TO.token_logprobs(x.cuda(), y.long())
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.entropy, b.entropy)


# ---- many short rows that do not lie one behind the other ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 13, 40, 64])
@pytest.mark.parametrize("view", ["shifted", "columns", "transposed", "expanded"])
def test_many_short_strided_rows(view, V, dtype):
    """From 65,536 rows on, a view of short rows: the same bits as its contiguous copy (which is tested against the definition)."""
    g = torch.Generator().manual_seed(V)
    n = 66000
    if view == "shifted":
        base, x = (b := torch.randn(120, 551, V, generator=g).to(DTYPES[dtype]).cuda()), b[:, :-1]
    elif view == "columns":
        base, x = (b := torch.randn(n, V + 3, generator=g).to(DTYPES[dtype]).cuda()), b[:, 1:V + 1]
    elif view == "transposed":
        base, x = (b := torch.randn(550, 120, V, generator=g).to(DTYPES[dtype]).cuda()), b.transpose(0, 1)
    else:
        base, x = (b := torch.randn(1, 550, V, generator=g).to(DTYPES[dtype]).cuda()), b.expand(120, 550, V)
    lead = x.shape[:-1]
    y = torch.randint(0, V, lead, generator=g).cuda()
    y.view(-1)[::7] = IGN
    k = min(V, 5)
    a, b = TO.token_logprobs(x, y, top_k=k), TO.token_logprobs(x.contiguous(), y, top_k=k)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    ids, t = a.top_ids, a.top_logprobs
    w = torch.rand(lead, generator=g).cuda()
    for tail in ("drop", "bucket"):
        a, b = (TO.topk_distill_grad(v, ids, t, tail=tail, weight=w) for v in (x, x.contiguous()))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        xa = x.detach().requires_grad_(True)
        loss = TO.topk_distill_loss(xa, ids, t, tail=tail, weight=w)
        assert torch.equal(loss.detach(), b[0])


@pytest.mark.parametrize("V", [40, 300, 9000, 70001, 140001])
def test_rare_rows_captured_and_replayed(V):
    """What only some rows take -- a rest with its own reference, ids that repeat, large values -- is decided anew on every
    replay, forward and backward."""
    g = torch.Generator().manual_seed(V)
    plain = torch.randn(12, V, generator=g)
    ids = torch.rand(12, V, generator=g).argsort(-1)[:, :6].contiguous()
    t = (torch.log_softmax(torch.randn(12, 6, generator=g), -1) + math.log(0.9)).contiguous()
    sure = plain.scatter(1, ids, torch.tensor([0.0, 50.0, 120.0] * 4)[:, None] + torch.rand(12, 6, generator=g))
    large = plain.clone()
    large[::3] = 1e10
    twice = ids.clone()
    twice[::2, 4] = ids[::2, 1]
    z, i, tt = plain.cuda(), ids.cuda(), t.cuda()

    def call(z, i):
        x = z.detach().requires_grad_(True)
        loss = TO.topk_distill_loss(x, i, tt, tail="bucket")
        dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        s = TO.token_logprobs(z, i[:, 0], top_k=3)
        return (loss.detach(), dx) + TO.topk_distill_grad(z, i, tt, tail="bucket") + tuple(s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(z, i)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call(z, i)
    for src, si in ((plain, ids), (sure, ids), (large, twice), (sure, twice), (plain, ids)):
        z.copy_(src)
        i.copy_(si)
        want = [v.clone() for v in call(src.cuda(), si.cuda())]
        gr.replay()
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(out, want))
