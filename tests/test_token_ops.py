"""Token operators (ops/token_ops.py) on the CPU: the torch forms against the definitions in 64 bits, and the refusals."""
import math

import pytest
import torch

from . import token_oracle as O
from serann.ops import token_ops as TO

IGN = -100


def _rows(R, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * 3).to(dtype), torch.randint(0, V, (R,), generator=g), g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,k", [(1, 1), (40, 5), (300, 0)])
def test_score_matches_the_definition(V, k, dtype):
    x, y, g = _rows(8, V, V, dtype)
    y[2] = IGN
    gl, gh = torch.randn(8, generator=g), torch.randn(8, generator=g)
    x[3, 1:] = -math.inf
    ref = O.score(x, y, 0.7, k, IGN, gl, gh)
    xd = x.clone().requires_grad_(True)
    r = TO.token_logprobs(xd, y, temperature=0.7, top_k=k)
    tol = 64 * O.U * 20
    assert torch.allclose(r.logprob.double(), ref["logprob"], rtol=tol, atol=tol)
    assert torch.allclose(r.entropy.double(), ref["entropy"], rtol=tol, atol=tol)
    dx, = torch.autograd.grad([r.logprob, r.entropy], [xd], [gl, gh])
    lim = O.half_ulp(ref["grad"], dtype) + tol * 4
    assert ((dx.double() - ref["grad"]).abs() <= lim).all()
    if k:
        assert torch.equal(r.top_ids, ref["top_ids"])
    else:
        assert r.top_ids is None and r.top_logprobs is None


def test_score_odd_rows():
    x, y, _ = _rows(6, 40, 1)
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2, 3] = math.inf
    x[3] = math.nan
    y[3] = IGN
    y[4] = 40
    x.requires_grad_(True)
    r = TO.token_logprobs(x, y, top_k=3)
    ref = O.score(x.detach(), y, 1.0, 3, IGN)
    assert r.logprob[0] == -math.inf and r.entropy[0] == 0
    assert r.logprob[[1, 2, 4]].isnan().all() and r.logprob[3] == 0 and r.entropy[3] == 0
    assert torch.equal(r.top_ids, ref["top_ids"])
    assert r.top_ids[[1, 2, 3]].eq(-1).all()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("V,K", [(1, 1), (40, 8), (40, 40), (300, 12)])
def test_distill_matches_the_definition(V, K, tail):
    x, _, g = _rows(7, V, K)
    ids = torch.randint(0, V, (7, K), generator=g)
    t = torch.log_softmax(torch.randn(7, K + 3, generator=g), -1)[:, :K].contiguous()
    if K > 4:
        ids[0, 1] = ids[0, 0]
        ids[1, 2:] = -1
        ids[2, 3] = V
        ids[3] = -1
        t[4, 1] = -math.inf
    w = torch.rand(7, generator=g) + 0.5
    w[6] = 0
    x[6] = math.nan
    loss, dx = O.distill(x, ids, t, 2.0, tail, w)
    l, d = TO.topk_distill_grad(x, ids, t, temperature=2.0, tail=tail, weight=w)
    assert torch.allclose(l.double(), loss, rtol=4 * O.U, atol=1e-9)
    assert torch.allclose(d.double(), dx, rtol=4 * O.U, atol=4 * O.U)
    xd = x.clone().requires_grad_(True)
    l2 = TO.topk_distill_loss(xd, ids, t, temperature=2.0, tail=tail, weight=w)
    d2, = torch.autograd.grad(l2.sum(), xd)
    assert torch.equal(l2.detach(), l) and torch.equal(d2, d)


def test_teacher_to_student():
    t, y, g = _rows(9, 40, 4)
    s = t + torch.randn(9, 40, generator=g)
    y[1] = IGN
    r = TO.token_logprobs(t, y, top_k=6, temperature=1.5)
    loss = TO.topk_distill_loss(s, r.top_ids, r.top_logprobs, temperature=1.5)
    want, _ = O.distill(s, r.top_ids, r.top_logprobs, 1.5, "drop", None)
    assert loss[1] == 0 and torch.allclose(loss.double(), want, rtol=4 * O.U, atol=1e-9)


def test_score_refusals():
    x, y, _ = _rows(4, 10, 0)
    ok = TO.token_logprobs
    for bad in (x.double(), x.long(), [[1.0]]):
        with pytest.raises(TypeError):
            ok(bad, y)
    for bad in (torch.zeros(4, 0), torch.tensor(1.0), torch.zeros(1, (1 << 20) + 1)):
        with pytest.raises(ValueError):
            ok(bad)
    for T in (0.0, -1.0, math.nan, math.inf, 1e-9):
        with pytest.raises(ValueError):
            ok(x, y, temperature=T)
    for k in (-1, 11, 200):
        with pytest.raises(ValueError):
            ok(x, y, top_k=k)
    with pytest.raises(ValueError):
        ok(torch.zeros(2, 500), top_k=129)
    for kw in (dict(top_k=2.0), dict(top_k=None), dict(ignore_index=None), dict(ignore_index=-1.0)):
        with pytest.raises(TypeError):
            ok(x, y, **kw)
    with pytest.raises(ValueError):
        ok(x, y, ignore_index=1 << 70)
    with pytest.raises(TypeError):
        ok(x, y.float())
    with pytest.raises(TypeError):
        ok(x, [1, 2, 3, 4])
    for bad in (y[:3], y[:, None], y.new_zeros(())):
        with pytest.raises(ValueError):
            ok(x, bad)
    with pytest.raises(ValueError):
        ok(x, torch.zeros(4, dtype=torch.int64, device="meta"))


def test_distill_refusals():
    x, _, _ = _rows(4, 10, 0)
    ids, t = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    for f in (TO.topk_distill_loss, TO.topk_distill_grad):
        for args in ((x.double(), ids, t), (x, ids.float(), t), (x, ids, t.double()), (x, ids, t.long())):
            with pytest.raises(TypeError):
                f(*args)
        for args in ((x, ids[:, :2], t), (x, ids[:3], t[:3]), (x, ids[..., None], t[..., None]),
                     (x, torch.zeros(4, 0, dtype=torch.int64), torch.zeros(4, 0)),
                     (x, torch.zeros(4, 257, dtype=torch.int64), torch.zeros(4, 257)),
                     (x, ids, t.clone().requires_grad_(True))):
            with pytest.raises(ValueError):
                f(*args)
        with pytest.raises(ValueError):
            f(x, ids, t, tail="sum")
        with pytest.raises(ValueError):
            f(x, ids, t, temperature=0)
        with pytest.raises(ValueError):
            f(x, ids, t, weight=torch.ones(3))
        with pytest.raises(TypeError):
            f(x, ids, t, weight=torch.ones(4, dtype=torch.int64))
        with pytest.raises(ValueError):
            f(x, ids, t, weight=torch.ones(4, requires_grad=True))
    for out in (torch.zeros(4, 9), torch.zeros(4, 10, dtype=torch.bfloat16), torch.zeros(4, 20)[:, ::2], x):
        with pytest.raises(ValueError):
            TO.topk_distill_grad(x, ids, t, out=out)


def test_gradient_into_a_given_tensor():
    """``out`` may lie beside the arguments in one allocation, but overlap none of them; autograd sees that it was written."""
    g = torch.Generator().manual_seed(11)
    ids = torch.randint(0, 10, (4, 3), generator=g)
    flat = torch.randn(140, generator=g)
    x, t, w = flat[:40].view(4, 10), flat[40:52].view(4, 3), flat[52:56]
    want_loss, want = TO.topk_distill_grad(x, ids, t, weight=w)
    for start in (1, 13, 39, 40, 51, 55):                  # over the logits, the teacher, the weights
        with pytest.raises(ValueError):
            TO.topk_distill_grad(x, ids, t, weight=w, out=flat[start:start + 40].view(4, 10))
    with pytest.raises(ValueError):
        TO.topk_distill_grad(x, ids, t, out=torch.zeros(4, 10, requires_grad=True))
    with pytest.raises(TypeError):
        TO.topk_distill_grad(x, ids, t, out=[0.0])
    out = flat[56:96].view(4, 10)
    loss, dx = TO.topk_distill_grad(x, ids, t, weight=w, out=out)
    assert dx is out and torch.equal(dx, want) and torch.equal(loss, want_loss)
    a = torch.ones(4, 10, requires_grad=True)
    out = torch.zeros(4, 10)
    y = (a * out).sum()
    TO.topk_distill_grad(x, ids, t, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_row_layouts():
    """Strided rows are described, not copied, where two strides do."""
    x = torch.zeros(3, 6, 10)
    for v, want in ((x, (18, 18, 0, 10)), (x[:, :-1], (15, 5, 60, 10)), (x[..., 1:9], (18, 18, 0, 10)),
                    (x.transpose(0, 1), (18, 3, 10, 60)), (x[:, :1], (3, 3, 0, 60)), (x[:1].expand(4, 6, 10), (24, 6, 0, 10))):
        y, rows, n1, s0, s1 = TO._rows(v)
        assert y.data_ptr() == v.data_ptr() and (rows, n1, s0, s1) == want, (v.shape, v.stride())
        off = [(r // n1) * s0 + (r % n1) * s1 for r in range(rows)]
        base = torch.arange(x.numel()).as_strided(v.shape, v.stride())
        assert off == (base[..., 0].reshape(-1)).tolist()
    y = TO._rows(torch.zeros(3, 5, 20)[..., ::2])[0]
    assert y.is_contiguous()
    y = TO._rows(torch.zeros(2, 3, 4, 7).permute(2, 0, 1, 3)[:, :, :2])[0]
    assert y.is_contiguous()


@pytest.mark.parametrize("T", [1.0, 0.05])
def test_bucket_of_a_student_sure_of_its_list(T):
    """The student's mass outside the list counts by its logarithm, down to exp(-745); below that it is ruled out."""
    p = 0.9
    for gap in (30.0, 87.0, 110.0, 200.0, 500.0, 740.0):
        x = torch.tensor([[gap * T, 0.0, 0.0, 0.0]])
        ids, t = torch.tensor([[0]]), torch.tensor([[math.log(p)]])
        p64 = math.exp(float(t.double()))
        gap64 = float(x[0, 0].double()) / T
        p0, lq0 = 1 - p64, math.log(3) - gap64 - math.log1p(3 * math.exp(-gap64))
        want = T * T * (p64 * (math.log(p64) + math.log1p(3 * math.exp(-gap64))) + p0 * (math.log(p0) - lq0))
        loss, dx = TO.topk_distill_grad(x, ids, t, temperature=T, tail="bucket")
        assert abs(float(loss) - want) <= 4 * O.U * abs(want), gap
        want_dx = torch.tensor([[p0, -p0 / 3, -p0 / 3, -p0 / 3]]).double() * T
        assert torch.allclose(dx.double(), want_dx, rtol=4 * O.U + 3 * math.exp(-gap64) * 10, atol=0), gap
    for rest in (-800 * T, torch.finfo(torch.float32).min, -math.inf):
        x = torch.tensor([[0.0, rest, rest, rest]])
        loss, dx = TO.topk_distill_grad(x, ids, t, temperature=T, tail="bucket")
        assert abs(float(loss) - T * T * p64 * math.log(p64)) <= 4 * O.U * T * T and float(dx.abs().max()) == 0


def test_bucket_of_a_row_that_is_not_a_number():
    """A teacher row without entries compares the whole rows: nothing is lost, unless the student is not a number."""
    x = torch.tensor([[0.0, 1.0], [math.nan, 1.0]])
    loss = TO.topk_distill_loss(x, torch.full((2, 1), -1), torch.zeros(2, 1), tail="bucket")
    assert abs(float(loss[0])) <= 1e-12 and loss[1].isnan()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_a_token_listed_in_parts_counts_as_one(tail):
    """Entries of one id add up before the logarithm: two halves on a student's sure token are no divergence."""
    x = torch.tensor([[30.0, 0.0, 0.0]])
    loss, dx = TO.topk_distill_grad(x, torch.tensor([[0, 0]]), torch.tensor([[0.5, 0.5]]).log(), tail=tail)
    whole, dwhole = TO.topk_distill_grad(x, torch.tensor([[0]]), torch.zeros(1, 1), tail=tail)
    # each half's logarithm is rounded once: 2 |ln 0.5| U of the mass
    assert abs(float(loss - whole)) <= 2 * O.U and float((dx - dwhole).abs().max()) <= 2 * O.U
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 40, generator=g) * 3
    tok = torch.rand(6, 40, generator=g).argsort(-1)[:, :3]
    p = torch.softmax(torch.randn(6, 3, generator=g), -1) * 0.8
    parts_ids = torch.cat([tok[:, 1:], torch.full((6, 1), 40), tok, tok[:, :1]], 1)
    parts = torch.cat([p[:, 1:] * 0.25, torch.ones(6, 1), p * torch.tensor([0.5, 0.75, 0.75]), p[:, :1] * 0.5], 1).log()
    loss, dx = TO.topk_distill_grad(x, parts_ids, parts, tail=tail)
    want, dwant = TO.topk_distill_grad(x, tok, p.log(), tail=tail)
    tol = 12 * O.U * (1 + parts.abs().amax(-1))
    assert ((loss - want).abs() <= tol + 4 * O.U * want.abs()).all()
    assert ((dx - dwant).abs() <= 12 * O.U).all()


def test_launchers_refuse_tensors_without_storage():
    """Pointer 0 (a functionalised tensor's) never reaches a kernel."""
    from serann.ops import hip_ops as H
    lib = H.lib(required=False)
    if lib is None:
        pytest.skip("extension not built")
    P = 64                                    # P: never read, every call is refused before its launch
    score = [P, 0, 1, 1, 0, 9, 9, 1.0, P, 1, 0, 1, -100, 2, P, P, P, P, 0, 0, 0]
    sgrad = [P, 0, 1, 1, 0, 9, 9, 1.0, P, 1, 0, 1, -100, P, P, P, P, 0]
    dist = [P, 0, 1, 1, 0, 9, 9, 1.0, P, 1, P, 0, 3, 0, P, 0, P, P, 0, 0]
    dgrad = [P, 0, 1, 1, 0, 9, 9, 1.0, P, 1, 0, 3, 0, P, P, P, 0]
    for f, args, needed in ((lib.tok_score, score, (0, 8, 15, 16, 17)), (lib.tok_score_grad, sgrad, (0, 15, 16)),
                            (lib.tok_distill, dist, (0, 8, 10, 14)), (lib.tok_distill_grad, dgrad, (0, 8, 13, 14, 15))):
        for i in needed:
            with pytest.raises(RuntimeError, match="no storage"):
                f(*(0 if j == i else v for j, v in enumerate(args)))


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_inference_mode(tail):
    """The gradient in one call needs no autograd of the caller's: inference mode and its tensors do, inside and outside."""
    x, _, g = _rows(5, 12, 2)
    ids, t, w = torch.randint(0, 12, (5, 3), generator=g), torch.full((5, 3), -1.5), torch.rand(5, generator=g)
    want = TO.topk_distill_grad(x, ids, t, weight=w, tail=tail)
    with torch.inference_mode():
        a = [v.clone() for v in (x, ids, t, w)]
        assert a[0].is_inference()
        got = TO.topk_distill_grad(*a[:3], weight=a[3], tail=tail, out=torch.empty_like(a[0]))
        mixed = TO.topk_distill_grad(x, ids, t, weight=w, tail=tail)
        score = TO.token_logprobs(a[0], a[1][:, 0], top_k=2)
    later = TO.topk_distill_grad(*a[:3], weight=a[3], tail=tail)
    for r in (got, mixed, later):
        assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])
    assert all(torch.equal(p, q) for p, q in zip(score, TO.token_logprobs(x, ids[:, 0], top_k=2)))


def test_ignore_index_beyond_the_targets_type():
    """int32 targets and an index of 64 bits: none of them is ignored."""
    x, _, _ = _rows(4, 10, 5)
    y = torch.arange(4, dtype=torch.int32)
    a = TO.token_logprobs(x, y, ignore_index=1 << 40)
    b = TO.token_logprobs(x, y.long())
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.entropy, b.entropy)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_per_row_transforms(tail):
    """On the CPU a row at a time under vmap, and its gradient, are the batch's."""
    x, _, g = _rows(5, 12, 4)
    ids, t = torch.randint(0, 12, (5, 3), generator=g), torch.full((5, 3), -1.5)
    loss, dx = TO.topk_distill_grad(x, ids, t, tail=tail)
    f = lambda a, b, c: TO.topk_distill_loss(a, b, c, tail=tail)
    assert torch.allclose(torch.func.vmap(f)(x, ids, t), loss, rtol=2 * O.U, atol=1e-9)
    assert torch.allclose(torch.func.vmap(torch.func.grad(f))(x, ids, t), dx, rtol=4 * O.U, atol=4 * O.U)
