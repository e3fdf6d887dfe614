"""Operators on rows of token logits: log-probabilities of given tokens with the entropy and the top alternatives of each
position, and the distillation loss from a teacher's top tokens, each with its gradient.

The reference scores a sequence as a whole (ribosomal_autoencoder/model.py:45-59: log_softmax, gather, sum over the positions;
``ops.riboae_ops.categorical_loglik`` here).  These give what that sum hides -- how sure a decode is of every token, and which
tokens come next -- and train a model from another one's answers:

* :func:`token_logprobs`     -- log p of the given tokens, entropy, the ``top_k`` best tokens; differentiable;
* :func:`topk_distill_loss`  -- KL divergence from a teacher's top tokens, a loss for each row; differentiable;
* :func:`topk_distill_grad`  -- the same loss and its gradient in one pass over the logits, for trainers that run their own
  backward (``riboae.hip_trainer``).

Logits are ``(..., V)``, float32, bfloat16 or float16, 1 <= V <= 1,000,000.  Leading dimensions may have any strides (a slice
``logits[:, :-1]`` is read in place); the last one is copied if it is not contiguous.  Sums are taken in float32 or wider,
whatever the logits' type; results are float32, gradients (in backward mode; tensors with a forward-mode tangent are an error on
a GPU) have the logits' type.  ``-inf`` logits are tokens ruled out: they have probability 0, and gradient 0 unless they are the
target or in the teacher's list (the formula's then, next to an infinite loss).  A row of nothing but ``-inf`` has
log-probabilities ``-inf``, entropy 0 and no gradient.  A row with a NaN or ``+inf`` logit gives NaN.

On a GPU the HIP kernels of ``csrc/hip/token_score.hip`` and ``csrc/hip/token_distill.hip`` run, on the current stream of the
logits' device; a GPU without the built extension is an error.  On the CPU the same formulas run as torch operations.
"""
from __future__ import annotations

import functools
import math
import operator
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import hip_ops as H

MAX_TOP_K = 128          # csrc/hip/token.h TOK_MAX_K
MAX_TEACHER_K = 256      # csrc/hip/token_distill.hip DIST_MAX_K
MAX_VOCAB = 1_000_000    # csrc/hip/token.h TOK_MAX_V
MIN_LOG_REST = -745.0    # the least logarithm of the student's mass outside the list, csrc/hip/token_distill.hip dist_finish
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TAILS = {"drop": 0, "bucket": 1}


class TokenLogprobs(NamedTuple):
    """Results of :func:`token_logprobs`; ``None`` for what was not asked for."""
    logprob: Optional[torch.Tensor]         # (...) float32
    entropy: torch.Tensor                   # (...) float32, natural logarithm
    top_ids: Optional[torch.Tensor]         # (..., top_k) int64
    top_logprobs: Optional[torch.Tensor]    # (..., top_k) float32


# ------------------------------------------------------------------------------------------------
# argument checks
# ------------------------------------------------------------------------------------------------
def _check_logits(logits, temperature):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        raise TypeError("logits must be a float32, bfloat16 or float16 tensor")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"logits must be (..., V) with 1 <= V <= {MAX_VOCAB}, got {tuple(logits.shape)}")
    if logits.numel() // logits.shape[-1] >= 1 << 31:
        raise ValueError("logits must have fewer than 2**31 rows")
    temperature = float(temperature)
    if not (1e-4 <= temperature <= 1e4):
        raise ValueError(f"temperature must be in [1e-4, 1e4], got {temperature}")
    return temperature


def _check_ints(t, name, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be an int64 or int32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits on {device}")


def _check_teacher(logits, ids, logprobs, tail, weight):
    if not isinstance(logprobs, torch.Tensor) or logprobs.dtype not in _DTYPES:
        raise TypeError("teacher_logprobs must be a float32, bfloat16 or float16 tensor")
    if logprobs.dim() != logits.dim() or logprobs.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"teacher_logprobs must be {tuple(logits.shape[:-1])} + (K,), got {tuple(logprobs.shape)}")
    if not 1 <= logprobs.shape[-1] <= MAX_TEACHER_K:
        raise ValueError(f"1 to {MAX_TEACHER_K} teacher entries a row, got {logprobs.shape[-1]}")
    if logprobs.device != logits.device:
        raise ValueError(f"teacher_logprobs is on {logprobs.device}, the logits on {logits.device}")
    _check_ints(ids, "teacher_ids", logprobs.shape, logits.device)
    if tail not in _TAILS:
        raise ValueError(f"tail must be one of {sorted(_TAILS)}, got {tail!r}")
    if logprobs.requires_grad:
        raise ValueError("teacher_logprobs must not require a gradient (detach the teacher)")
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or not weight.is_floating_point():
            raise TypeError("weight must be a floating point tensor")
        if weight.shape != logits.shape[:-1]:
            raise ValueError(f"weight must have shape {tuple(logits.shape[:-1])}, got {tuple(weight.shape)}")
        if weight.device != logits.device:
            raise ValueError(f"weight is on {weight.device}, the logits on {logits.device}")
        if weight.requires_grad:
            raise ValueError("weight must not require a gradient")


# ------------------------------------------------------------------------------------------------
# layouts: rows of an (n0, n1, V) view, read in place
# ------------------------------------------------------------------------------------------------
def _two_dims(shape, strides):
    """(n1, s0, s1): strides in elements of leading dimensions joined to at most two, or None."""
    dims = []                                     # outermost first; joined where the strides allow
    for n, s in zip(shape, strides):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    if len(dims) == 0:
        return 1, 0, 0
    if len(dims) == 1:
        return dims[0][0], 0, dims[0][1]
    if len(dims) == 2:
        return dims[1][0], dims[0][1], dims[1][1]
    return None


def _rows(x):
    """x (..., V) -> (x or a copy, rows, n1, s0, s1) with a unit stride inside a row."""
    V = x.shape[-1]
    if x.is_contiguous():
        rows = x.numel() // V
        return x, rows, max(rows, 1), 0, V
    lay = _two_dims(x.shape[:-1], x.stride()[:-1]) if V == 1 or x.stride(-1) == 1 else None
    if lay is None:
        return _rows(x.contiguous())
    return (x, x.numel() // V) + lay


def _same_rows(y, n1, rows):
    """Strides of y's rows for rows numbered as (r // n1, r % n1), or a contiguous copy."""
    if not y.is_contiguous():
        lay = _two_dims(y.shape, y.stride())
        if lay is not None and (lay[0] == n1 or n1 == rows == lay[0]):
            return y, lay[1], lay[2]
        y = y.contiguous()
    return y, n1, 1


@functools.lru_cache(maxsize=1024)
def _score_segments(V, code):
    return H.lib().tok_score_segments(V, code)


@functools.lru_cache(maxsize=1024)
def _distill_segments(V, code, grad):
    return H.lib().tok_distill_segments(V, code, grad)


def _span(t):
    """[first, last) byte of what a tensor's elements cover."""
    if t.numel() == 0:
        return 0, 0
    n = 1 + sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _check_out(out, logits, *inputs):
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a tensor")
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of the logits' shape, type and device")
    if out.requires_grad:
        raise ValueError("out must not require a gradient")
    lo, hi = _span(out)
    for t in (logits,) + inputs:
        if t is not None:
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError("out must not share memory with the logits or another argument")


def _no_tangent(*tensors):
    """Forward-mode differentiation: the kernels go by a tensor's pointer and would drop its tangent without a word."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the token operators have no forward-mode derivative on a GPU")


# the current stream of a device as the launchers take it; torch.cuda.current_stream() builds a Stream object first (2 of the
# 16 us that a small call took)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on_device(f):
    """f(logits, ...) with the logits' device as the current one; entering a device context costs more than to ask."""
    @functools.wraps(f)
    def run(logits, *args):
        if torch.cuda.current_device() == logits.device.index:
            return f(logits, *args)
        with torch.cuda.device(logits.device):
            return f(logits, *args)
    return run


def _once(backward):
    """``once_differentiable`` whose wrapping is paid for only under create_graph (5 us a call otherwise)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


# ------------------------------------------------------------------------------------------------
# log-probabilities
# ------------------------------------------------------------------------------------------------
@_on_device
def _score_hip(logits, targets, temperature, top_k, ignore_index, want_stat):
    """(logprob, entropy, top ids, top log-probabilities, what the backward pass needs)."""
    x, rows, n1, s0, s1 = _rows(logits)
    shape, V, code = logits.shape, logits.shape[-1], _DTYPES[logits.dtype]
    lead = shape[:-1]
    lp = ids = top = saved = ws = None
    y, y64, t0, t1, yp, lpp = None, False, 0, 0, 0, 0
    if targets is not None:
        y, t0, t1 = _same_rows(targets, n1, rows)
        y64 = y.dtype == torch.int64
        lp = x.new_empty(lead, dtype=torch.float32)
        yp, lpp = y.data_ptr(), lp.data_ptr()
    ent = x.new_empty(lead, dtype=torch.float32)
    idp = topp = stp = wsp = 0
    if top_k:
        ids = x.new_empty(lead + (top_k,), dtype=torch.int64)
        top = x.new_empty(lead + (top_k,), dtype=torch.float32)
        idp, topp = ids.data_ptr(), top.data_ptr()
    if want_stat:
        stat = x.new_empty((rows, 3), dtype=torch.float32)
        stp = stat.data_ptr()
        saved = (x, y, stat)
    nseg = _score_segments(V, code)
    if nseg > 1:
        ws = x.new_empty(rows * nseg * (2 + top_k), dtype=torch.int64)
        wsp = ws.data_ptr()
    H.lib().tok_score(x.data_ptr(), code, rows, n1, s0, s1, V, temperature, yp, y64, t0, t1, ignore_index, top_k, lpp,
                      ent.data_ptr(), idp, topp, stp, wsp, _raw_stream(logits.device.index))
    return lp, ent, ids, top, saved


@_on_device
def _score_grad_hip(x, y, stat, temperature, ignore_index, glp, gent, shape):
    # the layout again: saved tensors may come back elsewhere and with other strides (saved-tensor hooks)
    x, rows, n1, s0, s1 = _rows(x)
    y, t0, t1 = _same_rows(y, n1, rows) if y is not None else (None, 0, 0)
    dx = x.new_empty(shape)
    H.lib().tok_score_grad(x.data_ptr(), _DTYPES[x.dtype], rows, n1, s0, s1, x.shape[-1], temperature, H.ptr(y),
                           y is not None and y.dtype == torch.int64, t0, t1, ignore_index, H.ptr(glp), H.ptr(gent),
                           stat.contiguous().data_ptr(), dx.data_ptr(), _raw_stream(x.device.index))
    return dx


def _f32(g):
    return g if g is None or (g.dtype == torch.float32 and g.is_contiguous()) else g.float().contiguous()


class _Score(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, top_k, ignore_index, extra):
        lp, ent, ids, top, saved = _score_hip(logits, targets, temperature, top_k, ignore_index, True)
        ctx.save_for_backward(*saved)
        ctx.args = (temperature, ignore_index)
        ctx.shape = logits.shape
        ctx.set_materialize_grads(False)
        extra += (ids, top)                     # no gradients: kept out of the graph
        return ent if lp is None else (ent, lp)

    @staticmethod
    @_once
    def backward(ctx, gent, glp=None):
        if glp is None and gent is None:
            return None, None, None, None, None, None
        x, y, stat = ctx.saved_tensors
        dx = _score_grad_hip(x, y, stat, *ctx.args, _f32(glp), _f32(gent), ctx.shape)
        return dx, None, None, None, None, None


def _log_softmax(logits, temperature):
    """(x / T in float32 or wider, its log-softmax, rows that are all -inf)."""
    z = (logits if logits.dtype == torch.float64 else logits.float()) / temperature
    none = (z == -math.inf).all(-1, keepdim=True)
    lq = torch.log_softmax(torch.where(none, 0.0, z), -1)
    return torch.where(none, -math.inf, lq), none


def _score_torch(logits, targets, temperature, top_k, ignore_index):
    skip = (targets.long() == ignore_index) if targets is not None else None      # an int32 comparison would wrap the index
    if skip is not None:
        logits = torch.where(skip.unsqueeze(-1), 0.0, logits)           # not read
    lq, none = _log_softmax(logits, temperature)
    # the discarded branch of a where must not put a NaN into the gradient: 0 * log 0 is taken over finite values
    ent = -(lq.exp() * torch.where(lq > -math.inf, lq, torch.where(lq.isnan(), lq, 0.0))).sum(-1)
    lp = ids = top = None
    if targets is not None:
        V = logits.shape[-1]
        ok = (targets >= 0) & (targets < V)
        lp = lq.gather(-1, torch.where(ok, targets, 0).long().unsqueeze(-1)).squeeze(-1)
        lp = lp * torch.where(ok | skip, 1.0, math.nan)
        lp, ent = torch.where(skip, 0.0, lp), torch.where(skip, 0.0, ent)
    if top_k:
        with torch.no_grad():
            bad = lq.isnan().any(-1, keepdim=True)
            ids = torch.sort(logits.detach().float(), dim=-1, descending=True, stable=True).indices[..., :top_k]
            top = torch.where(bad, math.nan, lq.gather(-1, ids))
            ids = torch.where(bad, -1, ids)
            if skip is not None:
                ids = torch.where(skip.unsqueeze(-1), -1, ids)
                top = torch.where(skip.unsqueeze(-1), -math.inf, top)
    return TokenLogprobs(lp, ent, ids, top)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, temperature: float = 1.0, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log-probabilities of ``targets`` under ``softmax(logits / temperature)``, with the entropy of each row and its
    ``top_k`` most likely tokens (0: none, at most 128).

    ``targets`` (int64 / int32, the shape of ``logits`` without its last dimension): rows whose target is ``ignore_index`` are
    not read -- log-probability and entropy 0, top ids -1 with ``-inf``, gradient 0.  Any other target outside ``[0, V)``
    gives NaN.  Without ``targets`` there is no ``logprob``.

    ``top_ids`` are ordered by logit, equal ones by index; ``top_logprobs`` are their log-probabilities.  Rows whose
    log-probabilities are NaN have ids -1.  ``logprob`` and ``entropy`` have gradients, the alternatives do not."""
    temperature = _check_logits(logits, temperature)
    if targets is not None:
        _check_ints(targets, "targets", logits.shape[:-1], logits.device)
    top_k, ignore_index = operator.index(top_k), operator.index(ignore_index)
    if not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must fit 64 bits")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"top_k must be in [0, min({MAX_TOP_K}, V = {logits.shape[-1]})], got {top_k}")
    if not logits.is_cuda:
        return _score_torch(logits, targets, temperature, top_k, ignore_index)
    _no_tangent(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        extra = []
        out = _Score.apply(logits, targets, temperature, top_k, ignore_index, extra)
        return TokenLogprobs(None, out, *extra) if targets is None else TokenLogprobs(out[1], out[0], *extra)
    return TokenLogprobs(*_score_hip(logits, targets, temperature, top_k, ignore_index, False)[:4])


# ------------------------------------------------------------------------------------------------
# distillation
# ------------------------------------------------------------------------------------------------
@_on_device
def _distill_hip(logits, ids, logprobs, temperature, bucket, weight, dx, save):
    """(loss, what the backward pass needs).  dx: None, or where the gradient for a loss gradient of 1 a row goes (True: into
    a new tensor); returned in the second place then."""
    x, rows, n1, s0, s1 = _rows(logits)
    V, K, code = logits.shape[-1], ids.shape[-1], _DTYPES[logits.dtype]
    loss = x.new_empty(logits.shape[:-1], dtype=torch.float32)
    if dx is True:
        dx = x.new_empty(logits.shape)
    stp = pkp = wsp = 0
    nseg = _distill_segments(V, code, dx is not None)
    stat = pk = None
    if save or dx is not None and nseg > 0:
        stat = x.new_empty((rows, 8), dtype=torch.float32)
        pk = x.new_empty((rows, K), dtype=torch.float32)
        stp, pkp = stat.data_ptr(), pk.data_ptr()
    if nseg > 1:
        ws = x.new_empty((rows * nseg, 4), dtype=torch.float32)
        wsp = ws.data_ptr()
    H.lib().tok_distill(x.data_ptr(), code, rows, n1, s0, s1, V, temperature, ids.data_ptr(), ids.dtype == torch.int64,
                        logprobs.data_ptr(), 0 if weight is None else weight.data_ptr(), K, bucket, loss.data_ptr(),
                        0 if dx is None else dx.data_ptr(), stp, pkp, wsp, _raw_stream(logits.device.index))
    return loss, (x, stat, pk) if dx is None else dx


@_on_device
def _distill_grad_hip(x, ids, weight, stat, pk, g, temperature, shape):
    # every pointer and stride anew, as in _score_grad_hip
    x, rows, n1, s0, s1 = _rows(x)
    ids, stat, pk = ids.contiguous(), stat.contiguous(), pk.contiguous()
    weight = None if weight is None else weight.contiguous()
    dx = x.new_empty(shape)
    H.lib().tok_distill_grad(x.data_ptr(), _DTYPES[x.dtype], rows, n1, s0, s1, x.shape[-1], temperature, ids.data_ptr(),
                             ids.dtype == torch.int64, H.ptr(weight), ids.shape[-1], g.data_ptr(), stat.data_ptr(),
                             pk.data_ptr(), dx.data_ptr(), _raw_stream(x.device.index))
    return dx


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, temperature, bucket, weight):
        loss, (x, stat, pk) = _distill_hip(logits, ids, logprobs, temperature, bucket, weight, None, True)
        ctx.save_for_backward(x, ids, weight, stat, pk)
        ctx.args = (temperature, logits.shape)
        return loss

    @staticmethod
    @_once
    def backward(ctx, g):
        return _distill_grad_hip(*ctx.saved_tensors, _f32(g), *ctx.args), None, None, None, None, None


def _distill_torch(logits, ids, logprobs, temperature, tail, weight):
    """The loss as torch operations, its K terms in float64."""
    V = logits.shape[-1]
    if weight is not None:
        logits = torch.where((weight == 0).unsqueeze(-1), 0.0, logits)  # not read
    z = logits.double() / temperature
    none = (z == -math.inf).all(-1, keepdim=True)
    lq_all = torch.log_softmax(torch.where(none, 0.0, z), -1)
    there = (ids >= 0) & (ids < V)
    at = torch.where(there, ids, 0).long()
    lq = torch.where(none, -math.inf, lq_all.gather(-1, at))
    t = torch.where(there, logprobs.double(), -math.inf)
    if tail == "drop":
        any_ = (t > -math.inf).any(-1, keepdim=True) | t.isnan().any(-1, keepdim=True)
        t = t - torch.where(any_, torch.logsumexp(torch.where(any_, t, 0.0), -1, keepdim=True), 0.0)
    p = t.exp()
    live = p != 0
    # an id that occurs several times is one token: each of its entries takes the logarithm of their sum
    count = torch.zeros_like(lq_all).scatter_add(-1, at, there.double())
    whole = torch.zeros_like(lq_all).scatter_add(-1, at, p).gather(-1, at)
    t = torch.where(there & (count.gather(-1, at) > 1), whole.log(), t)
    kl = torch.where(live, p * (torch.where(live, t, 0.0) - torch.where(live, lq, 0.0)), 0.0).sum(-1)
    if tail == "bucket":
        # as logarithms: far below the row's maximum the rest's own sum would lose its digits, then itself
        rest = lq_all.masked_fill((count > 0) | none, -math.inf)
        some = ~(rest == -math.inf).all(-1)
        lq0 = torch.logsumexp(torch.where(some.unsqueeze(-1), rest, 0.0), -1)
        p0 = 1 - p.sum(-1)
        on = (p0 > 0) & some & ~(lq0 < MIN_LOG_REST)
        p0 = torch.where(on, p0, 1.0)
        kl = kl + torch.where(on, p0 * (p0.log() - lq0), 0.0)
    loss = kl * (temperature * temperature)
    if weight is not None:
        loss = torch.where(weight != 0, loss * weight.double(), 0.0)
    return loss.float()


def check_distill(logits, teacher_ids, teacher_logprobs, *, temperature=1.0, tail="drop", weight=None) -> float:
    """The checks of :func:`topk_distill_loss` alone: raises as it would, returns the temperature as a float."""
    temperature = _check_logits(logits, temperature)
    _check_teacher(logits, teacher_ids, teacher_logprobs, tail, weight)
    return temperature


def topk_distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      temperature: float = 1.0, tail: str = "drop", weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """KL divergence from a teacher's top tokens to ``softmax(logits / temperature)``, times ``temperature ** 2`` and the row's
    ``weight``: one float32 loss a row (the shape of ``logits`` without its last dimension), not reduced.

    ``teacher_ids`` / ``teacher_logprobs`` ``(..., K)``, 1 <= K <= 256: tokens and their log-probabilities at the same
    temperature, as ``token_logprobs(teacher_logits, temperature=..., top_k=K)`` returns them.  Ids outside ``[0, V)`` are
    absent entries (shorter lists are padded with -1); entries of the same id add up.  ``tail`` says what becomes of the mass
    outside the list: ``"drop"`` renormalises the teacher over its list (a constant added to a row's values changes nothing,
    so logits divided by the temperature will do), ``"bucket"`` compares the remaining mass of both models as one more
    outcome, however small the student's is; it is left out where the student rules the rest out (``-inf``, or finite mask
    values that leave it less than ``exp(-745)``, where 64 bits end).  A row without entries has loss 0 under ``"drop"``.
    Rows of weight 0 are not read; their loss and gradient are 0.  Only ``logits`` have a gradient."""
    temperature = check_distill(logits, teacher_ids, teacher_logprobs, temperature=temperature, tail=tail, weight=weight)
    if not logits.is_cuda:
        return _distill_torch(logits, teacher_ids, teacher_logprobs, temperature, tail, weight)
    _no_tangent(logits, teacher_logprobs, weight)
    ids, lp, weight = teacher_ids.contiguous(), _f32(teacher_logprobs), _f32(weight)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distill.apply(logits, ids, lp, temperature, _TAILS[tail], weight)
    return _distill_hip(logits, ids, lp, temperature, _TAILS[tail], weight, None, False)[0]


def topk_distill_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      temperature: float = 1.0, tail: str = "drop", weight: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The losses of :func:`topk_distill_loss` and the gradient of their sum with respect to ``logits``, in one pass over the
    logits where a row fits a block's registers.  The gradient has the logits' shape and type, is contiguous, and goes to
    ``out`` when given (which must not share memory with any argument).  Nothing is recorded for autograd."""
    temperature = check_distill(logits, teacher_ids, teacher_logprobs, temperature=temperature, tail=tail, weight=weight)
    if out is not None:
        _check_out(out, logits, teacher_ids, teacher_logprobs, weight)
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)      # autograd notices if it had been saved for a backward pass
    logits = logits.detach()
    if not logits.is_cuda:
        with torch.inference_mode(False), torch.enable_grad():      # whatever the caller's mode, autograd works here
            x = logits.clone().requires_grad_(True)
            ids, lp, weight = (t.clone() if t is not None and t.is_inference() else t
                               for t in (teacher_ids, teacher_logprobs, weight))
            loss = _distill_torch(x, ids, lp, temperature, tail, weight)
            dx, = torch.autograd.grad(loss.sum(), x)
        return loss.detach(), dx.contiguous() if out is None else out.copy_(dx)
    ids, lp, weight = teacher_ids.contiguous(), _f32(teacher_logprobs), _f32(weight)
    return _distill_hip(logits, ids, lp, temperature, _TAILS[tail], weight, True if out is None else out, False)
