"""Definitions of the token operators in 64 bits on the CPU, row by row, and the error bounds that their fp32 forms are held to."""
import math

import torch

U = 2.0 ** -24          # unit rounding of fp32


def log_q(x, T):
    """(rows, V) float64 log-softmax of x / T; rows of nothing but -inf stay -inf."""
    z = x.double() / T
    none = (z == -math.inf).all(-1, keepdim=True)
    return torch.where(none, -math.inf, torch.log_softmax(z.masked_fill(none, 0.0), -1)), none.squeeze(-1)


def score(x, y, T, k, ignore, g_lp=None, g_h=None):
    """logprob, entropy, top ids, top log-probabilities and dx of rows x (R, V), y (R,) or None."""
    V = x.shape[-1]
    lq, none = log_q(x, T)
    q = lq.exp()
    h = -torch.where(q > 0, q * lq, q * 0).sum(-1)
    h[none] = 0
    nan = lq.isnan().any(-1)
    h[nan] = math.nan
    out = {"entropy": h}
    skip = torch.zeros(x.shape[0], dtype=torch.bool)
    hot = torch.zeros_like(lq)
    if y is not None:
        skip = y == ignore
        ok = (y >= 0) & (y < V)
        at = torch.where(ok, y, 0).long()
        lp = lq.gather(-1, at[:, None])[:, 0]
        lp[~ok] = math.nan
        lp[skip] = 0
        h[skip] = 0
        out["logprob"] = lp
        hot[torch.arange(len(at)), at] = 1
    if k:
        ids = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :k]
        top = lq.gather(-1, ids)
        ids, top = ids.clone(), top.clone()
        ids[nan | skip] = -1
        top[nan] = math.nan
        top[skip] = -math.inf
        out["top_ids"], out["top_logprobs"] = ids, top
    if g_lp is not None or g_h is not None:
        gl = torch.zeros(x.shape[0]).double() if g_lp is None or y is None else g_lp.double()
        gh = torch.zeros(x.shape[0]).double() if g_h is None else g_h.double()
        ent_part = torch.where(q > 0, q * lq, 0.0) + q * torch.nan_to_num(h)[:, None]
        dx = (gl[:, None] * (hot - q) - gh[:, None] * ent_part) / T
        dx[skip | none] = 0
        if y is not None and g_lp is not None:
            dx[~ok & ~skip] = math.nan
        dx[nan & ~skip] = math.nan
        out["grad"] = dx
    return out


def distill(x, ids, t, T, tail, w):
    """Row losses and the gradient of their sum."""
    R, V = x.shape
    lq, none = log_q(x, T)
    q = lq.exp()
    loss, dx = torch.zeros(R).double(), torch.zeros(R, V).double()
    for r in range(R):
        wr = 1.0 if w is None else float(w[r])
        if wr == 0:
            continue
        entries = [(int(i), float(v)) for i, v in zip(ids[r], t[r]) if 0 <= int(i) < V]
        p = torch.zeros(V).double()
        kl = 0.0
        if tail == "drop":
            top = max([v for _, v in entries], default=-math.inf)
            tot = sum(math.exp(v - top) for _, v in entries) if top > -math.inf else 0.0
            entries = [(i, v - top - math.log(tot) if tot > 0 else -math.inf) for i, v in entries]
        for i, v in entries:
            p[i] += math.exp(v)
        parts = [i for i, _ in entries]
        for i, v in sorted(dict(reversed(entries)).items(), key=lambda e: parts.index(e[0])):
            pi = float(p[i])                          # entries of one id are one token
            if pi > 0:
                kl += pi * ((v if parts.count(i) == 1 else math.log(pi)) - float(lq[r, i]))
        P = float(p.sum())
        A = B = P
        if tail == "bucket":
            hit = torch.zeros(V, dtype=torch.bool)
            hit[[i for i, _ in entries]] = True
            q0 = float(q[r][~hit].sum()) if not none[r] else 0.0
            p0 = max(0.0, 1 - P) if q0 > 0 else 0.0
            if p0 > 0:
                # of a rest that is nearly everything, 1 - (listed) keeps the digits of its logarithm
                lq0 = math.log1p(-float(q[r][hit].sum())) if q0 > 0.5 else math.log(q0)
                kl += p0 * (math.log(p0) - lq0)
                A, B = P + p0, P + p0 - p0 / q0
            d = torch.where(hit, A * q[r] - p, B * q[r])
        else:
            d = P * q[r] - p
        loss[r] = wr * T * T * kl
        if not none[r]:
            dx[r] = wr * T * d
    return loss, dx


def sum_error(x, T):
    """Bound of the relative error of sum exp(z - max) as the kernels take it, a number a row.

    An exponent d = fma(x, c, -mc) is rounded once (|d| U) and c = log2(e) / T once (|d| U again); exp2 is off by an ulp (2 U).
    A relative error a |d| + 2 U of exp2(d) is weighted by exp2(d): |d| counts as its average under softmax, at most
    log2(V) + 2 (the entropy bound in bits, plus the bits of the remainder).  A thread adds at most 129 terms in sequence, the
    tree over lanes, waves and segments adds 6 + 2 + 64 more; the reference to the maximum is corrected by one product (2 U)."""
    V = x.shape[-1]
    return U * (2 * 0.7 * (math.log2(max(V, 2)) + 2) + 2 + 129 + 72 + 2)


def half_ulp(t, dtype):
    """Half a step of the output type at the values t, subnormals' step included."""
    fi = torch.finfo(dtype)
    return fi.eps / 2 * t.abs().double() + fi.smallest_normal * fi.eps / 2
