"""Cases of the token operators: log-probabilities of given tokens (with entropy and top alternatives) and the distillation
loss from a teacher's top tokens, each with its gradient.

A case has ``batch`` x ``length`` rows of ``vocab`` logits.  ``op`` says which call a user makes:

* ``score``        -- ``token_logprobs`` without gradients: scoring, and reading a teacher's top tokens;
* ``score_grad``   -- ``token_logprobs`` and its backward pass (likelihood with an entropy bonus);
* ``distill``      -- ``topk_distill_loss`` and its backward pass;
* ``distill_step`` -- ``topk_distill_grad``, the loss and the gradient in one call (a trainer that runs its own backward).
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_IGNORE = -100


def _case(name, op, batch, length, vocab, dtype, top_k, temperature, shifted=False, masked=0, tail="drop", truncated=False):
    return {"name": name, "op": op, "batch": batch, "length": length, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "temperature": temperature, "shifted": shifted, "masked": masked, "tail": tail, "truncated": truncated}


def listed():
    return [
        # one genotype's phenotype: 350 positions of the ribosomal autoencoder's vocabulary, with the next-best tokens
        _case("score_one_genotype", "score", 1, 350, 40, "fp32", 5, 1.0),
        # a training batch of the autoencoder scored
        _case("score_codec_batch", "score", 512, 350, 40, "fp32", 5, 1.0),
        # one token of a generating model with a mid-sized vocabulary: latency
        _case("score_one_token", "score", 1, 1, 32000, "bf16", 20, 0.8),
        # a serving batch with a large, odd vocabulary, some of it masked out
        _case("score_serving_batch", "score", 48, 1, 128001, "bf16", 64, 1.0, masked=513),
        # log-probabilities of long prompts: position t scores token t + 1, so logits and targets are shifted views
        _case("score_prompts", "score", 4, 2048, 32000, "bf16", 0, 1.0, shifted=True),
        # the teacher's side of a distillation: its top tokens over a batch of text
        _case("score_teacher", "score", 2, 1000, 50001, "fp32", 32, 2.0),
        # likelihood with an entropy bonus on the autoencoder's batch
        _case("score_grad_codec", "score_grad", 512, 350, 40, "bf16", 0, 1.0),
        # the same on sequences over a large vocabulary, shifted views
        _case("score_grad_text", "score_grad", 4, 1023, 50001, "fp32", 0, 1.0, shifted=True),
        # an autoencoder learning from another one's eight best tokens at each position
        _case("distill_step_codec", "distill_step", 512, 350, 40, "bf16", 8, 1.0),
        # text distillation, the teacher's remaining mass kept as one bucket
        _case("distill_step_text", "distill_step", 4, 2048, 32000, "bf16", 64, 2.0, tail="bucket"),
        # a short batch in half precision through autograd
        _case("distill_short", "distill", 2, 61, 8193, "fp16", 16, 2.0, tail="bucket", truncated=True),
        # a large vocabulary in fp32 through autograd, teacher lists of different lengths
        _case("distill_wide", "distill", 1, 1000, 100003, "fp32", 32, 1.0, truncated=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["score", "score", "score_grad", "distill", "distill_step"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    vocab = log_int(33, 131072) | rng.choice([0, 1])
    rows = min(log_int(1, 200000), max(1, (1 << 27) // vocab))
    batch = min(rows, rng.choice([1, 2, 5, 16]))
    top_k = min(vocab, log_int(1, 128))
    if op == "score" and rng.random() < 0.3 or op == "score_grad":
        top_k = 0
    return {"op": op, "batch": batch, "length": max(1, rows // batch), "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "temperature": rng.choice([0.7, 1.0, 1.0, 2.0]), "shifted": op.startswith("score") and rng.random() < 0.5,
            "masked": vocab // 9 if rng.random() < 0.3 else 0, "tail": rng.choice(["drop", "bucket"]),
            "truncated": rng.random() < 0.5}


def _logits(g, shape, dtype, masked):
    """Logits of a trained model: a spread of 2.5, one token a row favoured by up to 12, the last ``masked`` tokens ruled out."""
    x = torch.randn(shape, generator=g, device="cuda").mul_(2.5)
    live = shape[-1] - masked
    at = torch.randint(0, live, shape[:-1] + (1,), generator=g, device="cuda")
    x.scatter_add_(-1, at, torch.rand(at.shape, generator=g, device="cuda") * 12)
    if masked:
        x[..., live:] = -math.inf
    return x.to(dtype), at.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, L, V, T = case["batch"], case["length"], case["vocab"], case["temperature"]
    more = 1 if case["shifted"] else 0
    x, best = _logits(g, (B, L + more, V), _TYPES[case["dtype"]], case["masked"])
    st = {"case": case, "logits": x}
    if case["op"].startswith("score"):
        # half the given tokens are the favoured ones, the others any; a tenth of the positions carry no token
        other = torch.randint(0, V - case["masked"], best.shape, generator=g, device="cuda")
        y = torch.where(torch.rand(best.shape, generator=g, device="cuda") < 0.5, best, other)
        if more:
            y = torch.cat([other[:, :1], y[:, :-1]], 1)      # the token that position t - 1 predicts
            y[torch.rand(y.shape, generator=g, device="cuda") < 0.1] = _IGNORE
        st["targets"] = y
        st["g_logprob"] = torch.randn((B, L), generator=g, device="cuda")
        st["g_entropy"] = torch.randn((B, L), generator=g, device="cuda") * 0.01
        return st
    # a teacher that agrees with the student up to noise; its list may end early where little mass is left
    t = x.float() + torch.randn(x.shape, generator=g, device="cuda")
    t = torch.log_softmax(t.div_(T), -1)
    lp, ids = t.topk(case["top_k"], -1)
    del t
    if case["truncated"]:
        ids = torch.where(lp.exp().cumsum(-1) - lp.exp() < 0.9, ids, -1)
    st["ids"], st["teacher"] = ids.contiguous(), lp.contiguous()
    # a weight for each position, none for a tenth of them (padding)
    w = torch.rand((B, L), generator=g, device="cuda")
    st["weight"] = torch.where(w > 0.1, w + 0.5, 0.0)
    return st


def _views(st):
    """The logits and targets that a call is given."""
    x = st["logits"]
    if not st["case"]["shifted"]:
        return x, st.get("targets")
    return x[:, :-1], st["targets"][:, 1:]


def run(st):
    c = st["case"]
    return (_own if own else _plain)(st, c["op"], c["temperature"], c["top_k"], c["tail"])


def _own(st, op, T, k, tail):
    from serann.ops import token_ops as O
    x, y = _views(st)
    if op == "score":
        r = O.token_logprobs(x, y, temperature=T, top_k=k, ignore_index=_IGNORE)
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if k:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if op == "score_grad":
        x = x.detach().requires_grad_(True)
        r = O.token_logprobs(x, y, temperature=T, ignore_index=_IGNORE)
        dx, = torch.autograd.grad([r.logprob, r.entropy], [x], [st["g_logprob"], st["g_entropy"]])
        return {"logprob": r.logprob.detach(), "entropy": r.entropy.detach(), "grad": dx}
    if op == "distill":
        x = x.detach().requires_grad_(True)
        loss = O.topk_distill_loss(x, st["ids"], st["teacher"], temperature=T, tail=tail, weight=st["weight"])
        dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        return {"loss": loss.detach(), "grad": dx}
    loss, dx = O.topk_distill_grad(x, st["ids"], st["teacher"], temperature=T, tail=tail, weight=st["weight"])
    return {"loss": loss, "grad": dx}


# -- plain form: elementary torch operations in fp32, rounded once at the end ----------------------------------------
def _plain(st, op, T, k, tail):
    x, y = _views(st)
    z = x.float() / T
    z = z - z.amax(-1, keepdim=True)
    if not op.startswith("score"):
        return _plain_distill(x, z, st, T, tail)
    # summed in 64 bits: of a row that is nearly sure, 1 + 1e-6 would keep no digits of its small log-probability
    lse = z.exp().sum(-1, keepdim=True, dtype=torch.float64).log().float()
    logq = z - lse
    q = logq.exp()
    live = y != _IGNORE
    at = torch.where(live, y, 0).unsqueeze(-1)
    lp = logq.gather(-1, at).squeeze(-1)
    part = torch.where(q > 0, q * logq, 0.0)
    H = -part.sum(-1)
    out = {"logprob": torch.where(live, lp, 0.0), "entropy": torch.where(live, H, 0.0)}
    if op == "score_grad":
        gl = torch.where(live, st["g_logprob"], 0.0).unsqueeze(-1)
        gh = torch.where(live, st["g_entropy"], 0.0).unsqueeze(-1)
        dz = -gl * q - gh * (part + q * H.unsqueeze(-1))
        dz.scatter_add_(-1, at, gl)
        out["grad"] = (dz / T).to(x.dtype)
    elif k:
        V = x.shape[-1]
        # unique 64-bit keys: the value's bits in their order, then the lowest index first
        bits = (x.float() + 0.0).view(torch.int32).long()
        key = (bits ^ ((bits >> 63) & 0x7FFFFFFF)) * (1 << 32) + (V - 1 - torch.arange(V, device=x.device))
        ids = V - 1 - (key.topk(k, -1).values & 0xFFFFFFFF)
        out["top_ids"] = torch.where(live.unsqueeze(-1), ids, -1)
        out["top_logprobs"] = torch.where(live.unsqueeze(-1), logq.gather(-1, ids), -math.inf)
    return out


def _plain_distill(x, z, st, T, tail):
    # the loss is a small difference of large terms: its logarithms and its few terms a row are taken in 64 bits
    ids, w = st["ids"], st["weight"].unsqueeze(-1)
    V = x.shape[-1]
    e = z.exp()
    S = e.sum(-1, keepdim=True, dtype=torch.float64)
    q = e / S.float()
    there = (ids >= 0) & (ids < V)
    at = torch.where(there, ids, 0)
    t = torch.where(there, st["teacher"], -math.inf).double()
    lq = z.gather(-1, at).double() - S.log()
    if tail == "drop":
        m = t.amax(-1, keepdim=True)
        t = t - torch.where(m > -math.inf, m, 0.0)
        total = t.exp().sum(-1, keepdim=True)
        t = t - torch.where(total > 0, total, 1.0).log()
    p = t.exp()
    kl = torch.where(p > 0, p * (t - lq), 0.0).sum(-1, keepdim=True)
    P = p.sum(-1, keepdim=True)
    dz = q * P.float()
    if tail == "bucket":
        listed_ = torch.zeros(x.shape, device=x.device).scatter_add_(-1, at, there.float()) > 0
        e0 = torch.where(listed_, 0.0, e).sum(-1, keepdim=True, dtype=torch.float64)
        p0 = torch.where(e0 > 0, (1 - P).clamp_min(0.0), 0.0)          # a student without mass there: no bucket
        kl = kl + torch.where(p0 > 0, p0 * (p0.log() - e0.log() + S.log()), 0.0)
        out = torch.where(p0 > 0, p0 / e0 * S, 0.0)
        dz = q * torch.where(listed_, (P + p0).float(), (P + p0 - out).float())
    dz = dz.scatter_add(-1, at, -p.float())
    return {"loss": (kl * w * (T * T)).float().squeeze(-1), "grad": torch.where(w != 0, dz * w * T, 0.0).to(x.dtype)}


# -- the definitions in 64 bits, row blocks at a time -----------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    x, y = _views(st)
    T, k, op = case["temperature"], case["top_k"], case["op"]
    V = x.shape[-1]
    shape = x.shape[:-1]
    x = x.reshape(-1, V)
    parts = []
    step = max(1, (1 << 26) // V)
    for r0 in range(0, x.shape[0], step):
        sl = slice(r0, r0 + step)
        lq = torch.log_softmax(x[sl].double() / T, -1)
        n = torch.arange(lq.shape[0], device=lq.device)
        if op.startswith("score"):
            tok = y.reshape(-1)[sl]
            live = tok != _IGNORE
            lp = lq[n, tok.clamp_min(0)]
            q = lq.exp()
            H = -torch.special.xlogy(q, q).sum(-1)
            part = {"logprob": torch.where(live, lp, 0.0), "entropy": torch.where(live, H, 0.0)}
            if op == "score_grad":
                gl = st["g_logprob"].reshape(-1)[sl].double()[:, None]
                gh = st["g_entropy"].reshape(-1)[sl].double()[:, None]
                hot = torch.zeros_like(q)
                hot[n, tok.clamp_min(0)] = 1
                d = (gl * (hot - q) - gh * (torch.special.xlogy(q, q) + q * H[:, None])) / T
                part["grad"] = d * live[:, None]
            elif k:
                s, i = torch.sort(x[sl].float(), dim=-1, descending=True, stable=True)
                i = i[:, :k]
                part["top_ids"] = torch.where(live[:, None], i, -1)
                part["top_logprobs"] = torch.where(live[:, None], lq.gather(-1, i), -math.inf)
        else:
            ids = st["ids"].reshape(x.shape[0], -1)[sl]
            w = st["weight"].reshape(-1)[sl].double()
            there = (ids >= 0) & (ids < V)
            t = st["teacher"].reshape(x.shape[0], -1)[sl].double().masked_fill(~there, -math.inf)
            # the teacher's distribution over the vocabulary, one column behind it for the bucket
            p = torch.zeros((lq.shape[0], V), dtype=torch.float64, device=lq.device)
            some = there.any(-1, keepdim=True)
            pk = torch.softmax(t.masked_fill(~some, 0.0), -1) * some if case["tail"] == "drop" else t.exp()
            p.scatter_add_(-1, ids.clamp(0, V - 1), pk * there)
            hit = torch.zeros_like(p).scatter_add_(-1, ids.clamp(0, V - 1), there.double()) > 0
            q = lq.exp()
            terms = torch.special.xlogy(p, p) - torch.where(p > 0, p * lq, 0.0)
            kl, d = terms.sum(-1), q * p.sum(-1, keepdim=True) - p
            if case["tail"] == "bucket":
                q0 = (q * ~hit).sum(-1)
                p0 = (1 - p.sum(-1)).clamp_min(0) * (q0 > 0)
                kl = kl + torch.special.xlogy(p0, p0) - torch.special.xlogy(p0, q0)
                d = d + p0[:, None] * q - torch.where(hit, 0.0, q * torch.where(p0 > 0, p0 / q0, 0.0)[:, None])
            part = {"loss": T * T * w * kl, "grad": (T * w)[:, None] * d}
        parts.append(part)
    return {key: torch.cat([p[key] for p in parts]).reshape(shape + parts[0][key].shape[1:]) for key in parts[0]}


def work(case):
    rows, V, k = case["batch"] * case["length"], case["vocab"], case["top_k"]
    size = 4 if case["dtype"] == "fp32" else 2
    logits = rows * V * size
    if case["op"] == "score":
        return {"bytes": logits + rows * (8 + 8 + 12 * k), "flops": 7 * rows * V}
    if case["op"] == "score_grad":
        return {"bytes": 2 * logits + rows * (8 + 8 + 8), "flops": 14 * rows * V}
    return {"bytes": 2 * logits + rows * (8 + 12 * k), "flops": 10 * rows * V}
