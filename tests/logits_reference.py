"""The operators on logits in 64 bits, from their definitions, for the GPU tests."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative


def bounds(vocab):
    """Relative error of a row's sum of exponentials: every addition rounds by at most 2^-24 of the running sum, a thread adds
    up to vocab / 64 + 40 terms (64 threads at least, four windows of 8 at a time), a warp, a CTA and a cluster 16 more, and
    each term is within 2^-22 of the power plus 2^-22 of its exponent, which weighted by the term is below 1."""
    return 2.0 ** -24 * (vocab / 64 + 40 + 16 + 8)


def rows64(logits, vocab, scale):
    x = logits.reshape(-1, logits.shape[-1])[:, :vocab].double()
    m = x.amax(1)
    safe = torch.where(m > -math.inf, m, 0.0)
    z = scale * (x - safe[:, None])
    e = z.exp()
    total = e.sum(1)
    return x, m, z, e, total, total.log()


def token_logprobs(logits, targets, vocab, scale, top_k=0):
    x, m, z, e, total, l = rows64(logits, vocab, scale)
    p = e / torch.where(total > 0, total, 1.0)[:, None]
    out = {"m": m, "l": l, "entropy": torch.where(total > 0, l - torch.where(p > 0, p * z, 0.0).sum(1), 0.0), "p": p, "z": z}
    if targets is not None:
        t = targets.reshape(-1).long()
        ok = (t >= 0) & (t < vocab)
        lp = z.gather(1, torch.where(ok, t, 0)[:, None])[:, 0] - torch.where(total > 0, l, 0.0)
        out["logp"] = torch.where(ok, torch.where(m > -math.inf, lp, -math.inf), 0.0)
        out["missed"] = int((~ok).sum())
    if top_k:
        v, i = (x + 0.0).sort(dim=1, descending=True, stable=True)
        v, i = v[:, :top_k], i[:, :top_k]
        there = v > -math.inf
        out["top_ids"] = torch.where(there, i, -1)
        out["top_logp"] = torch.where(there, scale * (v - torch.where(m > -math.inf, m, 0.0)[:, None]) - torch.where(total > 0, l, 0.0)[:, None], -math.inf)
    return out


def token_grad(logits, targets, dlogp, dentropy, vocab, scale):
    """(gradient [rows, vocab], the size of the share of p that each element has, the row's results, the target's share)"""
    r = token_logprobs(logits, targets, vocab, scale)
    p, z = r["p"], r["z"]
    t = targets.reshape(-1).long()
    ok = (t >= 0) & (t < vocab)
    g = torch.where(ok, dlogp.reshape(-1).double(), 0.0)
    one = torch.zeros_like(p)
    one[ok, t[ok]] = 1.0
    d = g[:, None] * (one - p)
    size = g.abs()[:, None] * p
    if dentropy is not None:
        h = dentropy.reshape(-1).double()[:, None]
        lp = torch.where(p > 0, z - torch.where(r["l"] > -math.inf, r["l"], 0.0)[:, None], 0.0)
        d = d - h * p * (lp + r["entropy"][:, None])
        size = size + h.abs() * p * (lp.abs() + r["entropy"][:, None] + 1)
    return scale * d, scale * size, r, scale * g.abs()[:, None] * one


def lists(ids, teacher, vocab, tail):
    ids, w = ids.reshape(-1, ids.shape[-1]).long(), teacher.reshape(-1, ids.shape[-1]).double()
    ok = (ids >= 0) & (ids < vocab)
    w = torch.where(ok, w, -math.inf)
    if tail:
        q = w.exp()
        return ok, ids, q, w, (1 - q.sum(1)).clamp_min(0.0)
    none = w.amax(1) == -math.inf
    lq = torch.log_softmax(torch.where(none[:, None], 0.0, w), 1)
    lq = torch.where(none[:, None] | ~ok, -math.inf, lq)
    return ok, ids, lq.exp(), lq, torch.zeros_like(w[:, 0])


def listed(ok, ids, vocab):
    mask = torch.zeros(ids.shape[0], vocab, dtype=torch.bool, device=ids.device)
    r, k = ok.nonzero(as_tuple=True)
    mask[r, ids[r, k]] = True
    return mask


def distill(logits, ids, teacher, vocab, scale, tail):
    x, m, z, e, total, l = rows64(logits, vocab, scale)
    ok, ids, q, lq, left = lists(ids, teacher, vocab, tail)
    lp = z.gather(1, torch.where(ok, ids, 0)) - l[:, None]
    terms = torch.where(q > 0, q * (lq - lp), 0.0)
    loss, size = terms.sum(1), torch.where(q > 0, q * (lq.abs() + lp.abs() + 1), 0.0).sum(1)
    rest = torch.where(listed(ok, ids, vocab), 0.0, e).sum(1)
    lr = rest.log()
    if tail:
        use = (left > 0) & (rest > 0)
        loss = loss + torch.where(use, left * (left.clamp_min(1e-300).log() - lr + l), 0.0)
        size = size + torch.where(use, left * (left.clamp_min(1e-300).log().abs() + (lr - l).abs() + 1) + 2, 0.0)
    return {"loss": loss, "size": size, "m": m, "l": l, "lr": lr, "missed": int((~ok).sum())}


def distill_grad(logits, ids, teacher, dloss, vocab, scale, tail, targets=None, dlogp=None):
    x, m, z, e, total, l = rows64(logits, vocab, scale)
    ok, ids, q, lq, left = lists(ids, teacher, vocab, tail)
    p = e / torch.where(total > 0, total, 1.0)[:, None]
    weight = (q.sum(1) + left)[:, None]
    d, size = weight * p, weight * p
    if tail:
        mask = listed(ok, ids, vocab)
        rest = torch.where(mask, 0.0, e).sum(1, keepdim=True)
        share = torch.where(mask | (rest == 0), 0.0, e / torch.where(rest > 0, rest, 1.0)) * left[:, None]
        d, size = d - share, size + share
    push = torch.zeros(d.shape[0], vocab + 1, dtype=torch.float64, device=d.device)
    push.scatter_add_(1, torch.where(ok, ids, vocab), torch.where(ok, q, 0.0))
    d, size = d - push[:, :vocab], size + push[:, :vocab]
    w = scale * dloss.reshape(-1).double()[:, None]
    d, size = w * d, w.abs() * size
    if targets is not None:
        h, s, _, share = token_grad(logits, targets, dlogp, None, vocab, 1.0)
        return d + h, size + s, share
    return d, size, torch.zeros_like(d)
