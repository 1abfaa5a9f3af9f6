"""The operators of a training step around the attention from their definitions, in 64 bits on the CPU, and the tolerances that their
roundings add up to."""
import numpy as np
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    return torch.finfo(t).eps / 2


def attend(q, k, v, keep, scale):
    """q, k, v [B, L, H, d], keep [heads, L, L]: o [B, L, H, d] and the log-sums [B, H, L]."""
    q, k, v = (x.double() for x in (q, k, v))
    x = scale * torch.einsum("blhd,bmhd->bhlm", q, k)
    x = x.masked_fill(~keep[None], -np.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.where(lse[..., None] > -np.inf, (x - lse[..., None]).exp(), 0.0)
    return torch.einsum("bhlm,bmhd->blhd", p, v), lse


def attend_grad(q, k, v, o, do, lse, keep, scale):
    """(dq, dk, dv), and for each the sums of the magnitudes of what it adds up (of the roundings of P and dS to 16 bits an entry's share
    is at most half a step of it)."""
    q, k, v, o, do, lse = (x.double() for x in (q, k, v, o, do, lse))
    x = scale * torch.einsum("blhd,bmhd->bhlm", q, k)
    p = torch.where(keep[None] & (lse > -np.inf)[..., None], (x - lse[..., None]).exp(), 0.0)
    dp = torch.einsum("blhd,bmhd->bhlm", do, v)
    delta = torch.einsum("blhd,blhd->bhl", do, o)
    ds = scale * p * (dp - delta[..., None])
    grads = (torch.einsum("bhlm,bmhd->blhd", ds, k), torch.einsum("bhlm,blhd->bmhd", ds, q), torch.einsum("bhlm,blhd->bmhd", p, do))
    # magnitudes: a rounding of P, or of dP - delta (fp32 sums of d products), is relative to these
    wide = scale * p * (torch.einsum("blhd,bmhd->bhlm", do.abs(), v.abs()) + torch.einsum("blhd,blhd->bhl", do.abs(), o.abs())[..., None])
    sizes = tuple(torch.einsum(e, a, b.abs()) for e, a, b in (("bhlm,bmhd->blhd", ds.abs(), k), ("bhlm,blhd->bmhd", ds.abs(), q), ("bhlm,blhd->bmhd", p, do)))
    loose = tuple(torch.einsum(e, a, b.abs()) for e, a, b in (("bhlm,bmhd->blhd", wide, k), ("bhlm,blhd->bmhd", wide, q), ("bhlm,blhd->bmhd", p, do)))
    return grads, sizes, loose


def grad_tolerance(grads, sizes, loose, dtype, lse, d, terms, scale, qk):
    """What each entry may be off by: half a step of the result; for 16-bit types half a step of P or dS as operands; and in fp32 the
    scores, their exponential and sums.  An error e of a log2-score makes P wrong by e ln 2 of itself: the score's d products are each
    off by a rounding (2^-24) and the tensor cores' additions drop at most a unit of 2^-23 of their largest addend 4 times per 16
    products; the log-sum's rounding is 2^-24 of its size.  qk: the largest sum of magnitudes of a score's products."""
    fin = lse[lse > -np.inf]
    top = float(fin.abs().max()) if fin.numel() else 0.0
    e = 2.0 ** -23 * (scale * qk * (2 + d / 16) + 2 * top + 4) + 2.0 ** -22
    chain = 2.0 ** -23 * (4 + d / 16 + terms / 16)
    h = half_step(dtype)
    out = []
    for g, s, w in zip(grads, sizes, loose):
        t = h * g.abs() + (e + chain) * w + 1e-30
        if dtype != torch.float32:
            t = t + h * s * (1 + h)
            if dtype == torch.float16:                               # entries below 2^-14 are rounded to multiples of 2^-24
                t = t + 2.0 ** -25 * (terms * float(qk_unit(g, dtype)) + 1)
        out.append(t)
    return out


def qk_unit(g, dtype):
    """The largest magnitude of an operand that a subnormal entry of P or dS meets: normal random numbers stay below 6."""
    return 6.0


def blocks_to_elements(blocks, bs):
    return torch.from_numpy(blocks.astype(bool)).repeat_interleave(bs, 1).repeat_interleave(bs, 2)


def pack_bits(keep, blocks, bs):
    """Element masks [heads, kept blocks, bs] of a layout whose heads keep equally many blocks: bit c of word r of a block."""
    heads, nb = blocks.shape[0], blocks.shape[1]
    tiles = keep.view(-1, nb, bs, nb, bs).permute(0, 1, 3, 2, 4)
    if tiles.shape[0] != heads:
        tiles = tiles.expand(heads, -1, -1, -1, -1)
    words = (tiles[torch.from_numpy(blocks.astype(bool))].long() << torch.arange(bs)).sum(-1)
    return words.view(heads, -1, bs).to(torch.int64 if bs == 64 else torch.int32).contiguous()


def embed_grad(dout, ids, vocab, scale):
    """dtable, dpos, and the sums of magnitudes of the first."""
    d = dout.double().view(-1, dout.shape[-1])
    at = ids.flatten().long()
    there = (at >= 0) & (at < vocab)
    table = torch.zeros(vocab, d.shape[1], dtype=torch.float64).index_add_(0, at[there], scale * d[there])
    size = torch.zeros(vocab, d.shape[1], dtype=torch.float64).index_add_(0, at[there], abs(scale) * d[there].abs())
    return table, dout.double().sum(0), size, dout.double().abs().sum(0)
