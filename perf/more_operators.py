"""The operators of a training step around the attention, as cases to time: block-sparse attention that keeps a log-sum per row
instead of its probabilities, its backward pass that makes them again, the scaled embedding lookup and the gradients of its tables,
and the global norm of a list of gradients with clipping.  Each case has a plain form in elementary torch operations (`own` false) and
the package's calls (`own` true)."""
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _attention(kind, dtype, B, H, L, d, bs, layout, p=(0, 0, 0, 0), **more):
    """kind: "attend" (output and log-sums) or "attend_grad".  layout, p: the block pattern.  causal: earlier positions only (an element
    mask on the diagonal blocks).  valid: positions that are tokens, the rest is padding that nobody attends to (0: all are).
    per_head: a pattern of its own for each head.  packed: q, k, v (and their gradients) are slices of [B, L, 3, H, d] tensors,
    as one projection leaves them."""
    case = dict(kind=kind, dtype=dtype, B=B, H=H, L=L, d=d, bs=bs, layout=layout, p0=p[0], p1=p[1], p2=p[2], p3=p[3], causal=False, valid=0,
                per_head=False, packed=False)
    case.update(more)
    return case


def _table(kind, dtype, B, L, vocab, hidden, **more):
    """kind: "embed" or "embed_grad".  positions: a position table is added (its gradient asked for).  scale: what the token's row
    is multiplied by.  missing: the share of ids that are -1 (padding).  grad: the type of the gradients."""
    case = dict(kind=kind, dtype=dtype, B=B, L=L, vocab=vocab, hidden=hidden, positions=True, scale=1.0, missing=0.0, grad="f32")
    case.update(more)
    return case


def _clip(dtype, layers, hidden, vocab, **more):
    """Gradients of `layers` encoder layers of width `hidden`, an embedding table of `vocab` rows (0: none) beside them.  master: they come
    from a loss that was scaled up and go, unscaled and clipped, into fp32 buffers; otherwise they are clipped in place, and as in
    most steps of a settled run their norm is below the limit.  odd: sizes that are not multiples of anything."""
    case = dict(kind="clip", dtype=dtype, layers=layers, hidden=hidden, vocab=vocab, master=False, odd=False)
    case.update(more)
    return case


def listed():
    return [
        # Forward of a training step over long sequences: BERT-base heads, band plus every 8th column, fp16.
        dict(_attention("attend", "f16", 8, 12, 4096, 64, 64, "stride", (4, 8, 0, 0)), name="attend_stride_f16"),
        # A small causal batch, q, k, v as one projection leaves them, an odd number of blocks, 20 positions of padding.
        dict(_attention("attend", "bf16", 3, 12, 832, 64, 64, "full", causal=True, valid=812, packed=True), name="attend_causal_bf16"),
        # The backward pass of the first case: the largest.
        dict(_attention("attend_grad", "f16", 8, 12, 4096, 64, 64, "stride", (4, 8, 0, 0)), name="attend_grad_stride_f16"),
        # Backward over rows and columns of very different length (global rows and columns, window, random blocks).
        dict(_attention("attend_grad", "bf16", 8, 12, 4096, 64, 64, "bigbird", (1, 1, 1, 3)), name="attend_grad_bigbird_bf16"),
        # Backward of the small causal batch; the gradients go into one packed tensor, as the projection's backward wants them.
        dict(_attention("attend_grad", "bf16", 3, 12, 832, 64, 64, "full", causal=True, valid=812, packed=True), name="attend_grad_causal_bf16"),
        # Backward in fp32 with 32x32 blocks, 128-wide heads and a pattern per head.
        dict(_attention("attend_grad", "f32", 32, 4, 320, 128, 32, "fixed", (5, 0, 0, 0), per_head=True), name="attend_grad_fixed_f32"),
        # The front of a training step: 8 sequences of 4096 tokens, rows times the root of their length, positions added.
        dict(_table("embed", "bf16", 8, 4096, 30522, 768, scale=math.sqrt(768)), name="embed_texts_bf16"),
        # One token of each of 64 requests, a table without positions: the smallest lookup.
        dict(_table("embed", "f16", 64, 1, 30522, 1024, scale=32.0, positions=False), name="embed_tokens_f16"),
        # Gradients of both tables for 8 x 4096 tokens of text (few words are most of it), a tenth padding.
        dict(_table("embed_grad", "bf16", 8, 4096, 30522, 768, scale=math.sqrt(768), missing=0.1), name="embed_grad_texts_bf16"),
        # One short sequence in fp32: nearly all of the table's gradient is zeros.
        dict(_table("embed_grad", "f32", 1, 320, 30522, 768), name="embed_grad_short_f32"),
        # One small layer's gradients in place: the smallest list.
        dict(_clip("f32", 1, 256, 0), name="clip_layer_f32"),
        # BERT-large's gradients from a scaled fp16 loss into fp32 buffers: 24 layers and the table, 386 tensors.
        dict(_clip("f16", 24, 1024, 30522, master=True), name="clip_model_f16"),
    ]


# ---- block patterns and masks ---------------------------------------------------------------------------------------------
def _blocks(case):
    """Which blocks of [heads, nb, nb] are kept, on the host."""
    nb = case["L"] // case["bs"]
    heads = case["H"] if case["per_head"] else 1
    i, j = np.arange(nb)[None, :, None], np.arange(nb)[None, None, :]
    p0, p1, p2, p3 = (case["p%d" % k] for k in range(4))
    h = np.arange(heads)[:, None, None]
    kind = case["layout"]
    if kind == "full":
        keep = np.ones((heads, nb, nb), bool)
    elif kind == "fixed":                                               # its own chunk and one column of every other; which one: by head
        keep = (j // p0 == i // p0) | (j % p0 == (p0 - 1 - h) % p0)
    elif kind == "stride":
        keep = ((j <= i) & (j + p0 > i)) | (j % p1 == 0)
    elif kind == "local":
        keep = (j + p0 >= i) & (j <= i + p1)
    else:                                                               # bigbird: window, global rows and columns, random blocks
        keep = (abs(i - j) <= p0) | (i < p1) | (i + p2 >= nb) | (j < p1) | (j + p2 >= nb)
        keep = keep | (np.random.RandomState(17).rand(1, nb, nb) < p3 / nb)
    keep = np.broadcast_to(keep, (heads, nb, nb)).copy()
    if case["causal"]:
        keep &= j <= i
    if case["valid"]:
        some = -(-case["valid"] // case["bs"])
        keep[:, some:] = False
        keep[:, :, some:] = False
    return keep


def _elements(case, blocks):
    """Kept elements [heads, L, L] on the GPU."""
    bs, L = case["bs"], case["L"]
    keep = torch.from_numpy(blocks).cuda().repeat_interleave(bs, 1).repeat_interleave(bs, 2)
    at = torch.arange(L, device="cuda")
    if case["causal"]:
        keep &= at[:, None] >= at[None, :]
    if case["valid"]:
        keep &= (at[:, None] < case["valid"]) & (at[None, :] < case["valid"])
    return keep


def _masked(case):
    return bool(case["causal"] or case["valid"])


def _plan(case, blocks, keep):
    """The package's layout with its tables, and the element mask as bits, block by block in the order of its block ids."""
    sfb = importlib.import_module("sf-bert_b200")
    lay = sfb.BlockLayout(torch.from_numpy(blocks.astype(np.uint8)).cuda(), case["bs"])
    lay.tn_lut
    if _masked(case):
        bs, nb = case["bs"], case["L"] // case["bs"]
        tiles = keep.view(-1, nb, bs, nb, bs).permute(0, 1, 3, 2, 4)[torch.from_numpy(blocks).cuda()]
        words = (tiles.long() << torch.arange(bs, device="cuda")).sum(-1)
        lay.mask_np = words.view(keep.shape[0], -1, bs).to(torch.int64 if bs == 64 else torch.int32).contiguous()
    return lay


# ---- what a case costs ------------------------------------------------------------------------------------------------------
def _shapes(case):
    """The gradients of a list: sizes as a model has them."""
    h, o = case["hidden"], 1 if case["odd"] else 0
    layer = [(h, h + o), (h + o,)] * 4 + [(h, 4 * h + o), (4 * h + o,), (4 * h + o, h), (h,)] + [(h + o,)] * 4
    return layer * case["layers"] + ([(case["vocab"], h), (512 + o, h)] if case["vocab"] else [])


def _chances(vocab):
    """How often a token comes up in text, by rank."""
    p = 1.0 / (np.arange(vocab) + 2.7)
    return p / p.sum()


def work(case):
    e = BYTES[case["dtype"]]
    kind = case["kind"]
    if kind in ("attend", "attend_grad"):
        rows = case["B"] * case["L"] * case["H"]
        kept = int(_blocks(case).sum()) * case["B"] * (1 if case["per_head"] else case["H"])
        product = 2 * case["bs"] ** 2 * case["d"] * kept
        if kind == "attend":
            return {"bytes": rows * (4 * case["d"] * e + 4), "flops": 2 * product}
        return {"bytes": rows * (8 * case["d"] * e + 4), "flops": 5 * product}
    if kind == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": n * (e + (4 if case["master"] else 0)), "flops": n * (3 if case["master"] else 2)}
    n, h = case["B"] * case["L"], case["hidden"]
    if kind == "embed":
        p = _chances(case["vocab"])
        rows = float(-np.expm1(n * (1 - case["missing"]) * np.log1p(-p)).sum())           # different tokens among them
        return {"bytes": int((n + rows) * h * e) + 4 * n + (case["L"] * h * e if case["positions"] else 0), "flops": 2 * n * h}
    g = BYTES[case["grad"]]
    return {"bytes": n * h * e + 4 * n + (case["vocab"] + (case["L"] if case["positions"] else 0)) * h * g,
            "flops": n * h * (2 if case["positions"] else 1)}


# ---- more cases of the same ranges --------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["attend"] * 2 + ["attend_grad"] * 4 + ["embed"] * 2 + ["embed_grad"] * 3 + ["clip"] * 2)
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    if kind == "clip":
        return _clip(dtype, rng.choice([0, 1, 2, _log(rng, 1, 24)]), 8 * _log(rng, 4, 160), rng.choice([0, _log(rng, 100, 40000)]),
                     master=rng.random() < 0.5, odd=rng.random() < 0.4)
    if kind in ("embed", "embed_grad"):
        L = _log(rng, 1, 4096)
        return _table(kind, dtype, _log(rng, 1, 128), L, _log(rng, 50, 131072), 8 * _log(rng, 2, 256), positions=rng.random() < 0.6,
                      scale=rng.choice([1.0, 0.5, 27.7]), missing=rng.choice([0.0, 0.0, 0.1, 0.7]), grad=rng.choice(["f32", "f32", dtype]))
    H = _log(rng, 1, 16)
    bs, d = (64, 64) if dtype != "f32" and rng.random() < 0.75 else (rng.choice([32, 32, 64]), rng.choice([32, 64, 128, 8 * rng.randint(1, 16)]))
    nb = _log(rng, 1, 64)
    layout = rng.choice(["full", "stride", "stride", "local", "local", "bigbird", "fixed"])
    p = {"full": (0, 0, 0, 0), "stride": (rng.randint(1, 8), rng.randint(4, 16), 0, 0), "local": (rng.randint(0, 10), rng.randint(0, 10), 0, 0),
         "bigbird": (rng.randint(0, 2), 1, 1, 3), "fixed": (1, 0, 0, 0)}[layout]
    per_head = False
    if layout == "fixed":
        p = (rng.choice([s for s in range(1, 17) if nb % s == 0]), 0, 0, 0)
        per_head = rng.random() < 0.5
    causal = not per_head and rng.random() < 0.4                        # the heads of a layout keep equally many blocks
    valid = rng.randint(1, nb * bs) if not per_head and rng.random() < 0.3 else 0
    return _attention(kind, dtype, _log(rng, 1, 16), H, nb * bs, d, bs, layout, p, causal=causal, valid=valid, per_head=per_head,
                      packed=rng.random() < 0.4)


def draw(rng):
    while True:
        case = _drawn(rng)
        if case["kind"] == "clip" and not _shapes(case):
            continue
        w = work(case)
        most = 1.8e11
        if case["kind"] in ("attend", "attend_grad") and (case["dtype"] == "f32" or case["bs"] != 64 or case["d"] != 64):
            most = 1.5e10
        if w["flops"] <= most and 1e4 <= w["bytes"] <= 1.9e9:
            return case


# ---- what a program has in hand -------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_attention(case, seed):
    g = _generator(seed)
    B, H, L, d, t = case["B"], case["H"], case["L"], case["d"], DTYPES[case["dtype"]]
    blocks = _blocks(case)
    keep = _elements(case, blocks)
    s = {"case": case, "scale": 1.0 / math.sqrt(d), "keep": keep}
    qkv = torch.randn(B, L, 3, H, d, device="cuda", generator=g).to(t)
    s["qkv"] = [qkv[:, :, i] if case["packed"] else qkv[:, :, i].contiguous() for i in range(3)]
    if case["kind"] == "attend_grad":
        # a mean over the tokens; fp16 training scales its loss up
        s["do"] = torch.randn(B, L, H, d, device="cuda", generator=g).to(t)
        o, lse = [], []
        for b in range(B):
            y, l = _exact_attend(*(x[b] for x in s["qkv"]), keep, s["scale"])
            o.append(y), lse.append(l)
        s["o"], s["lse"] = torch.stack(o).to(t), torch.stack(lse).float()
        if case["packed"]:
            into = torch.empty(B, L, 3, H, d, device="cuda", dtype=t)
            s["into"] = [into[:, :, i] for i in range(3)]
        else:
            s["into"] = None
    if own:
        s["lay"] = _plan(case, blocks, keep)
    return s


def _prepare_table(case, seed):
    g = _generator(seed)
    B, L, vocab, h, t = case["B"], case["L"], case["vocab"], case["hidden"], DTYPES[case["dtype"]]
    word = torch.randperm(vocab, device="cuda", generator=g)             # which token has which rank
    below = torch.from_numpy(_chances(vocab).cumsum()).cuda()
    rank = torch.searchsorted(below, torch.rand(B * L, device="cuda", dtype=torch.float64, generator=g)).clamp_max(vocab - 1)
    ids = word[rank].view(B, L)
    if case["missing"]:
        ids = torch.where(torch.rand(B, L, device="cuda", generator=g) < case["missing"], torch.full_like(ids, -1), ids)
    s = {"case": case, "ids": ids.to(torch.int32)}
    if case["kind"] == "embed":
        s["table"] = (torch.randn(vocab, h, device="cuda", generator=g) / math.sqrt(h)).to(t)
        s["pos"] = (0.02 * torch.randn(L, h, device="cuda", generator=g)).to(t) if case["positions"] else None
    else:
        s["dout"] = torch.randn(B, L, h, device="cuda", generator=g).to(t)
    return s


def _prepare_clip(case, seed):
    g = _generator(seed)
    t = DTYPES[case["dtype"]]
    up = 1024.0 if case["master"] else 1.0
    shapes = _shapes(case)
    n = sum(math.prod(x) for x in shapes)
    flat = torch.empty(n, device="cuda", dtype=t)                        # one buffer that the parameters' gradients are views of
    grads = _views(flat, shapes)
    for x in grads:
        x.copy_(up * 1e-3 * torch.randn(x.shape, device="cuda", generator=g))
    s = {"case": case, "grads": grads, "scale": 1.0 / up, "limit": 1e-3 * math.sqrt(n) * (0.25 if case["master"] else 1.5)}
    s["flat"] = torch.empty(n, device="cuda") if case["master"] else flat
    s["into"] = _views(s["flat"], shapes) if case["master"] else None
    return s


def _views(flat, shapes):
    return [x.view(s) for x, s in zip(flat.split([math.prod(s) for s in shapes]), shapes)]


def prepare(case, seed):
    if case["kind"] == "clip":
        return _prepare_clip(case, seed)
    return _prepare_table(case, seed) if case["kind"] in ("embed", "embed_grad") else _prepare_attention(case, seed)


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    sfb = importlib.import_module("sf-bert_b200")
    case = s["case"]
    kind = case["kind"]
    if kind == "attend":
        o, lse = sfb.fused_attention_stats(*s["qkv"], s["lay"], s["scale"], use_mask=_masked(case))
        return {"o": o, "lse": lse}
    if kind == "attend_grad":
        dq, dk, dv = sfb.attention_backward_recompute(*s["qkv"], s["o"], s["do"], s["lse"], s["lay"], s["scale"], use_mask=_masked(case),
                                                      out=s["into"])
        return {"dq": dq, "dk": dk, "dv": dv}
    if kind == "embed":
        out, bad = sfb.embedding(s["table"], s["ids"], s["pos"], scale=case["scale"])
        return {"out": out, "bad": bad}
    if kind == "embed_grad":
        dtable, dpos, bad = sfb.embedding_grad(s["dout"], s["ids"], case["vocab"], scale=case["scale"], positions=case["positions"],
                                               dtype=DTYPES[case["grad"]])
        return {"dtable": dtable, "dpos": dpos, "bad": bad} if case["positions"] else {"dtable": dtable, "bad": bad}
    norm = sfb.clip_grad_norm(s["grads"], s["limit"], scale=s["scale"], out=s["into"])
    return {"norm": norm, "grads": s["flat"]}


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "attend":
        parts = [_plain_attend(*(x[b].float() for x in s["qkv"]), s["keep"], s["scale"])[:2] for b in range(case["B"])]
        return {"o": torch.stack([p[0] for p in parts]).to(s["qkv"][0].dtype), "lse": torch.stack([p[1] for p in parts])}
    if kind == "attend_grad":
        t = s["do"].dtype
        parts = [_plain_attend_grad(*(x[b].float() for x in s["qkv"]), s["o"][b].float(), s["do"][b].float(), s["lse"][b], s["keep"], s["scale"])
                 for b in range(case["B"])]
        return {n: torch.stack([p[i] for p in parts]).to(t) for i, n in enumerate(("dq", "dk", "dv"))}
    if kind == "embed":
        table, ids = s["table"], s["ids"]
        inside = (ids >= 0) & (ids < table.shape[0])
        rows = table[torch.where(inside, ids, 0).long()].float() * case["scale"]
        out = torch.where(inside[..., None], rows, 0.0)
        if s["pos"] is not None:
            out = out + s["pos"].float()
        return {"out": out.to(table.dtype), "bad": (~inside).sum().to(torch.int32)[None]}
    if kind == "embed_grad":
        return _plain_embed_grad(s)
    total = torch.zeros(1, dtype=torch.float64, device="cuda")
    for x in s["grads"]:
        x = x.float() * s["scale"]
        total += (x * x).sum(dtype=torch.float64)
    norm = total.sqrt().float()
    factor = s["scale"] * (s["limit"] / (norm + 1e-6)).clamp_max(1.0)
    into = s["into"] or s["grads"]
    for x, y in zip(s["grads"], into):
        y.copy_(x.float() * factor)
    return {"norm": norm, "grads": s["flat"]}


def _scores(q, k, keep, scale):
    """[H, L, L], what is not kept at -inf."""
    x = scale * (q.transpose(0, 1) @ k.permute(1, 2, 0))
    return x.masked_fill_(~keep, -math.inf)


def _plain_attend(q, k, v, keep, scale):
    x = _scores(q, k, keep, scale)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    o = (e @ v.transpose(0, 1)) / torch.where(total > 0, total, 1.0)
    return o.transpose(0, 1), (top + total.log())[..., 0]


def _plain_attend_grad(q, k, v, o, do, lse, keep, scale):
    p = (_scores(q, k, keep, scale) - torch.where(lse > -math.inf, lse, 0.0)[..., None]).exp()
    qh, kh, vh, doh = (x.transpose(0, 1) for x in (q, k, v, do))
    ds = p * (doh @ vh.transpose(1, 2) - (do * o).sum(-1).t()[..., None]) * scale
    return (ds @ kh).transpose(0, 1), (ds.transpose(1, 2) @ qh).transpose(0, 1), (p.transpose(1, 2) @ doh).transpose(0, 1)


def _plain_embed_grad(s):
    case, dout, ids = s["case"], s["dout"], s["ids"]
    t = DTYPES[case["grad"]]
    inside = (ids >= 0) & (ids < case["vocab"])
    at = torch.where(inside, ids, case["vocab"]).long().flatten()
    sums = torch.zeros(case["vocab"] + 1, case["hidden"], device="cuda")
    sums.index_add_(0, at, dout.float().view(-1, case["hidden"]))
    out = {"dtable": (case["scale"] * sums[:-1]).to(t), "bad": (~inside).sum().to(torch.int32)[None]}
    if case["positions"]:
        out["dpos"] = dout.float().sum(0).to(t)
    return out


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_attend(q, k, v, keep, scale):
    """One batch element, head by head: o [L, H, d] and the log-sums [H, L]."""
    o, lse = [], []
    for h in range(q.shape[1]):
        x = scale * torch.mm(q[:, h].double(), k[:, h].double().t())
        x = x.masked_fill(~keep[h if keep.shape[0] > 1 else 0], -math.inf)
        l = torch.logsumexp(x, 1)
        p = torch.where(l[:, None] > -math.inf, (x - l[:, None]).exp(), 0.0)
        o.append(torch.mm(p, v[:, h].double()))
        lse.append(l)
    return torch.stack(o, 1), torch.stack(lse)


def _exact_attend_grad(q, k, v, o, do, lse, keep, scale):
    dq, dk, dv = [], [], []
    for h in range(q.shape[1]):
        qd, kd, vd, od, dod = (x[:, h].double() for x in (q, k, v, o, do))
        l = lse[h].double()
        p = torch.exp(scale * torch.mm(qd, kd.t()) - torch.where(l > -math.inf, l, 0.0)[:, None])
        p = torch.where(keep[h if keep.shape[0] > 1 else 0], p, 0.0)
        ds = scale * p * (torch.mm(dod, vd.t()) - (dod * od).sum(1)[:, None])
        dq.append(torch.mm(ds, kd)), dk.append(torch.mm(ds.t(), qd)), dv.append(torch.mm(p.t(), dod))
    return torch.stack(dq, 1), torch.stack(dk, 1), torch.stack(dv, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        parts = [_exact_attend(*(x[b] for x in s["qkv"]), s["keep"], s["scale"]) for b in range(case["B"])]
        return {"o": torch.stack([p[0] for p in parts]), "lse": torch.stack([p[1] for p in parts])}
    if kind == "attend_grad":
        parts = [_exact_attend_grad(*(x[b] for x in s["qkv"]), s["o"][b], s["do"][b], s["lse"][b], s["keep"], s["scale"])
                 for b in range(case["B"])]
        return {n: torch.stack([p[i] for p in parts]) for i, n in enumerate(("dq", "dk", "dv"))}
    if kind == "clip":
        norm = math.sqrt(sum(float(x.double().square().sum()) for x in s["grads"])) * s["scale"]
        factor = s["scale"] * min(1.0, s["limit"] / (norm + 1e-6))
        return {"norm": torch.tensor([norm], dtype=torch.float64, device="cuda"),
                "grads": torch.cat([x.double().flatten() for x in s["grads"]]) * factor}
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < case["vocab"])
    bad = (ids.numel() - there.sum()).to(torch.int32)[None]
    if kind == "embed":
        out = case["scale"] * s["table"].double()[ids.clamp(0, case["vocab"] - 1)]
        out[~there] = 0
        return {"out": out if s["pos"] is None else out + s["pos"].double(), "bad": bad}
    dout = s["dout"].double()
    dtable = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device="cuda")
    dtable.index_put_((ids[there],), case["scale"] * dout[there], accumulate=True)
    out = {"dtable": dtable, "bad": bad}
    if case["positions"]:
        out["dpos"] = dout.sum(0)
    return out
