"""What a model's logits are turned into, as cases to time: log probabilities of given tokens with entropy and top
alternatives, distillation from a teacher's top tokens, their gradients, and the scoring of tokens straight from hidden
states.  Each case has a plain form in elementary torch operations (`own` false) and the package's calls (`own` true)."""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(kind, dtype, rows, vocab, width, **more):
    """kind: the operator.  vocab: columns that are tokens, of `width` in memory (the rest is padding, as a tied table padded to a
    multiple of 16 leaves it).  top: alternatives asked for, or entries of the teacher's list.  scored: the share of
    rows that have a target.  banned: the share of columns at -inf.  uneven: teacher lists cut where their mass is reached.
    hard: the hard-label term in the same pass.  hidden: the length of a hidden state (scores)."""
    case = dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, width=width, top=0, entropy=False, scored=1.0, banned=0.0,
                scale=1.0, tail=False, uneven=False, hard=False, hidden=0, bias=False)
    case.update(more)
    return case


def listed():
    return [
        # One generated token of one request: its log probability, the entropy and 20 alternatives. The smallest call: latency.
        dict(_case("logprobs", "bf16", 1, 30522, 30528, top=20, entropy=True), name="logprobs_token_bf16"),
        # A batch of requests, one token each, over a large vocabulary of odd size (rows not 16-byte aligned), some tokens banned.
        dict(_case("logprobs", "f16", 64, 100003, 100003, top=5, entropy=True, banned=0.01), name="logprobs_batch_f16"),
        # The largest: every token of eight prompts of 1024 tokens over a large vocabulary, 8 alternatives each -- also what makes a teacher's list.
        dict(_case("logprobs", "bf16", 8192, 131072, 131072, top=8, entropy=True), name="logprobs_prompts_bf16"),
        # The loss of masked-token training: 32 sequences of 128 tokens, 15 % of them have a target, fp32 logits.
        dict(_case("logprobs", "f32", 4096, 30522, 30528, scored=0.15), name="logprobs_masked_f32"),
        # Gradient of a training step on whole sequences with an entropy bonus: 8 x 1024 tokens.
        dict(_case("logprobs_grad", "bf16", 8192, 30522, 30528, entropy=True), name="logprobs_grad_bf16"),
        # Gradient of the masked-token loss above: most rows are zeros.
        dict(_case("logprobs_grad", "f32", 4096, 30522, 30528, scored=0.15), name="logprobs_grad_masked_f32"),
        # A student against the teacher's 64 best tokens at temperature 2, 32 sequences of 128 tokens.
        dict(_case("distill", "bf16", 4096, 30522, 30528, top=64, scale=0.5), name="distill_bf16"),
        # A short batch, fp32, lists of uneven length (cut at a mass), what is left of the teacher as one more class.
        dict(_case("distill", "f32", 257, 50021, 50021, top=128, tail=True, uneven=True), name="distill_tail_f32"),
        # Gradient of the usual mixture: the teacher's 64 best at temperature 2 and the hard label, one pass.
        dict(_case("distill_grad", "bf16", 4096, 30522, 30528, top=64, scale=0.5, hard=True), name="distill_grad_bf16"),
        # Gradient with the remainder class over a large odd vocabulary, fp16.
        dict(_case("distill_grad", "f16", 300, 100003, 100003, top=100, tail=True), name="distill_grad_tail_f16"),
        # Scoring 32 sequences of 128 tokens from their BERT-base hidden states over the tied table with the decoder's bias.
        dict(_case("scores", "bf16", 4096, 30522, 30522, hidden=768, bias=True, entropy=True), name="scores_texts_bf16"),
        # Seven candidate tokens scored from BERT-large hidden states: the table is read once.
        dict(_case("scores", "f16", 7, 30522, 30522, hidden=1024), name="scores_few_f16"),
    ]


def _targets(case):
    return int(round(case["rows"] * case["scored"]))


def work(case):
    R, V, W, K, e = case["rows"], case["vocab"], case["width"], case["top"], BYTES[case["dtype"]]
    kind = case["kind"]
    if kind == "scores":
        nbytes = (R + V) * case["hidden"] * e + (4 * V if case["bias"] else 0) + 4 * R + R * (12 + 4 * case["entropy"])
        return {"bytes": nbytes, "flops": 2 * R * V * case["hidden"] + 4 * R * V}
    read = _targets(case) if kind.startswith("logprobs") and not (case["entropy"] or K) else R
    if kind == "logprobs":
        return {"bytes": read * V * e + 4 * R + R * (12 + 4 * case["entropy"] + 8 * K), "flops": read * V * (6 if case["entropy"] else 4)}
    if kind == "logprobs_grad":
        return {"bytes": read * V * e + R * W * e + R * (16 + 8 * case["entropy"]), "flops": read * V * (7 if case["entropy"] else 5)}
    if kind == "distill":
        return {"bytes": R * V * e + 8 * R * K + R * (16 if case["tail"] else 12), "flops": R * V * 4}
    return {"bytes": R * V * e + R * W * e + 8 * R * K + R * (16 + 16 * case["hard"]), "flops": R * V * (9 if case["hard"] else 5)}


# ---- more cases of the same ranges --------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["logprobs"] * 4 + ["logprobs_grad"] * 3 + ["distill"] * 3 + ["distill_grad"] * 3 + ["scores"] * 2)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if kind != "scores" else rng.choice(["bf16", "f16"])
        rows, vocab = _log(rng, 1, 8192), _log(rng, 1000, 131072)
        width = rng.choice([vocab, (vocab + 15) // 16 * 16, (vocab + 127) // 128 * 128])
        more = {}
        if kind.startswith("logprobs"):
            more = dict(entropy=rng.random() < 0.5, scored=rng.choice([1.0, 1.0, 0.15, 0.6]), scale=rng.choice([1.0, 1.0, 1.0 / 0.7]))
            if kind == "logprobs":
                more.update(top=rng.choice([0, 0, 1, 5, 20, rng.randint(1, 128)]), banned=rng.choice([0.0, 0.0, 0.01, 0.5]))
        elif kind.startswith("distill"):
            more = dict(top=_log(rng, 1, 128), scale=rng.choice([1.0, 0.5, 0.25]), tail=rng.random() < 0.4, uneven=rng.random() < 0.4)
            if kind == "distill_grad":
                more["hard"] = rng.random() < 0.5
        else:
            width = vocab
            more = dict(hidden=8 * _log(rng, 16, 256), bias=rng.random() < 0.5, entropy=rng.random() < 0.5, scale=rng.choice([1.0, 1.0, 1.0 / 0.7]))
        case = _case(kind, dtype, rows, vocab, width, **more)
        w = work(case)
        if w["bytes"] <= 2.1e9 and w["flops"] <= 1.9e11 and w["bytes"] + w["flops"] / 100 >= 2e4:
            return case


# ---- what a program has in hand -----------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, g, target):
    """Logits as a language model gives them: a broad spread, and for most rows a clearly raised target."""
    R, V, W = case["rows"], case["vocab"], case["width"]
    x = torch.empty(R, W, device="cuda", dtype=DTYPES[case["dtype"]])
    sure = 8.0 * torch.rand(R, device="cuda", generator=g)
    for r in range(0, R, 1024):
        part = 2.0 * torch.randn(min(1024, R - r), W, device="cuda", generator=g)
        part.scatter_add_(1, target[r:r + 1024, None], sure[r:r + 1024, None])
        if case["banned"]:
            ban = torch.rand(W, device="cuda", generator=g) < case["banned"]
            ban = ban[None, :] & (torch.arange(W, device="cuda")[None, :] != target[r:r + 1024, None])
            part.masked_fill_(ban, -math.inf)
        x[r:r + 1024] = part.to(x.dtype)
    return x


def _with_target(case, g, target):
    """The targets a program holds: -1 where a row has none."""
    given = torch.full_like(target, -1)
    rows = torch.randperm(case["rows"], device="cuda", generator=g)[:_targets(case)]
    given[rows] = target[rows]
    return given.to(torch.int32)


def _softmax_rows(x, vocab, scale):
    """What an earlier forward pass saved for a backward one, in 64 bits: maximum, log of the sum, entropy."""
    m, l, h = [], [], []
    for r in range(0, x.shape[0], 512):
        part = x[r:r + 512, :vocab].double()
        top = part.amax(1)
        z = scale * (part - top[:, None])
        total = z.exp().sum(1)
        m.append(top), l.append(total.log())
        h.append(total.log() - (z.exp() * z).sum(1) / total)
    return torch.stack([torch.cat(m), torch.cat(l)], 1).float(), torch.cat(h).float()


def prepare(case, seed):
    g = _generator(seed)
    R, V, W, K, t = case["rows"], case["vocab"], case["width"], case["top"], DTYPES[case["dtype"]]
    target = torch.randint(0, V, (R,), device="cuda", generator=g)
    s = {"case": case}
    if case["kind"] == "scores":
        hidden = case["hidden"]
        s["x"] = torch.randn(R, hidden, device="cuda", generator=g).to(t)                # behind a LayerNorm
        s["table"] = (2.0 / math.sqrt(hidden) * torch.randn(V, hidden, device="cuda", generator=g)).to(t)
        s["bias"] = 0.5 * torch.randn(V, device="cuda", generator=g) if case["bias"] else None
        s["targets"] = target.to(torch.int32)
        return s
    s["logits"] = _logits(case, g, target)
    if case["kind"].startswith("logprobs"):
        s["targets"] = _with_target(case, g, target)
    else:
        s["ids"], s["teacher"] = _teacher(case, g, s["logits"])
        if case["hard"]:
            s["targets"] = target.to(torch.int32)
    # a mean over the rows; fp16 training scales its loss up, or gradients of unlikely tokens would be lost as subnormals
    weight = torch.rand(R, device="cuda", generator=g) * (1024.0 if case["dtype"] == "f16" else 1.0 / R)
    if case["kind"] == "logprobs_grad":
        s["stats"], s["h"] = _softmax_rows(s["logits"], V, case["scale"])
        if not case["entropy"]:
            s["stats"][s["targets"] < 0] = 0
        s["dlogp"] = -weight
        s["dentropy"] = -0.01 * weight if case["entropy"] else None
    if case["kind"] == "distill_grad":
        s["stats"], _ = _softmax_rows(s["logits"], V, case["scale"])
        if case["tail"]:
            s["stats"] = torch.cat([s["stats"], _rest(s["logits"], V, case["scale"], s["ids"])], 1)
        s["dloss"] = weight
        if case["hard"]:
            s["token_stats"], _ = _softmax_rows(s["logits"], V, 1.0)
            s["dlogp"] = -0.5 * weight
    return s


def _teacher(case, g, logits):
    """The teacher's best tokens and their log probabilities at the temperature: the student's logits seen through noise."""
    V, K = case["vocab"], case["top"]
    ids, logp = [], []
    for r in range(0, logits.shape[0], 512):
        part = logits[r:r + 512, :V].float()
        part = part + 1.0 * torch.randn(part.shape, device="cuda", generator=g)
        lp = torch.log_softmax(case["scale"] * part, 1)
        v, i = lp.topk(K, 1)
        ids.append(i), logp.append(v)
    ids, logp = torch.cat(ids).to(torch.int32), torch.cat(logp).contiguous()
    if case["uneven"]:
        before = logp.exp().cumsum(1) - logp.exp()
        ids = torch.where(before < 0.9 * logp.exp().sum(1, keepdim=True), ids, torch.full_like(ids, -1))
    return ids.contiguous(), logp


def _rest(logits, vocab, scale, ids):
    """Log of the sum over the tokens that the teacher does not list, beside the row's maximum, in 64 bits."""
    out = []
    for r in range(0, logits.shape[0], 512):
        part = logits[r:r + 512, :vocab].double()
        z = scale * (part - part.amax(1, keepdim=True))
        some = ids[r:r + 512].long()
        z = torch.cat([z, z.new_zeros(z.shape[0], 1)], 1)                                # one more column takes the padding
        z.scatter_(1, torch.where(some < 0, torch.full_like(some, vocab), some), -math.inf)
        out.append(z[:, :vocab].exp().sum(1).log()[:, None])
    return torch.cat(out).float()


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    sfb = importlib.import_module("sf-bert_b200")
    case = s["case"]
    kind, V, scale = case["kind"], case["vocab"], case["scale"]
    if kind == "logprobs":
        logp, stats, entropy, top_logp, top_ids, missed = sfb.token_logprobs(s["logits"], s["targets"], vocab=V, scale=scale, entropy=case["entropy"],
                                                                             top_k=case["top"])
        return _named(logp=logp, stats=stats, entropy=entropy, top_logp=top_logp, top_ids=top_ids, missed=missed)
    if kind == "logprobs_grad":
        return sfb.token_logprobs_grad(s["logits"], s["targets"], s["stats"], s["dlogp"], entropy=s["h"] if case["entropy"] else None,
                                       dentropy=s["dentropy"], vocab=V, scale=scale)
    if kind == "distill":
        loss, stats, missed = sfb.distill_topk(s["logits"], s["ids"], s["teacher"], vocab=V, scale=scale, tail=case["tail"])
        return _named(loss=loss, stats=stats, missed=missed)
    if kind == "distill_grad":
        hard = dict(targets=s["targets"], token_stats=s["token_stats"], dlogp=s["dlogp"]) if case["hard"] else {}
        return sfb.distill_topk_grad(s["logits"], s["ids"], s["teacher"], s["stats"], s["dloss"], vocab=V, scale=scale, tail=case["tail"], **hard)
    logp, stats, entropy, missed = sfb.linear_logprobs(s["x"], s["table"], s["targets"], bias=s["bias"], scale=scale, entropy=case["entropy"])
    return _named(logp=logp, stats=stats, entropy=entropy, missed=missed)


def _named(**outputs):
    return {n: t for n, t in outputs.items() if t is not None}


def _plain(s):
    case = s["case"]
    kind, V, scale = case["kind"], case["vocab"], case["scale"]
    if kind == "scores":
        x = s["x"].float() @ s["table"].float().t()
        if s["bias"] is not None:
            x = x + s["bias"]
        return _plain_logprobs(x, s["targets"], scale, case["entropy"], 0)
    x = s["logits"][:, :V].float()
    if kind == "logprobs":
        return _plain_logprobs(x, s["targets"], scale, case["entropy"], case["top"])
    if kind == "distill":
        return _plain_distill(x, s["ids"], s["teacher"], scale, case["tail"])
    if kind == "logprobs_grad":
        d = _plain_logprobs_grad(x, s["targets"], s["stats"], s["dlogp"], s["h"], s["dentropy"], scale)
    else:
        d = _plain_distill_grad(x, s["ids"], s["teacher"], s["stats"], s["dloss"], scale, case["tail"])
        if case["hard"]:
            d += _plain_logprobs_grad(x, s["targets"], s["token_stats"], s["dlogp"], None, None, 1.0)
    out = torch.zeros_like(s["logits"])
    out[:, :V] = d.to(out.dtype)
    return out


def _plain_logprobs(x, targets, scale, entropy, top):
    V = x.shape[1]
    inside = (targets >= 0) & (targets < V)
    best = x.amax(1)
    z = scale * (x - best[:, None])
    e = z.exp()
    total = e.sum(1)
    l = total.log()
    at = torch.where(inside, targets, 0).long()[:, None]
    logp = torch.where(inside, z.gather(1, at)[:, 0] - l, 0.0)
    stats = torch.stack([best, l], 1)
    if not entropy and not top:                                         # rows without a target have nothing to give
        stats = torch.where(inside[:, None], stats, 0.0)
    out = dict(logp=logp, stats=stats, missed=(~inside).sum().to(torch.int32)[None])
    if entropy:
        out["entropy"] = l - torch.where(e > 0, e * z, 0.0).sum(1) / total
    if top:
        # whole-number keys: the value's bits in ascending order, then the lower index first
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits) * V + (V - 1 - torch.arange(V, device=x.device))
        ids = V - 1 - key.topk(top, 1).values % V
        picked = z.gather(1, ids)
        out["top_logp"] = picked - l[:, None]
        out["top_ids"] = torch.where(picked > -math.inf, ids, -1).to(torch.int32)
    return out


def _plain_logprobs_grad(x, targets, stats, dlogp, h, dentropy, scale):
    V = x.shape[1]
    inside = (targets >= 0) & (targets < V)
    g = torch.where(inside, dlogp, 0.0)
    lp = scale * (x - stats[:, :1]) - stats[:, 1:2]
    p = lp.exp()
    if dentropy is None:
        d = -g[:, None] * p
    else:
        d = -p * (g[:, None] + dentropy[:, None] * (torch.where(p > 0, lp, 0.0) + h[:, None]))
    if dentropy is None:
        d = torch.where(inside[:, None], d, 0.0)
    d.scatter_add_(1, torch.where(inside, targets, 0).long()[:, None], g[:, None])
    return scale * d


def _plain_lists(ids, teacher, vocab, tail):
    """Where a list's entries count, their columns (an extra one for those that do not) and the teacher's probabilities."""
    there = (ids >= 0) & (ids < vocab)
    at = torch.where(there, ids, vocab).long()
    lq = torch.where(there, teacher, -math.inf)
    if not tail:
        lq = lq - lq.amax(1, keepdim=True)
        lq = lq - lq.exp().sum(1, keepdim=True).log()
    q = lq.exp()
    rest = (1.0 - q.sum(1)).clamp_min(0.0) if tail else torch.zeros_like(q[:, 0])
    return there, at, torch.where(there, q, 0.0), lq, rest


def _plain_distill(x, ids, teacher, scale, tail):
    R, V = x.shape
    there, at, q, lq, rest = _plain_lists(ids, teacher, V, tail)
    best = x.amax(1)
    z = scale * (x - best[:, None])
    l = z.exp().sum(1).log()
    lp = z.gather(1, at.clamp_max(V - 1)) - l[:, None]
    loss = torch.where(q > 0, q * (lq - lp), 0.0).sum(1)
    stats = [best, l]
    if tail:
        other = torch.ones(R, V + 1, dtype=torch.bool, device=x.device).scatter_(1, at, False)[:, :V]
        lr = torch.where(other, z.exp(), 0.0).sum(1).log()
        loss = loss + torch.where((rest > 0) & (lr > -math.inf), rest * (rest.log() - (lr - l)), 0.0)
        stats.append(lr)
    return dict(loss=loss, stats=torch.stack(stats, 1), missed=(~there).sum().to(torch.int32)[None])


def _plain_distill_grad(x, ids, teacher, stats, dloss, scale, tail):
    R, V = x.shape
    there, at, q, _, rest = _plain_lists(ids, teacher, V, tail)
    p = (scale * (x - stats[:, :1]) - stats[:, 1:2]).exp()
    weight = q.sum(1) + rest
    d = weight[:, None] * p
    if tail:
        other = torch.ones(R, V + 1, dtype=torch.bool, device=x.device).scatter_(1, at, False)[:, :V]
        part = rest[:, None] * (scale * (x - stats[:, :1]) - stats[:, 2:3]).exp()        # the remainder's share of the unlisted tokens
        d = d - torch.where(other & (stats[:, 2:3] > -math.inf), part, 0.0)
    d = torch.cat([d, d.new_zeros(R, 1)], 1).scatter_add_(1, at, -q)[:, :V]
    return (scale * dloss)[:, None] * d


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    parts = []
    for r in range(0, case["rows"], 512):
        parts.append(_exact_rows(case, {n: t[r:r + 512] if torch.is_tensor(t) and n not in ("table", "bias") else t for n, t in s.items()}))
    if torch.is_tensor(parts[0]):
        return torch.cat(parts)
    return {n: sum(p[n] for p in parts) if n == "missed" else torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_rows(case, s):
    V, a, kind = case["vocab"], float(case["scale"]), case["kind"]
    if kind == "scores":
        x = torch.mm(s["x"].double(), s["table"].double().t())
        x = x if s["bias"] is None else x + s["bias"].double()
    else:
        x = s["logits"][:, :V].double()
    R = x.shape[0]
    rows = torch.arange(R, device=x.device)
    logz = torch.logsumexp(a * x, 1)
    if kind in ("logprobs", "scores"):
        t = s["targets"].long()
        hit = (t >= 0) & (t < V)
        peak = x.max(1).values
        out = {"logp": torch.where(hit, a * x[rows, t.clamp(0, V - 1)] - logz, 0.0), "stats": torch.stack([peak, logz - a * peak], 1),
               "missed": (R - hit.sum()).to(torch.int32)[None]}
        if not case["entropy"] and not case["top"]:
            out["stats"][~hit] = 0
        if case["entropy"]:
            lp = a * x - logz[:, None]
            out["entropy"] = -(lp.exp() * lp.clamp_min(-1e300)).sum(1)
        if case["top"]:
            v, i = s["logits"][:, :V].float().sort(dim=1, descending=True, stable=True)
            v, i = v[:, :case["top"]].double(), i[:, :case["top"]]
            out["top_logp"] = a * v - logz[:, None]
            out["top_ids"] = i.masked_fill(v == -math.inf, -1).to(torch.int32)
        return out
    if kind == "logprobs_grad":
        d = _exact_token_grad(case, s, x, a, s["stats"], s["dentropy"])
    else:
        q, q_rest, listed_ = _exact_lists(case, s, V)
        if kind == "distill":
            lp = a * x - logz[:, None]
            use = q > 0
            ids = s["ids"].long().clamp(0, V - 1)
            loss = (torch.where(use, q * (q.clamp_min(1e-300).log() - lp.gather(1, ids)), 0.0)).sum(1)
            peak = x.max(1).values
            stats = [peak, logz - a * peak]
            if case["tail"]:
                lrest = torch.logsumexp((a * x).masked_fill(listed_, -math.inf), 1)
                some = (q_rest > 0) & (lrest > -math.inf)
                loss = loss + torch.where(some, q_rest * (q_rest.clamp_min(1e-300).log() - (lrest - logz)), 0.0)
                stats.append(lrest - a * peak)
            there = (s["ids"] >= 0) & (s["ids"] < V)
            return {"loss": loss, "stats": torch.stack(stats, 1), "missed": (there.numel() - there.sum()).to(torch.int32)[None]}
        st = s["stats"].double()
        z = a * (x - st[:, :1])
        d = (q.sum(1) + q_rest)[:, None] * (z - st[:, 1:2]).exp()
        if case["tail"]:
            d = d - torch.where(listed_, 0.0, q_rest[:, None] * (z - st[:, 2:3]).exp())
        for k in range(q.shape[1]):
            d[rows, s["ids"][:, k].long().clamp(0, V - 1)] -= q[:, k]
        d = d * (a * s["dloss"].double())[:, None]
        if case["hard"]:
            d = d + _exact_token_grad(case, s, x, 1.0, s["token_stats"], None)
    full = torch.zeros(R, case["width"], dtype=torch.float64, device=x.device)
    full[:, :V] = d
    return full


def _exact_token_grad(case, s, x, a, stats, dentropy):
    V = x.shape[1]
    t = s["targets"].long()
    hit = (t >= 0) & (t < V)
    g = torch.where(hit, s["dlogp"].double(), 0.0)
    lp = a * (x - stats[:, :1].double()) - stats[:, 1:2].double()
    p = lp.exp()
    one = torch.zeros_like(p)
    one[hit.nonzero()[:, 0], t[hit]] = 1.0
    d = g[:, None] * (one - p)
    if dentropy is not None:
        d = d - dentropy.double()[:, None] * p * (lp.clamp_min(-1e300) + s["h"].double()[:, None])
    else:
        d[~hit] = 0
    return a * d


def _exact_lists(case, s, V):
    ids, w = s["ids"], s["teacher"].double()
    there = (ids >= 0) & (ids < V)
    w = w.masked_fill(~there, -math.inf)
    listed_ = torch.zeros(ids.shape[0], V, dtype=torch.bool, device=ids.device)
    r, k = there.nonzero(as_tuple=True)
    listed_[r, ids[r, k].long()] = True
    if case["tail"]:
        q = w.exp()
        return q, (1 - q.sum(1)).clamp_min(0), listed_
    return torch.softmax(w, 1), torch.zeros_like(w[:, 0]), listed_
