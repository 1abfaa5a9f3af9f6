"""GPU tests of the operators on logits where their arithmetic or their order could go wrong: against 64 bits, within derived bounds."""
import math

import pytest

torch = pytest.importorskip("torch")
import logits_reference as R  # noqa: E402
import test_gpu_logits as G  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(rows, width, dtype, seed, spread=2.5):
    return (spread * torch.randn(rows, width, device="cuda", generator=gen(seed))).to(TYPES[dtype])


# ---- alternatives whose rows are shared by several CTAs ---------------------------------------------------------------------
@pytest.mark.parametrize("rows,vocab,k", [(1, 9000, 20), (1, 30522, 5), (7, 16500, 1), (64, 100003, 5), (40, 131072, 40)])
def test_shared_rows_one_after_another(sfb, rows, vocab, k):
    """Calls that follow each other without a pause, each on logits of its own: every one finds its row's alternatives, ties by the
    lowest index, whichever of the row's CTAs starts or ends first."""
    xs = [make(rows, vocab, "bf16", n) for n in range(4)]
    want = [R.token_logprobs(x, None, vocab, 1.0, k) for x in xs]
    got = [sfb.token_logprobs(xs[n % 4], top_k=k) for n in range(200)]
    for n, g in enumerate(got):
        assert torch.equal(g[4].long(), want[n % 4]["top_ids"]), n
        assert torch.equal(g[3], got[n % 4][3]), n


# ---- distillation whose remainder is far below the row's largest logit -------------------------------------------------------
def divergence(x, ids, teacher, vocab, scale, tail):
    """The loss of each row in 64 bits from its definition, as something to differentiate: x double [rows, >= vocab].  Sums stand beside their
    largest logit: the logarithm of a sum, which a logit of -3.4e38 would swallow, is a value by itself."""
    x = x[:, :vocab]

    def beside_largest(x):
        top = x.detach().amax(1)
        return top, torch.where(x > -INF, scale * (x - top[:, None]), -INF)
    ids, w = ids.long(), teacher.double()
    ok = (ids >= 0) & (ids < vocab)
    w = torch.where(ok, w, -INF)
    lq = w if tail else torch.log_softmax(w, 1)
    q = lq.exp()
    m, z = beside_largest(x)
    l = z.exp().sum(1).log()
    lp = z.gather(1, torch.where(ok, ids, 0)) - l[:, None]
    loss = torch.where(q > 0, q * (torch.where(q > 0, lq, 0.0) - lp), 0.0).sum(1)
    out = {"q": q, "ok": ok, "m": m, "l": l.detach(), "lp": lp.detach(), "z": z.detach()}
    if tail:
        there = torch.zeros(x.shape[0], vocab + 1, dtype=torch.bool, device=x.device).scatter_(1, torch.where(ok, ids, vocab), True)[:, :vocab]
        left = (1 - q.sum(1)).clamp_min(0.0)
        some = (~there & (x > -INF)).any(1) & (left > 0)
        mu, zu = beside_largest(torch.where(some[:, None], x.masked_fill(there, -INF), torch.zeros_like(x)))
        lu = zu.exp().sum(1).log()
        lr = torch.where(some, scale * (mu - m) + lu, -INF)
        loss = loss + torch.where(some, left * (left.clamp_min(1e-300).log() - lr + l), 0.0)
        out.update(left=torch.where(some, left, 0.0), lr=lr.detach(), there=there, some=some, log_share=(zu - lu[:, None]).detach())
    return loss, out


def check_remainder(sfb, x, ids, teacher, vocab, scale, hard=False, seed=3):
    """Loss, statistics and gradient of lists with the remainder.  With u = 2^-24: the teacher's q, a power each and sums of them in
    at most 14 additions, are off by 2^-20, and so is what they leave, q_r; the loss gets that much of log p_r, and 2^-22 of each of its
    terms, and D for either sum (bounds).  A token's p is off by 2^-22 of its exponent, by D, and by what the sum's logarithm is;
    an unlisted token's share of the remainder by 2^-22 of the base-2 exponent it is made from: the distance to the largest unlisted token, and
    where the remainder's logarithm is at least -64, the distances of both to the row's largest.  Then a rounding to the type."""
    rows = x.shape[0]
    dtype = {v: k for k, v in TYPES.items()}[x.dtype]
    loss, stats, missed = sfb.distill_topk(x, ids, teacher, vocab=vocab, scale=scale, tail=True)
    y = x.double().requires_grad_(True)
    want, more = divergence(y, ids, teacher, vocab, scale, True)
    d = R.bounds(vocab)
    l, lr, lp = more["l"], more["lr"], more["lp"]
    q, left = more["q"], more["left"]
    size = torch.where(q > 0, q * (lp.abs() + 20), 0.0).sum(1) + torch.where(left > 0, left * (lr.abs() + l + 20), 0.0)
    lim = (d + 2.0 ** -20) * (1 + size) + 2.0 ** -20 * torch.where(left > 0, lr.abs(), 0.0)
    assert bool(loss.isfinite().all()) and int(missed) == int((~more["ok"]).sum())
    assert bool(((loss.double() - want.detach()).abs() <= lim).all()), float(((loss.double() - want.detach()).abs() / lim).max())
    assert bool(((stats[:, 1].double() - l).abs() <= d + 2.0 ** -22 * l).all())
    some = more["some"]
    assert bool(((stats[:, 2].double() - lr)[some].abs() <= d + 2.0 ** -22 * lr[some].abs()).all())

    g = torch.randn(rows, device="cuda", generator=gen(seed))
    total, args = (g.double() * want).sum(), {}
    if hard:
        t = torch.randint(-1, vocab, (rows,), device="cuda", generator=gen(seed + 1), dtype=torch.int32)
        t[0] = ids[0, 0]
        b = torch.randn(rows, device="cuda", generator=gen(seed + 2))
        _, ts, _, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab, entropy=True)
        args = dict(targets=t, token_stats=ts, dlogp=b)
        lp1 = torch.log_softmax(y[:, :vocab], 1)
        total = total + torch.where(t >= 0, b.double() * lp1.gather(1, t.clamp_min(0).long()[:, None])[:, 0], 0.0).sum()
    total.backward()
    dx = y.grad[:, :vocab]
    p, near = (more["z"] - l[:, None]).exp(), lr >= -64
    share = more["log_share"].exp().masked_fill(more["there"] | ~more["some"][:, None], 0.0)
    at_share = torch.where(share > 0, more["log_share"].abs(), 0.0) + math.log(vocab) + torch.where(near, 2 * lr.abs(), 0.0)[:, None]
    at_p = torch.where(p > 0, more["z"].abs(), 0.0) + l[:, None] + torch.where(near, lr.abs(), 0.0)[:, None]
    w = scale * g.double().abs()[:, None]
    rel = lambda e: 2.0 ** -22 * (e / math.log(2) + 2) + 2 * d + 2.0 ** -20
    push = torch.zeros(rows, vocab + 1, dtype=torch.float64, device="cuda").scatter_add_(1, torch.where(more["ok"], ids.long(), vocab), q)[:, :vocab]
    lim = w * (p * rel(at_p) + left[:, None] * share * rel(at_share) + 2.0 ** -20 * (push + share))
    if hard:
        p1, m1 = lp1.detach().exp(), y.detach()[:, :vocab].amax(1, keepdim=True)
        far = (y.detach()[:, :vocab] - m1).abs().clamp_max(1e4)
        lim = lim + b.double().abs()[:, None] * (p1 * rel(3 * far + 20) + 2.0 ** -22)
    lim = lim + R.EPS[x.dtype] * 1.001 * dx.abs() + (2.0 ** -25 if dtype == "f16" else 0) + 2.0 ** -126 * (1 + w)
    got = sfb.distill_topk_grad(x, ids, teacher, stats, g, vocab=vocab, scale=scale, tail=True, **args)
    # beyond the type's range a gradient rounds to an infinity (fp16: 0.5 * 10^6 * |g| against 65504 at the largest scale below)
    beyond = (dx.to(x.dtype).isinf()) & (got[:, :vocab] == dx.to(x.dtype))
    off = torch.where(beyond, 0.0, (got[:, :vocab].double() - dx).abs())
    assert bool((off <= lim).all()), "off by %g, %g times the bound" % (float(off.max()), float((off / lim).max()))
    assert not bool(got[:, vocab:].any())
    again = x.clone()
    assert torch.equal(sfb.distill_topk_grad(again, ids, teacher, stats, g, vocab=vocab, scale=scale, tail=True, out=again, **args), got)
    apart = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)[1:].view(x.shape)
    sfb.distill_topk_grad(x, ids, teacher, stats, g, vocab=vocab, scale=scale, tail=True, out=apart, **args)
    assert torch.equal(apart, got)


def far_lists(rows, vocab, k, seed):
    """k tokens per row, some of them twice, some no entries, half of the mass or less in the list."""
    g = gen(seed)
    ids = torch.rand(rows, vocab, device="cuda", generator=g).topk(k, 1).indices.to(torch.int32)
    teacher = (torch.log_softmax(torch.randn(rows, k, device="cuda", generator=g), 1) + math.log(0.5)).contiguous()
    if k > 3:
        ids[:, 2] = ids[:, 0]
        ids[-1, 1] = -1
    return ids.contiguous(), teacher


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width,k", [(5, 700, 704, 9), (1, 100003, 100003, 100), (1500, 1003, 1008, 5), (40, 30522, 30528, 64)])
def test_remainder_far_below(sfb, rows, vocab, width, k, dtype):
    """Listed logits stand 30 to 3000 above the rest, and some of the rest stand out of it."""
    ids, teacher = far_lists(rows, vocab, k, rows + k)
    at = torch.where(ids < 0, ids[:, :1], ids).long()
    for scale, gap in [(1.0, 30.0), (1.0, 62.0), (1.0, 80.0), (1.0, 88.0), (1.0, 104.0), (1.0, 300.0), (10.0, 9.0), (0.5, 3000.0), (64.0, 20.0)]:
        x = make(rows, width, dtype, int(gap), spread=0.5)
        x.scatter_(1, at, make(rows, k, dtype, 1, spread=0.5) + torch.tensor(gap, dtype=x.dtype, device="cuda"))
        check_remainder(sfb, x, ids, teacher, vocab, scale, hard=scale != 0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_remainder_of_the_lowest_values(sfb, dtype):
    """Everything that is not listed holds the type's lowest value, or all but one token does; one row has nothing in its list."""
    rows, vocab, k = 6, 5003, 12
    ids, teacher = far_lists(rows, vocab, k, 4)
    x = torch.full((rows, vocab), torch.finfo(TYPES[dtype]).min, device="cuda", dtype=TYPES[dtype])
    x.scatter_(1, torch.where(ids < 0, ids[:, :1], ids).long(), make(rows, k, dtype, 1))
    x[1, 77] = -200.0
    x[2, 78] = 3.0
    ids[3] = -1
    for scale in (1.0, 0.5, 0.25):
        check_remainder(sfb, x, ids, teacher, vocab, scale, hard=scale == 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width,k", [(5, 700, 704, 9), (300, 20011, 20011, 40)])
def test_remainder_of_nothing(sfb, rows, vocab, width, k, dtype):
    """Every token that is not listed is banned: the loss has no term for the remainder, and its gradient, whose sum over a row is 0, neither.
    One row has a token besides, and one a listed token that is banned, of weight 0."""
    ids, teacher = far_lists(rows, vocab, k, 5)
    x = torch.full((rows, width), -INF, device="cuda", dtype=TYPES[dtype])
    x.scatter_(1, torch.where(ids < 0, ids[:, :1], ids).long(), make(rows, k, dtype, 1))
    x[1, :vocab][torch.ones(vocab, dtype=torch.bool, device="cuda").scatter_(0, ids[1].long(), False).nonzero()[7]] = 1.0
    x[2, ids[2, 4].long()], teacher[2, 4] = -INF, -INF
    for scale in (1.0, 0.5):
        check_remainder(sfb, x, ids, teacher, vocab, scale, hard=scale == 1.0)
        _, stats, _ = sfb.distill_topk(x, ids, teacher, vocab=vocab, scale=scale, tail=True)
        assert torch.equal(stats[:, 2] == -INF, torch.arange(rows, device="cuda") != 1)
        got = sfb.distill_topk_grad(x, ids, teacher, stats, torch.ones(rows, device="cuda"), vocab=vocab, scale=scale, tail=True).double()
        # k entries, each rounded to the type, and the shares' own 2^-18
        assert bool((got.sum(1).abs() <= (R.EPS[x.dtype] + 2.0 ** -18) * got.abs().sum(1) + 1e-7).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_remainder_at_a_large_scale(sfb, dtype):
    """Products with the scale that reach 10^7: powers are of one token, or of ties."""
    rows, vocab, k = 9, 3001, 4
    ids, teacher = far_lists(rows, vocab, k, 4)
    x = make(rows, vocab, dtype, 2).round_()
    for scale in (1000.0, 1.0e6):
        check_remainder(sfb, x, ids, teacher, vocab, scale)


def test_remainder_against_differences(sfb):
    """Central differences of the 64-bit loss (step 1e-5: off by 1e-10 times its third derivative, and by 2^-52 of its value over the step)
    against the gradient's product with the direction, off by 2e-5 of the sum of absolute products: 2^-22 of exponents up to 92, sums."""
    rows, vocab, k = 4, 900, 7
    ids, teacher = far_lists(rows, vocab, k, 9)
    way = make(rows, vocab, "f32", 5).double()
    ones = torch.ones(rows, device="cuda")
    for gap, scale in [(50.0, 1.0), (88.0, 1.0), (150.0, 1.0), (300.0, 1.0), (12.0, 10.0)]:
        x = make(rows, vocab, "f32", 2, spread=1.0)
        x[torch.arange(rows, device="cuda")[:, None], torch.where(ids < 0, ids[:, :1], ids).long()] += gap
        _, stats, _ = sfb.distill_topk(x, ids, teacher, scale=scale, tail=True)
        got = sfb.distill_topk_grad(x, ids, teacher, stats, ones, scale=scale, tail=True).double()
        loss = [divergence(x.double() + s * way, ids, teacher, vocab, scale, True)[0] for s in (1e-5, -1e-5)]
        want = (loss[0] - loss[1]) / 2e-5
        assert bool((((got * way).sum(1) - want).abs() <= 2e-5 * (got * way).abs().sum(1) + 1e-7).all())
        assert bool((got.sum(1).abs() <= 2e-5 * got.abs().sum(1)).all())


# ---- rows whose gradient is not finite ---------------------------------------------------------------------------------------
def gradients(sfb, x, vocab, scale, targets, ids, teacher, g):
    """All of the gradients of some logits, by name: g is every factor that comes from behind."""
    _, stats, ent, _, _, _ = sfb.token_logprobs(x, targets, vocab=vocab, scale=scale, entropy=True)
    _, ts, _, _, _, _ = sfb.token_logprobs(x, targets, vocab=vocab, entropy=True)
    out = {"tokens": sfb.token_logprobs_grad(x, targets, stats, g, vocab=vocab, scale=scale),
           "entropy": sfb.token_logprobs_grad(x, targets, stats, g, ent, g, vocab=vocab, scale=scale)}
    for tail in (False, True):
        _, st, _ = sfb.distill_topk(x, ids, teacher, vocab=vocab, scale=scale, tail=tail)
        out["list", tail] = sfb.distill_topk_grad(x, ids, teacher, st, g, vocab=vocab, scale=scale, tail=tail)
        out["hard", tail] = sfb.distill_topk_grad(x, ids, teacher, st, g, vocab=vocab, scale=scale, tail=tail, targets=targets, token_stats=ts, dlogp=g)
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width", [(8, 997, 1008), (8, 30522, 30528), (600, 1003, 1003 + 37), (8, 4, 40)])
def test_padding_of_rows_that_are_not_finite(sfb, rows, vocab, width, dtype):
    """Columns behind the vocabulary get 0 whatever a row holds or is given; the other rows' gradients are what they are without it."""
    x = make(rows, width, dtype, 1)
    x[:, vocab:] = INF
    k = min(4, vocab - 1)
    ids, teacher = far_lists(rows, vocab, k, 3)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(2), dtype=torch.int32)
    g = torch.randn(rows, device="cuda", generator=gen(4))
    for scale in (1.0, 0.5):
        plain = gradients(sfb, x, vocab, scale, t, ids, teacher, g)
        y, h = x.clone(), g.clone()
        y[0, 1], y[1, vocab - 1], y[2, :vocab], y[3, 1] = math.nan, INF, -INF, -INF
        h[4], h[5], h[6] = INF, -INF, math.nan
        bad = torch.arange(rows, device="cuda") < 7
        for name, got in gradients(sfb, y, vocab, scale, t, ids, teacher, h).items():
            assert not bool(got[:, vocab:].any()), name
            assert torch.equal(got[~bad], plain[name][~bad]), name
            assert bool(got[[0, 1, 6], :vocab].isnan().all()), name
            assert bool((~got[4:6, :vocab].isfinite()).any(1).all()), name
            assert bool(got[2:4, :vocab].isfinite().all()), name


# ---- banned tokens, and factors of both softmaxes ----------------------------------------------------------------------------
def bounds_of(x, t, vocab, size, share, want):
    r = dict(R.token_logprobs(x, t, vocab, 1.0))
    r["l"] = r["l"].clamp_min(0.0)                                       # a row without a token has no sum, and no probability either
    return G.grad_bound(size, share, want, r, vocab, {v: k for k, v in TYPES.items()}[x.dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width", [(9, 700, 704), (9, 30522, 30528), (1400, 1003, 1003)])
def test_gradients_of_banned_tokens(sfb, rows, vocab, width, dtype):
    """-inf and the type's lowest value in a third of the columns each, among them a target; one row has nothing but -inf, one a single token."""
    x = make(rows, width, dtype, vocab)
    for r, value in ((0, -INF), (1, torch.finfo(TYPES[dtype]).min), (rows - 1, -INF)):
        x[r, ::3] = value
    x[2:4] = -INF
    x[3, 5] = 1.0
    x[4:, 1::3] = torch.finfo(TYPES[dtype]).min
    x[4:, 2::3] = -INF
    t = torch.randint(-1, vocab, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
    t[:5] = torch.tensor([3, 6, 7, 5, 2], device="cuda")
    a, b = torch.randn(rows, device="cuda", generator=gen(8)), torch.randn(rows, device="cuda", generator=gen(9))
    for scale, h in [(1.0, None), (1.0, b), (0.25, b)]:
        _, stats, ent, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab, scale=scale, entropy=True)
        got = sfb.token_logprobs_grad(x, t, stats, a, ent if h is not None else None, h, vocab=vocab, scale=scale)
        want, size, _, share = R.token_grad(x, t, a, h, vocab, scale)
        G.same(got[:, :vocab], want, bounds_of(x, t, vocab, size, share, want), "gradient")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,width,k", [(9, 700, 704, 12), (9, 30522, 30528, 64), (1400, 1003, 1003, 5)])
def test_distillation_with_banned_tokens(sfb, rows, vocab, width, k, tail, dtype):
    """The student's banned tokens beside the list's (rows 0 and 1), among them (2: a loss of +inf), and everywhere (3), at the temperatures
    where the hard label's softmax is a power of the student's and at one where it is not."""
    x = make(rows, width, dtype, k)
    ids, teacher = far_lists(rows, vocab, k, 6)
    listed = torch.zeros(rows, vocab + 1, dtype=torch.bool, device="cuda").scatter_(1, torch.where(ids < 0, vocab, ids).long(), True)[:, :vocab]
    third = torch.arange(vocab, device="cuda") % 3 == 0
    for r, value in ((0, -INF), (1, torch.finfo(TYPES[dtype]).min)):
        x[r, :vocab][third & ~listed[r]] = value
    x[2, ids[2, 3].long()] = -INF
    x[3] = -INF
    t = torch.randint(-1, vocab, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
    t[0], t[4], t[5] = 3, ids[4, 1], ids[5, 0]
    a, b = torch.randn(rows, device="cuda", generator=gen(8)), torch.randn(rows, device="cuda", generator=gen(9))
    _, ts, _, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab)
    d = R.bounds(vocab)
    for scale in (1.0, 0.5, 0.25, 0.375):
        loss, stats, missed = sfb.distill_topk(x, ids, teacher, vocab=vocab, scale=scale, tail=tail)
        want = R.distill(x, ids, teacher, vocab, scale, tail)
        want["loss"][3] = INF                                            # no token has a probability
        assert int(missed) == want["missed"] and bool(want["loss"][2:4].isinf().all())
        G.same(loss, want["loss"], (d + 2.0 ** -20) * (1 + want["size"].nan_to_num(0, 0, 0)), "loss")
        G.same(stats[:, 1], want["l"], d, "l")
        for hard in (False, True):
            more = dict(targets=t, token_stats=ts, dlogp=a) if hard else {}
            got = sfb.distill_topk_grad(x, ids, teacher, stats, b, vocab=vocab, scale=scale, tail=tail, **more)
            ref, size, share = R.distill_grad(x, ids, teacher, b, vocab, scale, tail, t if hard else None, a if hard else None)
            # beside the gradients' bounds: the list's probabilities are off by 2^-20 of themselves, the remainder by 2^-22 of 1
            tol = bounds_of(x, t, vocab, size, share, ref) + 2.0 ** -20 * size + (scale * b.double().abs()[:, None]) * 2.0 ** -22 * tail
            G.same(got[:, :vocab], ref, tol, "gradient")
            assert not bool(got[:, vocab:].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [4, 1400])
def test_distillation_of_rows_that_are_not_finite(sfb, rows, dtype):
    vocab, k = 5001, 10
    ids, teacher = far_lists(rows, vocab, k, 6)
    x = make(rows, vocab, dtype, 2)
    for at in (ids[1, 1].item(), (ids[1].amax().item() + 1) % vocab):    # a listed token, and (the odds are) another one
        for value in (math.nan, INF):
            y = x.clone()
            y[1, at] = value
            for tail in (False, True):
                loss, stats, _ = sfb.distill_topk(y, ids, teacher, tail=tail)
                bad = torch.arange(rows, device="cuda") == 1
                assert torch.equal(loss.isnan(), bad) and torch.equal(stats[:, 1:].isnan().all(1), bad) and torch.equal(stats[:, 1:].isnan().any(1), bad)


# ---- scores of few rows: how exact their logits are ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,vocab,k", [(1, 30522, 264), (7, 30522, 512), (7, 30522, 1024), (33, 5003, 520), (128, 2049, 1000), (100, 70001, 776), (5, 100003, 2048),
                                       (16, 37889, 1544)])
def test_logits_of_few_rows(sfb, m, vocab, k, dtype):
    """Products summed 512 of k at a time, from one tile per CTA to several.  A piece takes 32 additions, each of which drops up to a unit in the last
    place of what has been summed so far, half of one on average: at most 2^-24 of it.  Towards a row's largest logit a sum grows evenly, so it is half of
    its end on average: 32 * 2^-24 / 2 = 2^-20 of the logit in all, to which the additions of the pieces add 2^-24 of half the logit each.  In the
    2-norm over the rows' largest logits."""
    g = gen(m + k)
    x = torch.randn(m, k, device="cuda", generator=g).to(TYPES[dtype])
    table = (2.0 / math.sqrt(k) * torch.randn(vocab, k, device="cuda", generator=g)).to(TYPES[dtype])
    t = torch.randint(-1, vocab, (m,), device="cuda", generator=g, dtype=torch.int32)
    t[0] = vocab - 1
    bias = torch.randn(vocab, device="cuda", generator=g)
    for scale, b in [(1.0, None), (0.5, bias)]:
        logp, stats, ent, missed = sfb.linear_logprobs(x, table, t, bias=b, scale=scale, entropy=True)
        assert sfb.device_status() == 0
        z = x.double() @ table.double().t() + (0 if b is None else b.double())
        want = R.token_logprobs(z, t, vocab, scale)
        off = (stats[:, 0].double() - want["m"]).norm() / want["m"].norm()
        assert float(off) <= 2.0 ** -20 + 2.0 ** -25 * (k / 256 + 1), float(off)
        # a token's probability is off by its logit's error, and that of a sum of logits by no more: 2^-20 of the largest |x| |w| of a token, which bounds
        # every partial sum, and D
        d = R.bounds(vocab) + 2.0 ** -24 * 128 + 2 * scale * 2.0 ** -20 * float((x.double().abs() @ table.double().abs().t()).amax() + 4)
        G.same(logp, want["logp"], d + 2.0 ** -22 * want["logp"].abs(), "logp")
        G.same(ent, want["entropy"], 2 * d * (1 + 2 * want["entropy"].abs()), "entropy")
        again = sfb.linear_logprobs(x, table, t, bias=b, scale=scale, entropy=True)
        assert torch.equal(logp, again[0]) and torch.equal(stats, again[1])
