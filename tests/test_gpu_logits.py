"""GPU tests of the operators on logits against their definitions in 64 bits.

Forward results are fp32 whatever the logits' type.  With D = bounds(vocab) the relative error of a row's sum of exponentials
(logits_reference.bounds), l = log of it is off by D, and a value a (x - m) - l by D plus 2^-22 of its own size; the entropy is a
quotient of two such sums, off by 2 D of (1 + its size + the sum of p |log p|, the entropy again).  Gradients: an exponent t = log2 p
is off by 2^-22 |t| + 2^-22 l, so p by that share of itself, plus D for the sum, plus half a step of the type."""
import math

import pytest

torch = pytest.importorskip("torch")
import logits_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(rows, vocab, width, dtype, seed, spread=2.5, offset=0):
    """Logits [rows, width] that start `offset` elements into their memory."""
    g = gen(seed)
    flat = torch.empty(rows * width + offset, device="cuda", dtype=TYPES[dtype])
    x = flat[offset:].view(rows, width)
    x.copy_(spread * torch.randn(rows, width, device="cuda", generator=g))
    return x


def same(got, want, tol, what):
    """|got - want| <= tol, infinities and NaN alike."""
    got, want = got.reshape(want.shape).double(), want.double()
    fin = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), what
    err = (got - want)[fin].abs()
    lim = torch.broadcast_to(torch.as_tensor(tol, device=want.device, dtype=torch.float64), want.shape)[fin]
    assert bool((err <= lim).all()), "%s: off by %g, %g times the bound" % (what, float(err.max()), float((err / lim).max()))


def check_forward(sfb, x, targets, vocab, scale, entropy, top_k):
    logp, stats, ent, top_logp, top_ids, missed = sfb.token_logprobs(x, targets, vocab=vocab, scale=scale, entropy=entropy, top_k=top_k)
    want = R.token_logprobs(x, targets, vocab or x.shape[-1], scale, top_k)
    d = R.bounds(vocab or x.shape[-1])
    nothing = torch.zeros_like(want["m"], dtype=torch.bool)
    if targets is not None:
        if not entropy and not top_k:
            nothing = (targets.reshape(-1) < 0) | (targets.reshape(-1) >= (vocab or x.shape[-1]))
        same(logp, want["logp"], d + 2.0 ** -22 * want["logp"].abs(), "logp")
        assert int(missed) == want["missed"]
    else:
        assert logp is None and int(missed) == 0
    same(stats[..., 0], torch.where(nothing, 0.0, want["m"]), 0.0, "m")
    same(stats[..., 1], torch.where(nothing, 0.0, want["l"]), d, "l")
    if entropy:
        same(ent, want["entropy"], 2 * d * (1 + 2 * want["entropy"].abs()), "entropy")
    else:
        assert ent is None
    if top_k:
        assert torch.equal(top_ids.reshape(-1, top_k).long(), want["top_ids"])
        same(top_logp, want["top_logp"], d + 2.0 ** -22 * want["top_logp"].abs(), "top_logp")
    else:
        assert top_logp is None and top_ids is None
    return stats, ent


SIZES = [(1, 1, 1), (3, 2, 2), (2, 7, 9), (1, 8, 8), (5, 33, 33), (2, 129, 144), (37, 1000, 1000), (3, 2049, 2050), (1, 30522, 30528), (2, 30522, 30522),
         (300, 5003, 5003), (9, 100003, 100003), (700, 3000, 3008), (20, 131072, 131072), (1300, 517, 520), (6000, 1203, 1203)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_token_logprobs(sfb, rows, vocab, width, dtype):
    x = make(rows, vocab, width, dtype, rows + vocab)
    t = torch.randint(-1, vocab + 1, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
    for scale, entropy, k in [(1.0, False, 0), (0.7, True, 0), (1.0, False, min(5, vocab)), (1.3, True, min(128, vocab))]:
        check_forward(sfb, x, t, vocab, scale, entropy, k)
    check_forward(sfb, x, None, vocab, 1.0, True, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_rows_that_start_anywhere(sfb, dtype, offset):
    x = make(6, 4099, 4101, dtype, offset, offset=offset)
    x[:, 4099:] = INF                                                   # padding is never looked at
    t = torch.randint(0, 4099, (6,), device="cuda", generator=gen(6), dtype=torch.int32)
    check_forward(sfb, x, t, 4099, 1.0, True, 20)
    y = x[:, :4099].view(2, 3, 4099)                                    # leading dimensions, rows at a pitch
    check_forward(sfb, y, t.view(2, 3), None, 1.0, True, 20)
    check_forward(sfb, x[2, :4099], t[2], None, 1.0, True, 3)           # a single row without a leading dimension
    check_forward(sfb, x[::2, :4099], t[::2].contiguous(), None, 1.0, False, 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 400, 5000])
def test_values_that_are_not_ordinary(sfb, dtype, rows):
    vocab = 9000
    low = torch.finfo(TYPES[dtype]).min
    kinds = [lambda x: x.fill_(-INF), lambda x: x.fill_(0.5), lambda x: x.fill_(low), lambda x: x[50:].fill_(-INF), lambda x: x[3:].fill_(low),
             lambda x: x[:-1].fill_(-INF), lambda x: x.copy_(x.sort().values), lambda x: x.copy_(x.sort(descending=True).values), lambda x: x.add_(1000.0),
             lambda x: x.round_(), lambda x: x[::2].fill_(-0.0) + x[1::2].fill_(0.0).sum(), lambda x: x.fill_(-INF)[7].fill_(low),
             lambda x: x[4321:4322].fill_(INF), lambda x: x[4321:4322].fill_(math.nan), lambda x: x.fill_(-INF)[77].fill_(math.nan), lambda x: x.fill_(math.nan)]
    for n, change in enumerate(kinds):
        x = make(rows, vocab, vocab, dtype, n)
        for r in {0, rows // 2, rows - 1}:
            change(x[r])
        t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(n), dtype=torch.int32)
        t[0] = 7
        if n < 12:
            check_forward(sfb, x, t, vocab, 1.0, True, 20)
            check_forward(sfb, x, t, vocab, 1.0, True, 0)
            check_forward(sfb, x, t, vocab, 1.0, False, 0)
            continue
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[[0, rows // 2, rows - 1]] = True
        for k in (20, 0):
            logp, stats, ent, top_logp, top_ids, _ = sfb.token_logprobs(x, t, entropy=True, top_k=k)
            assert torch.equal(logp.isnan(), bad) and torch.equal(ent.isnan(), bad) and torch.equal(stats[:, 1].isnan(), bad)
            if k:
                assert torch.equal(top_logp.isnan().all(1), bad) and torch.equal((top_ids == -1).all(1), bad)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 30, 1500])
def test_ties_at_the_bound(sfb, rows, dtype):
    """More equal values than there are places for candidates, with more, fewer and no larger ones above them."""
    vocab = 20001
    for n, (value, larger) in enumerate([(0.0, 0), (1.5, 5), (-2.0, 19), (-2.0, 20), (torch.finfo(TYPES[dtype]).min, 3)]):
        x = torch.full((rows, vocab + 7), value, device="cuda", dtype=TYPES[dtype])
        at = torch.randint(0, vocab, (rows, max(larger, 1)), device="cuda", generator=gen(n))
        if larger:
            x.scatter_(1, at, 3.0 + torch.arange(larger, device="cuda").to(x.dtype).expand(rows, -1))
        x[0, :500] = -INF
        x[-1, vocab - 30:] = -INF
        some = [0, rows // 2, rows - 1]
        _, stats, _, top_logp, top_ids, _ = sfb.token_logprobs(x, vocab=vocab, top_k=20)
        want = R.token_logprobs(x[some], None, vocab, 1.0, 20)
        assert torch.equal(top_ids[some].long(), want["top_ids"])
        same(top_logp[some], want["top_logp"], R.bounds(vocab) + 2.0 ** -22 * want["top_logp"].abs(), "top_logp")


@pytest.mark.parametrize("rows", [2, 500])
def test_alternatives_that_sit_with_few_threads(sfb, rows):
    """Large values at one place of every 2048 elements: a thread or two hold most of them, and its neighbours' bound is far below."""
    x = make(rows, 131072, 131072, "bf16", 3)
    x[:, 5::2048] += 50.0
    x[:, 6::2048] += 50.0
    check_forward(sfb, x[:4], torch.zeros(min(4, rows), device="cuda", dtype=torch.int32), None, 1.0, False, 128)
    y = make(rows, 131072, 131072, "f32", 4)
    for k in range(19):                                                 # and thousands of others above what the rest of the threads hold
        y[:, 40 + 4 * k::1024] += 40.0
    check_forward(sfb, y[:4], None, None, 1.0, False, 100)


@pytest.mark.parametrize("rows", [2, 1300])
@pytest.mark.parametrize("vocab,k", [(65, 1), (300, 32), (1000, 33), (4100, 5), (8200, 32)])
def test_alternatives_of_short_rows(sfb, rows, vocab, k):
    """From two to eight warps per row, by their length, their number and the alternatives'."""
    for dtype in ("f32", "bf16"):
        x = make(rows, vocab, vocab, dtype, vocab).round_(decimals=1)      # with ties
        t = torch.randint(-1, vocab, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
        check_forward(sfb, x, t, None, 1.0, True, k)
        x[1:] = 2.0
        check_forward(sfb, x, t, None, 1.0, False, k)


def test_rows_without_a_target_are_not_read(sfb):
    x = make(50, 3001, 3001, "f32", 1)
    t = torch.randint(0, 3001, (50,), device="cuda", generator=gen(1), dtype=torch.int32)
    none = torch.arange(50, device="cuda") % 3 == 0
    t[none] = -100
    t[1] = 3001
    none[1] = True
    x[none] = math.nan
    logp, stats, _, _, _, missed = sfb.token_logprobs(x, t)
    assert int(missed) == int(none.sum()) and not bool(logp[none].any()) and not bool(stats[none].any())
    assert bool(stats[~none].isfinite().all())
    dx = sfb.token_logprobs_grad(x, t, stats, torch.ones_like(logp))
    assert not bool(dx[none].any()) and bool(dx.isfinite().all())


def test_many_targets_are_counted(sfb):
    for rows in (100, 3000, 40000):
        x = make(rows, 130, 136, "bf16", 2)
        t = torch.randint(-1, 2, (rows,), device="cuda", generator=gen(rows), dtype=torch.int32)
        assert int(sfb.token_logprobs(x, t, vocab=130)[5]) == int((t < 0).sum())
        ids = torch.randint(-1, 131, (rows, 3), device="cuda", generator=gen(rows), dtype=torch.int32)
        assert int(sfb.distill_topk(x, ids, torch.zeros(rows, 3, device="cuda"), vocab=130)[2]) == int(((ids < 0) | (ids >= 130)).sum())


# ---- gradients -------------------------------------------------------------------------------------------------------------
def grad_bound(size, share, result, r, vocab, dtype):
    """size: the sum of the absolute shares of p; see the module's comment.  share: the target's own, scale * dlogp: its product
    rounds once, so does its factor in c0 (2^-24 each), and the sum of what nearly cancels once more, by 2^-24 of either: 2^-22."""
    t = torch.where(r["p"] > 0, (r["z"] - r["l"][:, None]).abs() / math.log(2), 0.0)
    rel = R.bounds(vocab) * 2 + 2.0 ** -22 * (t + r["l"].abs()[:, None] / math.log(2) + 2)
    # what is below the smallest number of the type, or of the powers (2^-126), is lost
    return rel * size + 2.0 ** -22 * share + R.EPS[TYPES[dtype]] * result.abs() * 1.001 + (2.0 ** -25 if dtype == "f16" else 0) + 2.0 ** -126 * (1 + size.amax())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_token_logprobs_grad(sfb, rows, vocab, width, dtype):
    x = make(rows, vocab, width, dtype, rows + vocab)
    t = torch.randint(-1, vocab + 1, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
    dlogp = torch.randn(rows, device="cuda", generator=gen(8))
    dent = torch.randn(rows, device="cuda", generator=gen(9))
    for scale, h in [(1.0, None), (0.6, dent)]:
        _, stats, ent, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab, scale=scale, entropy=True)
        got = sfb.token_logprobs_grad(x, t, stats, dlogp, ent if h is not None else None, h, vocab=vocab, scale=scale)
        want, size, r, share = R.token_grad(x, t, dlogp, h, vocab, scale)
        assert got.dtype == x.dtype and got.shape == x.shape and not bool(got[:, vocab:].any())
        same(got[:, :vocab], want, grad_bound(size, share, want, r, vocab, dtype), "gradient")
        again = x.clone()
        assert sfb.token_logprobs_grad(again, t, stats, dlogp, ent if h is not None else None, h, vocab=vocab, scale=scale, out=again) is again
        assert torch.equal(again, got)                                  # in place
        apart = torch.empty(rows * width + 3, device="cuda", dtype=x.dtype)[3:].view(rows, width)
        sfb.token_logprobs_grad(x, t, stats, dlogp, ent if h is not None else None, h, vocab=vocab, scale=scale, out=apart)
        assert torch.equal(apart, got)                                  # windows that start elsewhere


def test_gradient_leaves_what_lies_between_the_rows(sfb):
    memory = torch.full((7, 4160), 3.0, device="cuda", dtype=torch.bfloat16)
    x = make(7, 4099, 4099, "bf16", 1)
    out = memory[:, 9:4108]
    t = torch.zeros(7, device="cuda", dtype=torch.int32)
    logp, stats, _, _, _, _ = sfb.token_logprobs(x, t)
    sfb.token_logprobs_grad(x, t, stats, torch.ones_like(logp), out=out)
    assert bool((memory[:, :9] == 3).all()) and bool((memory[:, 4108:] == 3).all())
    assert torch.equal(out, sfb.token_logprobs_grad(x, t, stats, torch.ones_like(logp)))


def test_gradients_against_differences(sfb):
    """Directional derivatives of the 64-bit definitions (central differences, step 1e-5: off by the third derivative times
    1e-10, and 1e-16 of the value over the step, 1e-10) against the gradients' products with the direction; those are off by the
    bounds above, here 2e-6 of the sum of absolute products."""
    rows, vocab, k = 5, 700, 9
    x, way = make(rows, vocab, vocab, "f32", 1), make(rows, vocab, vocab, "f32", 2).double()
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(5), dtype=torch.int32)
    a, b, c = (torch.randn(rows, device="cuda", generator=gen(n)) for n in (11, 12, 13))
    ids = torch.randint(0, vocab, (rows, k), device="cuda", generator=gen(3), dtype=torch.int32)
    teacher = torch.log_softmax(torch.randn(rows, k + 1, device="cuda", generator=gen(4)), 1)[:, :k].contiguous()

    def along(f):
        return (f(x.double() + 1e-5 * way) - f(x.double() - 1e-5 * way)) / 2e-5

    def agrees(d, want):
        prod = (d.double() * way).sum(1)
        assert bool(((prod - want).abs() <= 2e-6 * (d.double() * way).abs().sum(1) + 1e-8).all())

    _, stats, ent, _, _, _ = sfb.token_logprobs(x, t, scale=0.8, entropy=True)

    def tokens(y):
        r = R.token_logprobs(y, t, vocab, 0.8)
        return a.double() * r["logp"] + b.double() * r["entropy"]
    agrees(sfb.token_logprobs_grad(x, t, stats, a, ent, b, scale=0.8), along(tokens))
    for tail in (False, True):
        _, st, _ = sfb.distill_topk(x, ids, teacher, scale=0.5, tail=tail)
        agrees(sfb.distill_topk_grad(x, ids, teacher, st, c, scale=0.5, tail=tail),
               along(lambda y: c.double() * R.distill(y, ids, teacher, vocab, 0.5, tail)["loss"]))
        _, ts, _, _, _, _ = sfb.token_logprobs(x, t)
        agrees(sfb.distill_topk_grad(x, ids, teacher, st, c, scale=0.5, tail=tail, targets=t, token_stats=ts, dlogp=a),
               along(lambda y: c.double() * R.distill(y, ids, teacher, vocab, 0.5, tail)["loss"] + a.double() * R.token_logprobs(y, t, vocab, 1.0)["logp"]))


# ---- distillation ------------------------------------------------------------------------------------------------------------
def make_lists(x, vocab, k, seed, tail):
    """The teacher's k best: the logits through noise, some lists shorter, some with an id twice."""
    rows = x.shape[0]
    g = gen(seed)
    noisy = x[:, :vocab].float() + torch.randn(rows, vocab, device="cuda", generator=g)
    lp, ids = torch.log_softmax(noisy, 1).topk(min(k, vocab), 1)
    if k > vocab:
        ids = torch.cat([ids, ids[:, :1].expand(-1, k - vocab)], 1)
        lp = torch.cat([lp, lp[:, :1].expand(-1, k - vocab)], 1) - (math.log(4.0) if tail else 0.0)
    ids, lp = ids.to(torch.int32).contiguous(), lp.contiguous()
    if rows > 2:
        ids[1, k // 2:] = -1
        ids[2] = -5
    if rows > 4 and k > 3:
        ids[3, 2] = ids[3, 0]
        lp[4, 1] = -INF
        ids[4, 3] = vocab
    return ids, lp


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,width,k", [(1, 1, 1, 1), (3, 5, 8, 7), (5, 33, 33, 4), (37, 1000, 1000, 128), (6, 4099, 4101, 20), (1, 30522, 30528, 64), (400, 5003, 5003, 17), (1500, 1003, 1003, 40), (5000, 9001, 9008, 3),
                                               (9, 100003, 100003, 100)])
def test_distill(sfb, rows, vocab, width, k, tail, dtype):
    x = make(rows, vocab, width, dtype, rows + k)
    ids, teacher = make_lists(x, vocab, k, 7, tail)
    scale = 0.5
    loss, stats, missed = sfb.distill_topk(x, ids, teacher, vocab=vocab, scale=scale, tail=tail)
    want = R.distill(x, ids, teacher, vocab, scale, tail)
    d = R.bounds(vocab)
    assert int(missed) == want["missed"] and stats.shape == (rows, 3 if tail else 2)
    # a list's sum is of at most 128 terms in 4 per lane; 1 - sum loses 2^-23, its logarithm's product with itself at most 2^-20 of 1
    same(loss, want["loss"], (d + 2.0 ** -20) * (1 + want["size"]), "loss")
    same(stats[:, 0], want["m"], 0.0, "m")
    same(stats[:, 1], want["l"], d, "l")
    if tail:
        same(stats[:, 2], want["lr"], d + 2.0 ** -22 * want["lr"].abs().nan_to_num(0, 0, 0), "rest")
    dloss = torch.randn(rows, device="cuda", generator=gen(9))
    t = torch.randint(-1, vocab, (rows,), device="cuda", generator=gen(10), dtype=torch.int32)
    if rows > 3:
        t[3] = ids[3, 0]
    dlogp = torch.randn(rows, device="cuda", generator=gen(11))
    _, ts, _, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab, entropy=True)
    for hard in (False, True):
        more = dict(targets=t, token_stats=ts, dlogp=dlogp) if hard else {}
        got = sfb.distill_topk_grad(x, ids, teacher, stats, dloss, vocab=vocab, scale=scale, tail=tail, **more)
        ref, size, share = R.distill_grad(x, ids, teacher, dloss, vocab, scale, tail, t if hard else None, dlogp if hard else None)
        r = R.token_logprobs(x, t, vocab, 1.0)
        # the list's probabilities are off by 2^-20 of themselves, the remainder's by 2^-22 of 1 (a difference from 1)
        slack = (scale * dloss.double().abs()[:, None]) * 2.0 ** -22 * (1.0 if tail else 0.0)
        tol = grad_bound(size, share, ref, r, vocab, dtype) + 2.0 ** -20 * size + slack
        assert not bool(got[:, vocab:].any())
        same(got[:, :vocab], ref, tol, "gradient")
        again = x.clone()
        assert torch.equal(sfb.distill_topk_grad(again, ids, teacher, stats, dloss, vocab=vocab, scale=scale, tail=tail, out=again, **more), got)
        apart = torch.empty(rows * width + 1, device="cuda", dtype=x.dtype)[1:].view(rows, width)
        sfb.distill_topk_grad(x, ids, teacher, stats, dloss, vocab=vocab, scale=scale, tail=tail, out=apart, **more)
        assert torch.equal(apart, got)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows", [3, 2000])
def test_divergences_that_are_small(sfb, rows, tail):
    """A student next to its teacher, most of the mass outside the list (tail) or on it: the divergence is a thousandth of the
    logarithms it is made of.  Each of those, at most 16, rounds by 2^-21; they come weighted by the list's mass, at most 0.1 here
    with the tail, where the two remainders' logarithms are below 0.1 and round by 2^-27; sums of the list and the row are
    off by their bounds, once for each side: in all at most (2^-20 + 2 D) times that mass, D = bounds(vocab)."""
    vocab, k = (10413, 73) if tail else (400, 128)
    x = make(rows, vocab, vocab, "f32", 1, spread=2.0)
    if not tail:
        x[:, 128:] -= 12.0
    noisy = x + 0.1 * torch.randn(rows, vocab, device="cuda", generator=gen(2))
    lp, ids = torch.log_softmax(0.25 * noisy if tail else noisy, 1).topk(k, 1)
    ids, lp = ids.to(torch.int32).contiguous(), lp.contiguous()
    scale = 0.25 if tail else 1.0
    loss, _, _ = sfb.distill_topk(x, ids, lp, scale=scale, tail=tail)
    want = R.distill(x, ids, lp, vocab, scale, tail)
    mass = lp.double().exp().sum(1)
    assert float(mass.max()) < 0.1 if tail else float(mass.min()) > 0.9
    same(loss, want["loss"], (2.0 ** -20 + 2 * R.bounds(vocab)) * mass, "loss")


def test_weights_far_from_probabilities(sfb):
    """The renormalised list may be any log weights: their common offset does not matter, and costs nothing of the loss."""
    x = make(9, 3000, 3000, "f32", 1)
    ids, teacher = make_lists(x, 3000, 100, 7, False)
    for shift in (1024.0, -4096.0):                                     # exact sums: the list's values have 2^-11 to spare below
        moved = ((teacher * 2048).round() / 2048).contiguous()
        a, _, _ = sfb.distill_topk(x, ids, moved)
        b, _, _ = sfb.distill_topk(x, ids, moved + shift)
        same(b, a.double(), 2.0 ** -20 * (1 + a.double().abs()), "loss")


def test_remainder_that_is_small(sfb):
    """Nearly all of the student's mass is on the list: what it leaves is summed by itself, not as a difference from 1."""
    x = make(4, 20000, 20000, "f32", 1, spread=1.0)
    ids = torch.tensor([[3, 9, 19999, 12345]] * 4, device="cuda", dtype=torch.int32)
    x[:, ids[0].long()] += 40.0
    teacher = torch.log(torch.tensor([[0.2, 0.1, 0.1, 0.1]] * 4, device="cuda"))
    loss, stats, _ = sfb.distill_topk(x, ids, teacher, tail=True)
    want = R.distill(x, ids, teacher, 20000, 1.0, True)
    same(loss, want["loss"], (R.bounds(20000) + 2.0 ** -20) * (1 + want["size"]), "loss")
    dloss = torch.ones(4, device="cuda")
    got = sfb.distill_topk_grad(x, ids, teacher, stats, dloss, tail=True)
    ref, size, _ = R.distill_grad(x, ids, teacher, dloss, 20000, 1.0, True)
    # exponents are small here (unlisted tokens relative to their own sum): 2^-16 covers 2^-22 of an l of 60 and the sums
    same(got, ref, 2.0 ** -16 * size + 1e-30, "gradient")


# ---- as a program uses them ----------------------------------------------------------------------------------------------------
def test_a_training_step_on_the_logits(sfb):
    """Logits over a padded table, the teacher's list, the mixed loss and its gradient, and what goes back to the hidden states."""
    m, hidden, vocab, width = 96, 128, 1501, 1504
    g = gen(1)
    h = torch.randn(m, hidden, device="cuda", generator=g).to(torch.bfloat16)
    table = torch.zeros(width, hidden, device="cuda", dtype=torch.bfloat16)
    table[:vocab] = (0.2 * torch.randn(vocab, hidden, device="cuda", generator=g)).to(torch.bfloat16)
    teacher_h = (h.float() + 0.3 * torch.randn(m, hidden, device="cuda", generator=g)).to(torch.bfloat16)
    t = torch.randint(0, vocab, (m,), device="cuda", generator=g, dtype=torch.int32)
    _, _, _, top, ids, _ = sfb.token_logprobs(sfb.linear_nt(teacher_h, table), vocab=vocab, scale=0.5, top_k=32)
    x = sfb.linear_nt(h, table)
    logp, ts, _, _, _, _ = sfb.token_logprobs(x, t, vocab=vocab)
    loss, st, missed = sfb.distill_topk(x, ids, top, vocab=vocab, scale=0.5)
    assert int(missed) == 0 and float(loss.min()) > -1e-5
    dloss, dlogp = torch.full((m,), 4.0 / m, device="cuda"), torch.full((m,), -0.5 / m, device="cuda")
    dx = sfb.distill_topk_grad(x, ids, top, st, dloss, vocab=vocab, scale=0.5, targets=t, token_stats=ts, dlogp=dlogp, out=x)
    assert dx is x
    dh = sfb.linear(dx, table)
    y = sfb.linear_nt(h, table).double()[:, :vocab].requires_grad_(True)
    lq = torch.log_softmax(top.double(), 1)
    kd = (lq.exp() * (lq - torch.log_softmax(0.5 * y, 1).gather(1, ids.long()))).sum(1)
    total = (dloss.double() * kd + dlogp.double() * torch.log_softmax(y, 1).gather(1, t.long()[:, None])[:, 0]).sum()
    total.backward()
    same(kd.detach().float(), loss.double(), 1e-5 * (1 + loss.double().abs()), "loss")
    same(dx[:, :vocab], y.grad, 2.0 ** -8 * 1.01 * y.grad.abs() + 1e-7, "gradient")     # fp32 shares of at most 0.05, then one rounding to bf16
    want = dx.double() @ table.double()
    same(dh, want, 2.0 ** -8 * want.abs() + 1e-6 * (dx.double().abs() @ table.double().abs()) + 1e-9, "hidden")


def test_captured_and_replayed(sfb):
    x, t = make(64, 5000, 5008, "bf16", 1), torch.randint(0, 5000, (64,), device="cuda", generator=gen(1), dtype=torch.int32)
    ids, teacher = make_lists(x, 5000, 16, 2, True)
    w = torch.rand(64, device="cuda", generator=gen(4))

    def step():
        f = sfb.token_logprobs(x, t, vocab=5000, entropy=True, top_k=10)
        d = sfb.distill_topk(x, ids, teacher, vocab=5000, tail=True)
        return f + d + (sfb.token_logprobs_grad(x, t, f[1], w, f[2], w, vocab=5000),
                        sfb.distill_topk_grad(x, ids, teacher, d[1], w, vocab=5000, tail=True, targets=t, token_stats=f[1], dlogp=w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (2, 3):
        x.copy_(make(64, 5000, 5008, "bf16", seed))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once(sfb):
    xs = [make(8, 60000, 60000, "bf16", n) for n in (1, 2)]
    t = torch.zeros(8, device="cuda", dtype=torch.int32)
    want = [sfb.token_logprobs(x, t, entropy=True, top_k=30) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(sfb.token_logprobs(xs[n], t, entropy=True, top_k=30))
    torch.cuda.synchronize()
    for n in (0, 1):
        for g in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[n]))


def test_rows_far_apart(sfb):
    """Offsets beyond 32 bits, in elements and in bytes."""
    pitch = (1 << 30) + 5
    memory = torch.empty(4 * pitch, device="cuda", dtype=torch.bfloat16)
    x = memory.as_strided((4, 1000), (pitch, 1))
    x.copy_(make(4, 1000, 1000, "bf16", 1))
    t = torch.randint(0, 1000, (4,), device="cuda", generator=gen(5), dtype=torch.int32)
    stats, ent = check_forward(sfb, x, t, None, 1.0, True, 5)
    w = torch.ones(4, device="cuda")
    got = sfb.token_logprobs_grad(x, t, stats, w, ent, w, out=x)
    want = sfb.token_logprobs_grad(make(4, 1000, 1000, "bf16", 1), t, stats, w, ent, w)
    assert torch.equal(got, want)


def test_no_rows(sfb):
    x = torch.empty(0, 50, device="cuda")
    t = torch.empty(0, device="cuda", dtype=torch.int32)
    f = torch.empty(0, device="cuda")
    logp, stats, ent, top, ids, missed = sfb.token_logprobs(x, t, entropy=True, top_k=3)
    assert logp.shape == (0,) and stats.shape == (0, 2) and top.shape == (0, 3) and int(missed) == 0
    assert sfb.token_logprobs_grad(x, t, stats, f, ent, f).shape == (0, 50)
    ids, teacher = torch.empty(0, 4, device="cuda", dtype=torch.int32), torch.empty(0, 4, device="cuda")
    loss, st, missed = sfb.distill_topk(x, ids, teacher, tail=True)
    assert loss.shape == (0,) and st.shape == (0, 3) and int(missed) == 0
    assert sfb.distill_topk_grad(x, ids, teacher, st, f, tail=True).shape == (0, 50)


# ---- scores without logits -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,vocab,rows,k", [(1, 1, 1, 8), (1, 30522, 30528, 768), (7, 1000, 1000, 72), (128, 129, 129, 64), (129, 255, 256, 128), (300, 5003, 5003, 264),
                                            (700, 30522, 30528, 768), (2000, 2049, 2049, 40), (5000, 260, 260, 1024)])
def test_linear_logprobs(sfb, m, vocab, rows, k, dtype):
    """A logit is a sum of k exact products, rounded at most once per 16 of them and in the accumulator: off by 2^-22 (k / 16 + 4)
    of the sum of their sizes; a logarithm of a sum of exponentials by the largest such error, on top of the bounds above (a
    thread adds 128 terms, a row's parts are joined in at most vocab / 128 steps)."""
    g = gen(m + vocab)
    x = torch.randn(m, k, device="cuda", generator=g).to(TYPES[dtype])
    table = (2.0 / math.sqrt(k) * torch.randn(rows, k, device="cuda", generator=g)).to(TYPES[dtype])
    table[vocab:] = INF
    t = torch.randint(-1, vocab + 1, (m,), device="cuda", generator=g, dtype=torch.int32)
    t[0] = vocab - 1
    for scale, entropy, bias in [(1.0, False, None), (0.7, True, torch.randn(rows + 1, device="cuda", generator=g)[1:])]:
        logp, stats, ent, missed = sfb.linear_logprobs(x, table, t, bias=bias, vocab=vocab, scale=scale, entropy=entropy)
        assert sfb.device_status() == 0
        z = x.double() @ table[:vocab].double().t() + (0 if bias is None else bias[:vocab].double())
        off = scale * 2.0 ** -22 * (k / 16 + 4) * float((x.double().abs() @ table[:vocab].double().abs().t()).amax() + 4)
        want = R.token_logprobs(z, t, vocab, scale)
        d = R.bounds(vocab) + 2.0 ** -24 * 128 + 2 * off
        nothing = torch.zeros_like(want["m"], dtype=torch.bool) if entropy else (t < 0) | (t >= vocab)
        assert int(missed) == want["missed"]
        same(logp, want["logp"], d + 2.0 ** -22 * want["logp"].abs(), "logp")
        same(stats[:, 0], torch.where(nothing, 0.0, want["m"]), off / scale, "m")
        same(stats[:, 1], torch.where(nothing, 0.0, want["l"]), d, "l")
        if entropy:
            same(ent, want["entropy"], 2 * d * (1 + 2 * want["entropy"].abs()), "entropy")
        else:
            assert ent is None
        again = sfb.linear_logprobs(x, table, t, bias=bias, vocab=vocab, scale=scale, entropy=entropy)
        assert torch.equal(logp, again[0]) and torch.equal(stats, again[1])


def test_linear_logprobs_of_many_rows(sfb):
    """More rows than go through the workspace at a time."""
    m, vocab, k = 70001, 300, 16
    g = gen(5)
    x = torch.randn(m, k, device="cuda", generator=g).to(torch.bfloat16)
    table = torch.randn(vocab, k, device="cuda", generator=g).to(torch.bfloat16)
    t = torch.randint(-1, vocab, (m,), device="cuda", generator=g, dtype=torch.int32)
    logp, stats, ent, missed = sfb.linear_logprobs(x, table, t, entropy=True)
    want = R.token_logprobs(x.double() @ table.double().t(), t, vocab, 1.0)
    same(logp, want["logp"], 5e-5, "logp")                               # 16 products of at most 20: off by 2^-22 * 5 * 200 at most in a logit
    same(ent, want["entropy"], 5e-4, "entropy")
    assert int(missed) == want["missed"]


def test_linear_logprobs_of_what_is_not_finite(sfb):
    m, vocab, k = 200, 1000, 64
    g = gen(3)
    x = torch.randn(m, k, device="cuda", generator=g).to(torch.bfloat16)
    table = torch.randn(vocab, k, device="cuda", generator=g).to(torch.bfloat16)
    t = torch.full((m,), 5, device="cuda", dtype=torch.int32)
    t[1] = 900
    bias = torch.zeros(vocab, device="cuda")
    bias[700:] = -INF                                                    # banned tokens
    logp, stats, ent, _ = sfb.linear_logprobs(x, table, t, bias=bias, entropy=True)
    z = x.double() @ table.double().t() + bias.double()
    want = R.token_logprobs(z, t, vocab, 1.0)
    same(logp, want["logp"], 1e-4, "logp")                               # 64 products of size 1: off by 2^-22 * 8 * 64
    same(ent, want["entropy"], 1e-3, "entropy")
    bias[:] = -INF
    logp, stats, ent, _ = sfb.linear_logprobs(x, table, t, bias=bias, entropy=True)
    assert bool((logp == -INF).all()) and bool((stats == -INF).all()) and not bool(ent.any())
    x[3, 0] = math.nan
    logp, stats, _, _ = sfb.linear_logprobs(x, table, t)
    assert bool(logp[3].isnan()) and int(logp.isnan().sum()) == 1
    assert sfb.device_status() == 0


def test_linear_logprobs_captured_beside_another(sfb):
    """Two captured calls and an eager one between them: each has a workspace of its own."""
    g = gen(4)
    x = [torch.randn(2, 150, 256, device="cuda", generator=g).to(torch.float16) for _ in range(2)]
    table = (0.1 * torch.randn(7000, 256, device="cuda", generator=g)).to(torch.float16)
    t = torch.randint(0, 7000, (2, 150), device="cuda", generator=g, dtype=torch.int32)
    want = [sfb.linear_logprobs(y, table, t, entropy=True) for y in x]
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph() for _ in x], []
    for n in (0, 1):
        with torch.cuda.graph(graphs[n]):
            held.append(sfb.linear_logprobs(x[n], table, t, entropy=True))
    streams = [torch.cuda.Stream() for _ in x]
    for _ in range(5):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                graphs[n].replay()
        sfb.linear_logprobs(x[0], table, t)
    torch.cuda.synchronize()
    for a, b in zip(held, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].shape == (2, 150)
