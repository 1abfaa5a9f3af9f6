"""The operators of a training step around the attention where the tests beside this file do not reach."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_training import check_attention, check_embed_grad, layout, operands, plan                         # noqa: E402
from training_reference import DTYPES                                                                         # noqa: E402


# ---- attention ------------------------------------------------------------------------------------------------------------------
def rounding_variance(x):
    """Of the rounding of every entry of x to fp16: evenly spread over half a step to both sides, steps of 2^(e - 10) from 2^e on, of 2^-24 below 2^-14."""
    e = torch.frexp(x)[1] - 1                               # 2^e <= |x| < 2^(e + 1); of 0: no error
    half = torch.ldexp(torch.ones_like(x), e.clamp_min(-14) - 11)
    return torch.where(x == 0, 0.0, half * half / 3)


@pytest.mark.parametrize("bs,d,kind", [(64, 64, "full"), (64, 64, "causal"), (32, 64, "full"), (64, 128, "causal"), (32, 40, "full")])
@pytest.mark.parametrize("power", [6, 0, -5, -8, -12])
def test_fp16_gradients_of_small_losses(sfb, bs, d, kind, power):
    """dO of a mean over many tokens and rows of 2048 keys: most of dS is below fp16's normal numbers.  The norm of what dQ, dK and dV are off by,
    against that of the roundings that there have to be: P and P * (dO.V^T - delta) to fp16, as they are without the softmax scale, and the results'."""
    L, scale = 2048, 1 / math.sqrt(d)
    blocks = layout(kind, L // bs)
    at = torch.arange(L, device="cuda")
    keep = (at[:, None] >= at[None, :]) if kind == "causal" else torch.ones(L, L, dtype=torch.bool, device="cuda")
    lay = plan(sfb, blocks, bs, keep[None].cpu() if kind == "causal" else None)
    q, k, v, do = (x.cuda() for x in operands(1, L, 1, d, "f16", 40 + power))
    do = (do.float() * 2.0 ** power).half()
    o, lse = sfb.fused_attention_stats(q, k, v, lay, use_mask=kind == "causal")
    got = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay, use_mask=kind == "causal")
    q, k, v, do, o = (x[0, :, 0].double() for x in (q, k, v, do, o))
    x = scale * q @ k.t()
    p = torch.where(keep, (x - lse[0, 0].double()[:, None]).exp(), 0.0)
    e = p * (do @ v.t() - (do * o).sum(1)[:, None])
    want = scale * e @ k, scale * e.t() @ q, p.t() @ do
    ve, vp = rounding_variance(e), rounding_variance(p)
    spread = scale ** 2 * ve @ k.square(), scale ** 2 * ve.t() @ q.square(), vp.t() @ do.square()
    # fp32: the scores' d products and additions, the exponential and the sums, relative to the magnitudes as in grad_tolerance, of independent entries
    qk = float((q.abs() @ k.abs().t()).max())
    rel = 2.0 ** -23 * (scale * qk * (2 + d / 16) + 2 * float(lse.abs().max()) + 8 + d / 16 + L / 16) + 2.0 ** -22
    wide = p * (do.abs() @ v.abs().t() + (do * o).abs().sum(1)[:, None])
    loose = scale ** 2 * wide.square() @ k.square(), scale ** 2 * wide.square().t() @ q.square(), p.square().t() @ do.square()
    for name, a, w, s, l in zip(("dq", "dk", "dv"), got, want, spread, loose):
        off = float((a[0, :, 0].double() - w).norm())
        # 130000 entries and more: their norm is within some percent of the expected one; a quarter is allowed
        limit = 1.25 * math.sqrt(float(s.sum() + rounding_variance(w).sum())) + rel * math.sqrt(float(l.sum()))
        assert off <= limit, (name, off / float(w.norm()), limit / float(w.norm()))


@pytest.mark.parametrize("dtype,bs,d", [("f16", 64, 64), ("bf16", 64, 64), ("f16", 32, 64), ("bf16", 64, 40), ("f32", 32, 64)])
def test_softmax_scales_above_one(sfb, dtype, bs, d):
    check_attention(sfb, layout("stride", 4), bs, 1, 2, d, dtype, scale=1.5)


@pytest.mark.parametrize("dtype,bs,d", [("f16", 64, 64), ("bf16", 32, 64), ("f16", 64, 96), ("f32", 32, 64)])
@pytest.mark.parametrize("scale", [0.25, 3.0])
def test_a_negative_scale_is_that_of_negative_queries(sfb, dtype, bs, d, scale):
    nb = 4
    q, k, v, do = (x.cuda() for x in operands(1, nb * bs, 2, d, dtype, 21))
    lay = plan(sfb, layout("stride", nb), bs)
    o, lse = sfb.fused_attention_stats(q, k, v, lay, scale)
    a = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay, scale)
    b = sfb.attention_backward_recompute(-q, k, v, o, do, lse, lay, -scale)
    assert torch.equal(a[0], -b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("dtype,bs,d", [("f16", 64, 64), ("bf16", 32, 64), ("f32", 64, 64)])
def test_a_scale_of_zero(sfb, dtype, bs, d):
    """Every row is the mean of its values; dQ and dK are zeros."""
    nb = 3
    q, k, v, do = (x.cuda() for x in operands(1, nb * bs, 2, d, dtype, 22))
    lay = plan(sfb, layout("full", nb), bs)
    o, lse = sfb.fused_attention_stats(q, k, v, lay, 0.0)
    assert (lse - math.log(nb * bs)).abs().max() <= 2.0 ** -20
    dq, dk, dv = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay, 0.0)
    assert (dq == 0).all() and (dk == 0).all()
    want = do.double().sum(1, keepdim=True) / (nb * bs)
    size = do.double().abs().sum(1, keepdim=True) / (nb * bs)
    t = torch.finfo(DTYPES[dtype])
    # P: half a step; the sums as in grad_tolerance; the result's rounding
    assert ((dv.double() - want).abs() <= t.eps / 2 * want.abs() * 1.01 + ((t.eps / 2 if dtype != "f32" else 0) + 2.0 ** -18) * size + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype,bs,d", [("f16", 64, 64), ("bf16", 64, 64), ("bf16", 32, 40), ("f32", 32, 64)])
def test_log_sums_with_an_output_in_a_wider_tensor(sfb, dtype, bs, d):
    """Two heads of five: the neighbouring heads stay, the bits are those of a call without out."""
    nb, H = 5, 2
    q, k, v = (x.cuda() for x in operands(2, nb * bs, H, d, dtype, 23, n=3))
    lay = plan(sfb, layout("stride", nb), bs)
    want = sfb.fused_attention_stats(q, k, v, lay)
    wider = torch.full((2, nb * bs, 5, d), 7.0, dtype=DTYPES[dtype], device="cuda")
    o, lse = sfb.fused_attention_stats(q, k, v, lay, out=wider[:, :, 1:3])
    assert o.data_ptr() == wider[:, :, 1:3].data_ptr() and torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert (wider[:, :, :1] == 7).all() and (wider[:, :, 3:] == 7).all()
    grads = sfb.attention_backward_recompute(q, k, v, *want[:1], q, lse, lay)
    # gradients beside each other in rows that are wider still
    wide = torch.full((2, nb * bs, 4, H, d), 7.0, dtype=DTYPES[dtype], device="cuda")
    got = sfb.attention_backward_recompute(q, k, v, o, q, lse, lay, out=[wide[:, :, i] for i in (3, 0, 2)])
    for a, b in zip(grads, got):
        assert torch.equal(a, b)
    assert (wide[:, :, 1] == 7).all()


def test_differences_of_the_fp32_forward(sfb):
    """The gradient of <o, do> along a direction, by central differences of the package's own forward, without their second-order error."""
    bs, nb, d, H = 32, 5, 64, 2
    lay = plan(sfb, layout("stride", nb), bs)
    q, k, v, do = (x.cuda() for x in operands(1, nb * bs, H, d, "f32", 3))
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    grads = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
    for which in range(3):
        y = torch.randn(q.shape, generator=torch.Generator().manual_seed(9 + which)).cuda()

        def slope(eps):
            f = []
            for e in (eps, -eps):
                x = [q, k, v]
                x[which] = x[which] + e * y
                f.append(float((sfb.fused_attention_stats(*x, lay)[0].double() * do.double()).sum()))
            return (f[0] - f[1]) / (2 * eps)

        eps = 2.0 ** -6
        near, far = (4 * slope(eps) - slope(2 * eps)) / 3, (4 * slope(2 * eps) - slope(4 * eps)) / 3
        size = float((grads[which].double() * y.double()).abs().sum())
        # what is left of the differences goes with eps^4: a fifteenth of what the doubled step changes.  The forward's entries are off by 2^-20 of
        # the values' size (24 roundings of the scores and sums), independently, four times in a slope; the gradients by 1e-6
        noise = 4 * 2.0 ** -20 * float((do.double().square().sum() * v.double().square().mean()).sqrt()) / eps
        assert abs(near - float((grads[which].double() * y.double()).sum())) <= abs(near - far) / 15 * 2 + noise + 1e-6 * size


# ---- embedding ------------------------------------------------------------------------------------------------------------------
def test_a_position_table_longer_than_the_sequence(sfb):
    """Its first rows are added, as a view of them would be."""
    g = torch.Generator(device="cuda").manual_seed(25)
    table, pos = torch.randn(50, 16, device="cuda", generator=g), torch.randn(512, 16, device="cuda", generator=g)
    ids = torch.randint(0, 50, (3, 20), device="cuda", generator=g, dtype=torch.int32)
    want = sfb.embedding(table, ids, pos[:20].contiguous(), scale=2.0)[0]
    assert torch.equal(want, sfb.embedding(table, ids, pos, scale=2.0)[0])
    assert torch.equal(want, sfb.embedding(table, ids, pos[None, :20], scale=2.0)[0])


@pytest.mark.parametrize("B,L", [(0, 5), (3, 0), (0, 0)])
def test_a_lookup_of_no_tokens(sfb, B, L):
    """Its count is 0, whatever was in that memory before."""
    table, ids = torch.ones(9, 16, device="cuda"), torch.zeros(B, L, dtype=torch.int32, device="cuda")
    for _ in range(4):
        dirt = [torch.full((1,), 77, dtype=torch.int32, device="cuda") for _ in range(64)]
        del dirt
        out, bad = sfb.embedding(table, ids)
        assert out.shape == (B, L, 16) and int(bad) == 0


@pytest.mark.parametrize("n", [16383, 16384, 16385, 65535, 65536, 65537, 65541])
@pytest.mark.parametrize("off", [0, 1, 3])
@pytest.mark.parametrize("dtype,hidden", [("bf16", 8), ("f32", 24)])
def test_counts_of_ids_at_every_alignment(sfb, n, off, dtype, hidden):
    """One CTA counts, four ids per load where they are 16-byte aligned, or all that read them: on both sides of what decides, and ids that end inside a load."""
    vocab = 300
    g = torch.Generator(device="cuda").manual_seed(n)
    table = torch.randn(vocab, hidden, device="cuda", generator=g).to(DTYPES[dtype])
    flat = torch.full((n + 8,), -5, device="cuda", dtype=torch.int32)
    ids = flat[off:off + n].view(1, n)
    ids.copy_(torch.randint(-3, vocab + 3, (1, n), device="cuda", generator=g, dtype=torch.int32))
    for edge in ((0, -1), (n - 1, vocab), (n - 2, -2 ** 31)):
        ids[0, edge[0]] = edge[1]
    there = (ids >= 0) & (ids < vocab)
    for _ in range(2):
        out, bad = sfb.embedding(table, ids, scale=1.0)
        assert int(bad) == int((~there).sum())
        assert torch.equal(out, table[ids.clamp(0, vocab - 1).long()] * there[..., None])


def tokens(n, vocab, hidden, seed, B=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(-1, vocab + 1, (B, n // B), device="cuda", generator=g, dtype=torch.int32)
    return torch.randn(B, n // B, hidden, device="cuda", generator=g), ids


def test_tables_of_many_tokens_in_graphs_and_on_streams(sfb):
    """The three launches and their workspace: calls at once on two streams, captured, and replayed with other tokens in place."""
    vocab, hidden = 700, 96
    sets = [[x.clone() for x in tokens(4096, vocab, hidden, i, 4)] for i in range(2)]

    def step(dout, ids):
        return sfb.embedding_grad(dout, ids, vocab, 0.5, True)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for s, x in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([step(*x) for _ in range(4)][-1])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    graphs, outs = [], []
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*x))
        graphs.append(graph)
    for seed in range(3):
        for i, x in enumerate(sets):
            for y, z in zip(x, tokens(4096, vocab, hidden, 10 * seed + i, 4)):
                y.copy_(z)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, o in zip(sets, outs):
            for y, z in zip(o, step(*x)):
                assert torch.equal(y, z)
    check_embed_grad(sfb, sets[0][0].cpu(), sets[0][1].cpu(), vocab, 0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_many_tokens_whose_rows_are_not_finite(sfb, dtype):
    """They reach their own ids' and positions' rows only, beside others in their piece and over several pieces."""
    n, vocab, hidden = 5000, 60, 40
    ids = (torch.arange(n) % 50).to(torch.int32)
    ids[7::50], ids[9::50] = -1, vocab
    dout = torch.ones(n, hidden)
    dout[3], dout[77], dout[4999], dout[7], dout[59] = math.nan, math.inf, -math.inf, math.nan, math.inf      # 7, 59: ids that have no row
    dtable, dpos, bad = sfb.embedding_grad(dout.to(DTYPES[dtype]).view(1, n, hidden).cuda(), ids.view(1, n).cuda(), vocab, positions=True)
    assert int(bad) == 200
    assert dtable[3].isnan().all() and (dtable[27] == math.inf).all() and (dtable[49] == -math.inf).all()
    rest = [i for i in range(50) if i not in (3, 7, 9, 27, 49)]
    assert (dtable[rest] == 100).all() and (dtable[50:] == 0).all() and (dtable[[7, 9]] == 0).all()
    assert torch.equal(dpos.cpu().nan_to_num(5.0), dout.nan_to_num(5.0))


@pytest.mark.parametrize("n,piece", [(4096, 8), (65536, 16), (98304, 32), (196608, 64)])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_runs_at_the_ends_of_pieces(sfb, n, piece, shift):
    """Whole numbers, whose sums are exact: runs of one piece and of several, that end with a piece or beside its end, runs of up to 16 parts
    and of more, which a warp and a CTA add up, and a total that is a multiple of the piece."""
    parts = [1, 1, 2, 16, 17, 3, 33, 15]
    lengths = [shift] if shift else []
    while sum(lengths) < n:
        lengths += [p * piece for p in parts] + [piece // 2, piece // 2, 1, 16 * piece - 1, 17 * piece + 1, piece - 1]
    ids = torch.repeat_interleave(torch.arange(len(lengths)) * 2 + 1, torch.tensor(lengths))[:n]      # every other row has no token
    vocab, hidden = 2 * len(lengths) + 2, 24
    g = torch.Generator().manual_seed(n + shift)
    ids = ids[torch.randperm(n, generator=g)].to(torch.int32)
    dout = torch.randint(-8, 9, (n, hidden), generator=g)
    want = torch.zeros(vocab, hidden, dtype=torch.int64).index_add_(0, ids.long(), dout)
    for t in (torch.float32, torch.bfloat16):
        dtable, dpos, bad = sfb.embedding_grad(dout.to(t).view(2, n // 2, hidden).cuda(), ids.view(2, n // 2).cuda(), vocab, positions=True)
        assert int(bad) == 0
        assert torch.equal(dtable.cpu().long(), want)
        assert torch.equal(dpos.cpu().long(), dout.view(2, n // 2, hidden).sum(0))
    start = torch.randint(-8, 9, (vocab, hidden), generator=g).float().cuda()
    added, _, _ = sfb.embedding_grad(dout.float().view(1, n, hidden).cuda(), ids.view(1, n).cuda(), vocab, out=start.clone())
    assert torch.equal(added.cpu().long(), want + start.cpu().long())


# ---- threads ----------------------------------------------------------------------------------------------------------------------
def test_calls_from_several_threads(sfb):
    """Each thread on a stream of its own, all of them at once (a call lets other threads run while it launches): the bits of calls one by one."""
    import threading
    bs, nb, n = 64, 6, 4
    lay = plan(sfb, layout("stride", nb), bs)
    lay.tn_lut
    sets = []
    for i in range(n):
        dtype = ("f16", "bf16", "f32", "f16")[i]
        dout, ids = tokens(3000 if i % 2 else 300, 200, 64, 60 + i)
        grads = [torch.randn(7000 + i, device="cuda"), torch.randn(33, 5, device="cuda")]
        sets.append(([x.cuda() for x in operands(2, nb * bs, 3, 64, dtype, 50 + i)], dout, ids, grads))

    def step(x, dout, ids, grads):
        q, k, v, do = x
        o, lse = sfb.fused_attention_stats(q, k, v, lay)
        out = [torch.empty_like(g) for g in grads]
        norm = sfb.clip_grad_norm(grads, 1.0, out=out)
        return (o, lse, norm, *out, *sfb.attention_backward_recompute(q, k, v, o, do, lse, lay), *sfb.embedding_grad(dout, ids, 200, positions=True))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got, errors = [None] * n, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = step(*sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                               # reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
