"""The operators of a training step around the attention where the tests beside this file do not reach."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_training import check_attention, layout, operands, plan                                            # noqa: E402
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
