"""The operators of a training step around the attention against their definitions in 64 bits (training_reference.py), at the sizes, masks
and layouts where they can go wrong."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from training_reference import DTYPES, attend, attend_grad, blocks_to_elements, embed_grad, grad_tolerance, half_step, pack_bits   # noqa: E402


def layout(kind, nb, heads=1, seed=0):
    i, j = np.arange(nb)[:, None], np.arange(nb)[None, :]
    if kind == "full":
        keep = np.ones((nb, nb), bool)
    elif kind == "causal":
        keep = j <= i
    elif kind == "stride":
        keep = ((j <= i) & (j + 2 > i)) | (j % 4 == 0)
    elif kind == "local":
        keep = (j + 1 >= i) & (j <= i + 1)
    elif kind == "holes":                                   # rows and columns without blocks, pairs that are half empty
        keep = (i % 3 != 1) & (j % 4 != 2) & ((i + 2 * j) % 5 < 2)
        keep[0, 0] = True
    elif kind == "long":                                    # one row and one column with every block, little else
        keep = (i == nb - 1) | (j == nb // 2) | (i == j)
    elif kind == "random":
        keep = np.random.RandomState(seed).rand(nb, nb) < 0.3
        keep[0, 0] = True
    elif kind == "heads":                                   # equally many blocks per head
        return np.stack([(j == (i + h) % nb) | (j == i) if h % nb else (j == (i + 1) % nb) | (j == i) for h in range(heads)]).astype(np.uint8)
    return keep[None].astype(np.uint8)


def plan(sfb, blocks, bs, keep=None):
    lay = sfb.BlockLayout(torch.from_numpy(blocks).cuda(), bs)
    if keep is not None:
        lay.mask_np = pack_bits(keep, blocks, bs).cuda()
    return lay


def operands(B, L, H, d, dtype, seed, packed=False, n=4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, n, H, d, generator=g).to(DTYPES[dtype])
    return [x[:, :, i] if packed else x[:, :, i].contiguous() for i in range(n)]


def check_attention(sfb, blocks, bs, B, H, d, dtype, keep=None, packed=False, scale=None, seed=0, odd_base=False):
    """Forward and backward through the package against 64 bits; returns what the package gave."""
    t = DTYPES[dtype]
    L = blocks.shape[1] * bs
    scale = 1 / math.sqrt(d) if scale is None else scale
    elements = blocks_to_elements(blocks, bs)
    if keep is not None:
        elements = elements & keep
    lay = plan(sfb, blocks, bs, elements if keep is not None else None)
    q, k, v, do = operands(B, L, H, d, dtype, seed, packed)
    if packed:
        x = torch.stack([q, k, v], 2).cuda()
        dq_, dk_, dv_ = x[:, :, 0], x[:, :, 1], x[:, :, 2]
        into = torch.full_like(x, 7.0)
        out = [into[:, :, i] for i in range(3)]
    elif odd_base:                                          # one element off every alignment
        def shift(a):
            flat = torch.empty(a.numel() + 1, dtype=t, device="cuda")
            flat[1:] = a.flatten().cuda()
            return flat[1:].view(a.shape)
        dq_, dk_, dv_ = (shift(a) for a in (q, k, v))
        out = None
    else:
        dq_, dk_, dv_ = (a.cuda() for a in (q, k, v))
        out = None
    dod = do.cuda()
    o, lse = sfb.fused_attention_stats(dq_, dk_, dv_, lay, scale, use_mask=keep is not None)
    assert o.dtype == t and lse.dtype == torch.float32 and o.shape == q.shape and lse.shape == (B, H, L)
    qk = float(torch.einsum("blhd,bmhd->bhlm", q.double().abs(), k.double().abs()).max())
    want_o, want_l = attend(q, k, v, elements, scale)
    empty = want_l == -math.inf
    assert torch.equal((lse == -math.inf).cpu(), empty)
    got = lse.cpu().double()[~empty]
    # log2-scores off as in grad_tolerance, the sum of the powers by its roundings, the result by one
    top = float(want_l[~empty].abs().max()) if got.numel() else 0.0
    e = 2.0 ** -23 * (scale * qk * (2 + d / 16) + 2 * top + 4 + L / 64) + 2.0 ** -21
    assert (got - want_l[~empty]).abs().max().item() <= e if got.numel() else True
    h = half_step(t)
    size = torch.einsum("bhlm,bmhd->blhd", torch.where(empty[..., None], 0.0, (scale * torch.einsum("blhd,bmhd->bhlm", q.double(), k.double())).masked_fill(
        ~elements[None], -math.inf).sub(torch.where(empty, 0.0, want_l)[..., None]).exp()), v.double().abs())
    # 16 bits: every power half a step off, and the sum of the powers as they were
    tol = h * want_o.abs() + (2 * e + 2.0 ** -23 * (8 + L / 16)) * size + (h * size if dtype != "f32" else 0) + (2.0 ** -25 * L if dtype == "f16" else 0) + 1e-30
    assert ((o.cpu().double() - want_o).abs() <= tol).all()
    assert (o.cpu()[empty.transpose(1, 2)] == 0).all()

    grads = sfb.attention_backward_recompute(dq_, dk_, dv_, o, dod, lse, lay, scale, use_mask=keep is not None, out=out)
    again = sfb.attention_backward_recompute(dq_, dk_, dv_, o, dod, lse, lay, scale, use_mask=keep is not None)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)                            # the same bits, wherever they are written
    if packed:
        assert grads[0].data_ptr() == into.data_ptr()
    oc, lc = o.cpu(), lse.cpu()
    want, sizes, loose = attend_grad(q, k, v, oc, do, lc, elements, scale)
    tols = grad_tolerance(want, sizes, loose, t, lc, d, L, scale, qk)
    for name, a, w, tol in zip(("dq", "dk", "dv"), grads, want, tols):
        off = (a.cpu().double() - w).abs()
        assert (off <= tol).all(), (name, float((off / tol).max()))
        assert a.dtype == t and a.shape == q.shape
    # rows and columns that keep nothing
    assert (grads[0].cpu()[empty.transpose(1, 2)] == 0).all()
    none = ~elements.any(1)
    none = none.expand(H, L) if none.shape[0] == 1 else none
    for a in grads[1:]:
        assert (a.cpu().permute(2, 1, 0, 3)[none] == 0).all()
    assert sfb.device_status() == 0
    return (dq_, dk_, dv_, dod, lay), (o, lse), grads


SHAPES = [(64, 64, "f16"), (64, 64, "bf16"), (32, 64, "bf16"), (64, 128, "f16"), (32, 32, "f32"), (32, 64, "f32"), (64, 64, "f32"), (64, 128, "f32"), (32, 40, "f16"),
          (32, 7, "f32"), (64, 1, "f32"), (64, 33, "bf16")]


@pytest.mark.parametrize("bs,d,dtype", SHAPES)
@pytest.mark.parametrize("kind,nb", [("full", 1), ("full", 5), ("causal", 4), ("stride", 8), ("local", 7), ("holes", 9), ("long", 6), ("random", 8)])
def test_attention(sfb, kind, nb, bs, d, dtype):
    check_attention(sfb, layout(kind, nb), bs, 2, 3, d, dtype, seed=nb)


@pytest.mark.parametrize("bs,d,dtype", SHAPES[:7])
def test_a_pattern_per_head(sfb, bs, d, dtype):
    check_attention(sfb, layout("heads", 6, 4), bs, 2, 4, d, dtype)


def ragged(L, valid):
    at = torch.arange(L)
    return ((at[:, None] < valid) & (at[None, :] < valid))[None]


@pytest.mark.parametrize("bs,d,dtype", SHAPES[:8])
@pytest.mark.parametrize("mask", ["causal", "ragged", "one", "nothing", "random", "last bit"])
def test_element_masks(sfb, mask, bs, d, dtype):
    nb = 5
    L = nb * bs
    at = torch.arange(L)
    keep = {"causal": (at[:, None] >= at[None, :])[None], "ragged": ragged(L, 3 * bs + 11), "one": ragged(L, 1), "nothing": torch.zeros(1, L, L, dtype=torch.bool),
            "random": torch.rand(1, L, L, generator=torch.Generator().manual_seed(3)) < 0.05,
            "last bit": ((at[None, :] % bs == bs - 1) & (at[:, None] % 2 == 0))[None]}[mask]
    check_attention(sfb, layout("causal" if mask == "causal" else "full", nb), bs, 2, 2, d, dtype, keep=keep)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_mask_per_head(sfb, dtype):
    bs, nb, H = 64, 4, 3
    keep = torch.rand(H, nb * bs, nb * bs, generator=torch.Generator().manual_seed(5)) < 0.3
    check_attention(sfb, np.repeat(layout("full", nb), H, 0), bs, 2, H, 64, dtype, keep=keep)


@pytest.mark.parametrize("bs,d,dtype", SHAPES)
def test_slices_of_packed_tensors(sfb, bs, d, dtype):
    check_attention(sfb, layout("stride", 5), bs, 2, 2, d, dtype, packed=True)


@pytest.mark.parametrize("bs,d,dtype", [(64, 64, "f16"), (64, 64, "bf16"), (32, 64, "f16"), (64, 64, "f32")])
def test_bases_that_are_not_aligned(sfb, bs, d, dtype):
    check_attention(sfb, layout("stride", 5), bs, 2, 2, d, dtype, odd_base=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("scale", [1.0, 0.02])
def test_scales(sfb, dtype, scale):
    """Scores of up to about 30, and ones that are all alike."""
    check_attention(sfb, layout("stride", 6), 64, 1, 2, 64, dtype, scale=scale)


def test_the_forward_is_the_one_without_sums(sfb):
    for dtype, bs, d in (("f16", 64, 64), ("bf16", 64, 64), ("f32", 32, 64), ("f16", 32, 40)):
        for kind, nb in (("stride", 16), ("full", 4)):
            q, k, v = (x.cuda() for x in operands(2, nb * bs, 4, d, dtype, 1, n=3))
            lay = plan(sfb, layout(kind, nb), bs)
            assert torch.equal(sfb.fused_attention_stats(q, k, v, lay)[0], sfb.fused_attention(q, k, v, lay))


def test_the_gradient_is_the_one_from_saved_probabilities(sfb):
    """Beside attention_backward_fused, which reads P in 16 bits where this one makes dS of an unrounded one."""
    bs, nb, d = 64, 16, 64
    q, k, v, do = (x.cuda() for x in operands(2, nb * bs, 4, d, "f16", 2))
    lay = plan(sfb, layout("stride", nb), bs)
    p = sfb.fused_sddmm_softmax(q, k, lay, 0.125, torch.float16)
    o, lse = sfb.fused_attention_stats(q, k, v, lay, 0.125)
    a = sfb.attention_backward_fused(q, k, v, p, sfb.bst_sgemm_xn(p, v, lay), do, lay, 0.125)
    b = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay, 0.125)
    for x, y in zip(a, b):
        # half a step each of P, dS and the result, and O's in delta, on sums of a few dozen entries
        assert (x.float() - y.float()).norm() <= 4 * 2.0 ** -11 * x.float().norm()


def test_differences(sfb):
    """The gradient of <o, do> along a direction, by central differences of the fp32 forward."""
    bs, nb, d, H = 32, 5, 64, 2
    blocks = layout("stride", nb)
    lay = plan(sfb, blocks, bs)
    q, k, v, do = (x.cuda() for x in operands(1, nb * bs, H, d, "f32", 3))
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    grads = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
    dirs = [torch.randn(q.shape, generator=torch.Generator().manual_seed(9 + i)).cuda() for i in range(3)]
    keep = blocks_to_elements(blocks, bs)

    def value(eps):
        out, _ = attend(*((x.double() + eps * y.double()).cpu() for x, y in zip((q, k, v), dirs)), keep, 1 / math.sqrt(d))
        return float((out * do.cpu().double()).sum())

    eps = 1e-4
    num, ana = (value(eps) - value(-eps)) / (2 * eps), sum(float((g.double() * y.double()).sum()) for g, y in zip(grads, dirs))
    # third derivatives times eps^2, and fp32 gradients: 1e-6 of the sum of the magnitudes
    size = sum(float((g.double() * y.double()).abs().sum()) for g, y in zip(grads, dirs))
    assert abs(num - ana) <= 1e-5 * size


def test_one_tensor_as_q_k_and_v(sfb):
    bs, nb = 64, 4
    x = operands(2, nb * bs, 2, 64, "bf16", 4, n=1)[0].cuda()
    lay = plan(sfb, layout("full", nb), bs)
    do = torch.ones_like(x)
    o, lse = sfb.fused_attention_stats(x, x, x, lay)
    a = sfb.attention_backward_recompute(x, x, x, o, do, lse, lay)
    o2, lse2 = sfb.fused_attention_stats(x, x.clone(), x.clone(), lay)
    b = sfb.attention_backward_recompute(x, x.clone(), x.clone(), o2, do, lse2, lay)
    for y, z in zip(a, b):
        assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("bs,d", [(32, 8), (32, 72), (32, 96), (32, 100), (32, 126), (32, 128), (64, 16), (64, 48), (64, 96), (64, 104), (64, 127)])
def test_widths_of_the_general_path(sfb, bs, d, dtype):
    """Head sizes in every number of 32 columns, whole and not, with rows that can be read 16 bytes at a time and ones that cannot."""
    check_attention(sfb, layout("long", 5), bs, 2, 3, d, dtype, seed=d)
    at = torch.arange(5 * bs)
    check_attention(sfb, layout("causal", 5), bs, 1, 2, d, dtype, keep=(at[:, None] >= at[None, :])[None], packed=True, seed=d)


@pytest.mark.parametrize("bs,d", [(32, 40), (64, 128)])
def test_fp32_operands_whose_first_bf16_number_is_infinite(sfb, bs, d):
    """The largest fp32 number rounds to infinity in bf16: products of terms are NaN, the sum is not."""
    nb, big = 3, 3.4e38
    q, k, v, do = operands(1, nb * bs, 1, d, "f32", 4)
    do = do * 0
    do[0, 5, 0, 1], do[0, bs + 3, 0, 2], v = big, -big, v * 0
    blocks = layout("full", nb)
    lay = plan(sfb, blocks, bs)
    cuda = [x.cuda() for x in (q, k, v, do)]
    o, lse = sfb.fused_attention_stats(*cuda[:3], lay)
    dq, dk, dv = sfb.attention_backward_recompute(*cuda[:3], o, cuda[3], lse, lay)
    assert (dq == 0).all() and (dk == 0).all()
    scale = 1 / math.sqrt(d)
    want = attend_grad(q, k, v, o.cpu(), do, lse.cpu(), torch.ones(1, nb * bs, nb * bs, dtype=torch.bool), scale)[0][2]
    qk = float(torch.einsum("blhd,bmhd->bhlm", q.double().abs(), k.double().abs()).max())
    top = float(lse.abs().max())
    # P as in grad_tolerance; a sum of one product, rounded
    e = 2.0 ** -23 * (scale * qk * (2 + d / 16) + 2 * top + 4) + 2.0 ** -22 + 2.0 ** -23
    assert torch.isfinite(dv).all()
    assert ((dv.cpu().double() - want).abs() <= e * want.abs() + 1e-30).all()


def test_a_layout_of_no_blocks_but_one(sfb):
    blocks = np.zeros((1, 6, 6), np.uint8)
    blocks[0, 3, 2] = 1
    for bs, d, dtype in ((64, 64, "f16"), (32, 64, "f32")):
        check_attention(sfb, blocks, bs, 1, 2, d, dtype)


def test_infinities_outside_the_kept_blocks(sfb):
    """Positions that no kept block touches may hold anything."""
    bs, nb = 64, 6
    blocks = np.zeros((1, nb, nb), np.uint8)
    blocks[0, :4, :4] = np.tril(np.ones((4, 4)))
    for dtype, d, size in (("f16", 64, 64), ("f32", 64, 32), ("bf16", 32, 32)):
        lay = plan(sfb, blocks, size)
        xs = [x.cuda() for x in operands(1, nb * size, 2, d, dtype, 6)]
        clean = [x.clone() for x in xs]
        for i, x in enumerate(xs):
            x[:, 4 * size:] = [math.inf, math.nan, -math.inf, math.nan][i]
        res = []
        for q, k, v, do in (xs, clean):
            o, lse = sfb.fused_attention_stats(q, k, v, lay)
            o[:, 4 * size:] = 0                                  # the forward's zeros, or what a caller left there
            res.append((o, lse) + sfb.attention_backward_recompute(q, k, v, o, do, lse, lay))
        for a, b in zip(*res):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bs,d,dtype", [(64, 64, "f16"), (32, 40, "bf16"), (64, 128, "f16"), (32, 64, "f32")])
def test_streams_graphs_and_two_calls_at_once(sfb, bs, d, dtype):
    nb = 8
    lay = plan(sfb, layout("stride", nb), bs)
    lay.tn_lut
    sets = [[x.cuda() for x in operands(2, nb * bs, 4, d, dtype, 10 + i)] for i in range(2)]

    def step(q, k, v, do):
        o, lse = sfb.fused_attention_stats(q, k, v, lay)
        return (o, lse) + sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, x in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([step(*x) for _ in range(4)][-1])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    # two captured steps, replayed on two streams
    graphs, outs = [], []
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*x))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_long_rows_of_many_blocks(sfb):
    """More key blocks than the tensor-core kernels' lists hold: 300 blocks in a row."""
    bs, nb = 64, 300
    blocks = np.zeros((1, nb, nb), np.uint8)
    blocks[0, np.arange(nb), np.arange(nb)] = 1
    blocks[0, 5] = 1
    blocks[0, :, 7] = 1
    lay = plan(sfb, blocks, bs)
    q, k, v, do = (x.cuda() for x in operands(1, nb * bs, 1, 64, "f16", 7))
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    grads = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
    f = [x.float() for x in (q, k, v, do)]
    lay32 = lay
    o32, lse32 = sfb.fused_attention_stats(f[0], f[1], f[2], lay32)
    want = sfb.attention_backward_recompute(f[0], f[1], f[2], o.float(), f[3], lse32, lay32)
    assert (lse - lse32).abs().max() <= 1e-4
    for a, b in zip(grads, want):
        assert (a.float() - b).norm() <= 3 * 2.0 ** -11 * b.norm()
    assert sfb.device_status() == 0


@pytest.mark.parametrize("B,H,heads", [(3, 40, 1), (2, 100, 1), (1, 130, 130), (5, 40, 1), (7, 43, 1), (1, 310, 310)])
def test_more_heads_than_go_through_the_workspace_at_once(sfb, B, H, heads):
    """Whole batch elements at a time, and some heads of one: the same bits as calls for a few heads each, in place."""
    bs, nb, d = 32, 64, 8
    i, j = np.arange(nb)[:, None], np.arange(nb)[None, :]
    blocks = np.stack([(i == j) | (j == (i + 1 + h % 5) % nb) for h in range(heads)]).astype(np.uint8)
    q, k, v, do = (x.cuda() for x in operands(B, nb * bs, H, d, "f32", 13))
    lay = plan(sfb, blocks, bs)
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    whole = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
    for h0 in range(0, H, 37):
        h1 = min(H, h0 + 37)
        part = plan(sfb, blocks[h0:h1] if heads > 1 else blocks, bs)
        cut = [x[:, :, h0:h1] for x in (q, k, v, o, do)]
        got = sfb.attention_backward_recompute(*cut, lse[:, h0:h1].contiguous(), part)
        for a, b in zip(got, whole):
            assert torch.equal(a, b[:, :, h0:h1])


@pytest.mark.parametrize("flip", [False, True])
@pytest.mark.parametrize("nb", [2, 13, 33, 64])
def test_heads_in_groups(sfb, nb, flip):
    """Rows that grow from one end to the other: the same bits as calls for one batch element or a few heads, whichever group they are in."""
    B, H, bs, d = 3, 61, 64, 64
    blocks = np.ascontiguousarray(layout("causal", nb)[:, ::-1, ::-1] if flip else layout("causal", nb))
    if nb == 64:
        B, H = 2, 23
    q, k, v, do = (x.cuda() for x in operands(B, nb * bs, H, d, "bf16", 14))
    lay = plan(sfb, blocks, bs)
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    whole = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
    for b in range(B):
        for h0 in range(0, H, 7):
            h1 = min(H, h0 + 7)
            cut = [x[b:b + 1, :, h0:h1] for x in (q, k, v, o, do)]
            got = sfb.attention_backward_recompute(*cut, lse[b:b + 1, h0:h1].contiguous(), lay)
            for x, y in zip(got, whole):
                assert torch.equal(x, y[b:b + 1, :, h0:h1])
    assert sfb.device_status() == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["diagonal", "two", "three", "mixed", "empty rows"])
def test_many_short_rows(sfb, dtype, kind):
    """Dozens of row pairs (column pairs) per CTA, most of them with one to three steps: against the fp32 path."""
    bs, nb, B, H = 64, 64, 3, 12
    i, j = np.arange(nb)[:, None], np.arange(nb)[None, :]
    blocks = {"diagonal": i == j, "two": (i == j) | (j == (i ^ 1)), "three": (j >= i) & (j <= i + 1), "mixed": (j >= i) & (j <= i + i % 5) | (i == 40),
              "empty rows": (i == j) & (i % 7 < 3)}[kind][None].astype(np.uint8)
    lay = plan(sfb, blocks, bs)
    q, k, v, do = (x.cuda() for x in operands(B, nb * bs, H, 64, dtype, 12))
    o, lse = sfb.fused_attention_stats(q, k, v, lay)
    want = sfb.attention_backward_recompute(q.float(), k.float(), v.float(), o.float(), do.float(), lse, lay)
    for _ in range(3):
        got = sfb.attention_backward_recompute(q, k, v, o, do, lse, lay)
        assert sfb.device_status() == 0
        for a, b in zip(got, want):
            # half a step each of P, dS and the result, block by block of 64 positions and a head
            off, size = ((x.view(B, nb, bs, H, 64).square().sum((2, 4)).sqrt()) for x in (a.float() - b, b))
            assert (off <= 3 * half_step(DTYPES[dtype]) * size).all(), float((off / size).max())


# ---- embedding ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,L,hidden,scale,pos", [(1, 1, 8, 32.0, False), (3, 77, 768, 27.7, True), (5, 9, 264, -0.5, True), (64, 1, 1024, 32.0, False)])
def test_scaled_embedding(sfb, dtype, B, L, hidden, scale, pos):
    t, g = DTYPES[dtype], torch.Generator().manual_seed(1)
    vocab = 501
    table = torch.randn(vocab, hidden, generator=g).to(t)
    p = torch.randn(L, hidden, generator=g).to(t) if pos else None
    ids = torch.randint(-1, vocab + 1, (B, L), generator=g, dtype=torch.int32)
    there = (ids >= 0) & (ids < vocab)
    want = torch.where(there[..., None], scale * table.double()[ids.clamp(0, vocab - 1).long()], 0.0)
    size = want.abs()
    if pos:
        want, size = want + p.double(), size + p.double().abs()
    out, bad = sfb.embedding(table.cuda(), ids.cuda(), p.cuda() if pos else None, scale=scale)
    assert int(bad) == int((~there).sum())
    # scale is rounded to fp32, the sum once in fp32 and once to the type
    off = (out.cpu().double() - want).abs()
    assert (off <= half_step(t) * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -23 * size + (2.0 ** -25 if dtype == "f16" else 0)).all()


def check_embed_grad(sfb, dout, ids, vocab, scale=1.0, grad="f32", positions=True, out=None):
    t, g = dout.dtype, DTYPES[grad] if grad else dout.dtype
    start = [x.clone().cpu().double() for x in out] if out else None
    args = dict(scale=scale, positions=positions, dtype=g)
    if out:
        args["out"] = tuple(out) if positions else out[0]
    dtable, dpos, bad = sfb.embedding_grad(dout.cuda(), ids.cuda(), vocab, **args)
    want, wpos, size, spos = embed_grad(dout, ids, vocab, scale)
    assert int(bad) == int(((ids < 0) | (ids >= vocab)).sum())
    for got, w, s, k in ((dtable, want, size, 0), (dpos, wpos, spos, 1)):
        if got is None:
            assert not positions
            continue
        if start:
            w, s = w + start[k], s + start[k].abs()
        # each of the additions rounds in fp32: at most a share of 2^-24 of the magnitudes per level.  A piece has up to 64 tokens (few tokens: a warp up to
        # 128), 16 parts are added up in turn or by eight warps; of a run of very many parts the roundings' signs differ, and less is allowed than their worst
        tol = half_step(g) * w.abs() + 2.0 ** -24 * (128 + ids.numel() / 128 / 8 + 16) * s + (2.0 ** -25 if g == torch.float16 else 0)
        off = (got.cpu().double() - w).abs()
        assert (off <= tol).all(), float((off / (tol + 1e-300)).max())
        assert got.dtype == g
        assert (got.cpu()[(s == 0).all(1)] == 0).all()
    if not out:
        again = sfb.embedding_grad(dout.cuda(), ids.cuda(), vocab, **args)
        assert torch.equal(again[0], dtable) and (dpos is None or torch.equal(again[1], dpos))
    return dtable, dpos


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,L,vocab,hidden", [(1, 1, 1, 8), (1, 1, 30522, 768), (2, 33, 7, 40), (3, 77, 1000, 264), (7, 129, 131, 1032), (64, 1, 50, 768), (130, 3, 5, 16),
                                              (1, 4099, 200000, 8), (33, 65, 2, 520)])
@pytest.mark.parametrize("grad", ["f32", None])
def test_embedding_grad(sfb, dtype, B, L, vocab, hidden, grad):
    g = torch.Generator().manual_seed(B + L)
    dout = torch.randn(B, L, hidden, generator=g).to(DTYPES[dtype])
    ids = torch.randint(-1, vocab + 1, (B, L), generator=g, dtype=torch.int32)
    check_embed_grad(sfb, dout, ids, vocab, 2.5, grad, positions=L % 2 == 1)


@pytest.mark.parametrize("what", ["one id", "all missing", "two ids", "text", "sorted", "descending", "beyond"])
def test_runs_of_ids(sfb, what):
    """Runs that fill pieces exactly, cross several, begin and end in them; 70000 tokens: longer pieces."""
    for B, L in ((3, 128), (1, 31), (2, 50), (7, 10007)):
        n, vocab, hidden = B * L, 300, 24
        g = torch.Generator().manual_seed(n)
        ids = {"one id": torch.full((n,), 7), "all missing": torch.full((n,), -1), "two ids": torch.randint(0, 2, (n,), generator=g) * 299,
               "text": (300 ** torch.rand(n, generator=g)).long().clamp_max(299), "sorted": torch.arange(n) * 300 // n, "descending": 299 - torch.arange(n) * 300 // n,
               "beyond": torch.where(torch.arange(n) % 3 == 0, 2 ** 31 - 1, -2 ** 31)}[what].to(torch.int32).view(B, L)
        dout = torch.randn(B, L, hidden, generator=g)
        check_embed_grad(sfb, dout.bfloat16() if B == 7 else dout, ids, vocab)


@pytest.mark.parametrize("B,L,vocab,hidden,dtype", [(1, 2048, 700, 256, "bf16"), (1, 2049, 700, 256, "bf16"), (2, 213, 3000, 768, "f32"), (2, 214, 3000, 768, "f32"),
                                                     (1, 100, 200000, 8, "f16"), (5, 64, 9000, 2048, "f16"), (40, 16, 63, 64, "f32"), (300, 1, 77, 520, "bf16")])
@pytest.mark.parametrize("what", ["any", "one id", "last rows", "all missing"])
def test_few_tokens(sfb, B, L, vocab, hidden, dtype, what):
    """Numbers of tokens on both sides of what one launch takes, new gradients and added ones."""
    g = torch.Generator().manual_seed(B * L)
    ids = {"any": torch.randint(-1, vocab + 1, (B, L), generator=g), "one id": torch.full((B, L), vocab // 2), "last rows": vocab - 1 - torch.randint(0, 3, (B, L), generator=g),
           "all missing": torch.full((B, L), vocab)}[what].to(torch.int32)
    dout = torch.randn(B, L, hidden, generator=g).to(DTYPES[dtype])
    for grad in ("f32", None):
        check_embed_grad(sfb, dout, ids, vocab, -1.5, grad)
        t = torch.float32 if grad else DTYPES[dtype]
        out = [torch.randn(vocab, hidden, generator=g).to(t).cuda(), torch.randn(L, hidden, generator=g).to(t).cuda()]
        check_embed_grad(sfb, dout, ids, vocab, -1.5, grad, out=out)


@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("f16", None), ("bf16", None)])
def test_gradients_added_to_a_tied_tables(sfb, dtype, grad):
    g = torch.Generator().manual_seed(2)
    dout = torch.randn(4, 50, 72, generator=g).to(DTYPES[dtype])
    ids = torch.randint(0, 90, (4, 50), generator=g, dtype=torch.int32)
    t = DTYPES[grad] if grad else DTYPES[dtype]
    out = [torch.randn(100, 72, generator=g).to(t).cuda(), torch.randn(50, 72, generator=g).to(t).cuda()]
    before = out[0].clone()
    dtable, dpos = check_embed_grad(sfb, dout, ids, 100, 0.5, grad, out=out)
    assert dtable.data_ptr() == out[0].data_ptr() and dpos.data_ptr() == out[1].data_ptr()
    assert torch.equal(out[0][90:], before[90:])
    check_embed_grad(sfb, dout, ids, 100, 0.5, grad, positions=False, out=out[:1])


def test_embedding_grad_of_no_tokens(sfb):
    dtable, dpos, bad = sfb.embedding_grad(torch.zeros(0, 5, 16, device="cuda"), torch.zeros(0, 5, dtype=torch.int32, device="cuda"), 9, positions=True)
    assert (dtable == 0).all() and dtable.shape == (9, 16) and (dpos == 0).all() and dpos.shape == (5, 16) and int(bad) == 0


def test_embedding_grad_of_rows_that_are_not_finite(sfb):
    """They reach their own rows only."""
    dout = torch.ones(2, 40, 16)
    dout[0, 3] = math.nan
    dout[1, 39] = math.inf
    ids = torch.arange(80, dtype=torch.int32).view(2, 40) % 20
    dtable, dpos, _ = sfb.embedding_grad(dout.cuda(), ids.cuda(), 30, positions=True)
    assert dtable[3].isnan().all() and (dtable[19] == math.inf).all()
    rest = [i for i in range(20) if i not in (3, 19)]
    assert (dtable[rest] == 4).all() and (dtable[20:] == 0).all()
    assert dpos[3].isnan().all() and (dpos[39] == math.inf).all() and (dpos[[i for i in range(40) if i not in (3, 39)]] == 2).all()


def test_few_tokens_in_graphs(sfb):
    """The one-launch form captured and replayed with other ids and other gradients in place."""
    vocab, hidden = 500, 96
    dout = torch.zeros(3, 20, hidden, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(3, 20, dtype=torch.int32, device="cuda")
    sfb.embedding_grad(dout, ids, vocab, 2.0, True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dtable, dpos, bad = sfb.embedding_grad(dout, ids, vocab, 2.0, True)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        dout.copy_(torch.randn(3, 20, hidden, generator=gen).bfloat16())
        ids.copy_(torch.randint(-1, vocab, (3, 20), generator=gen, dtype=torch.int32))
        g.replay()
        for a, b in zip((dtable, dpos, bad), sfb.embedding_grad(dout, ids, vocab, 2.0, True)):
            assert torch.equal(a, b)
        check_embed_grad(sfb, dout.cpu(), ids.cpu(), vocab, 2.0)


# ---- norm and clipping ------------------------------------------------------------------------------------------------------------
def norm64(grads, scale=1.0):
    return scale * math.sqrt(sum(float(x.double().square().sum()) for x in grads))


def check_clip(sfb, grads, max_norm, scale=1.0, out=None):
    norm = norm64(grads, scale)
    factor = scale * min(1.0, max_norm / (norm + 1e-6))
    want = [x.double() * factor for x in grads]
    got = sfb.clip_grad_norm(grads, max_norm, scale=scale, out=out)
    # fp64 sums: the norm's rounding to fp32; max_norm and scale are rounded to fp32, so is the factor
    assert got.shape == (1,) and abs(float(got) - norm) <= 2.0 ** -23 * norm + 1e-45
    for x, w in zip(out or grads, want):
        sub = 2.0 ** -25 if x.dtype == torch.float16 else 1e-44
        assert ((x.double() - w).abs() <= (half_step(x.dtype) + 2.0 ** -22) * w.abs() + sub).all()


def some(shapes, dtype, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(size * torch.randn(s, device="cuda", generator=g)).to(DTYPES[dtype]) for s in shapes]


SIZES = [(1,), (7,), (8, 16), (0,), (3, 5, 7), (16384,), (16385,), (2, 50001), (1000, 257)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("max_norm", [1.0, 1e9, 0.0, math.inf])
def test_clip_in_place(sfb, dtype, max_norm):
    grads = some(SIZES, dtype)
    assert abs(float(sfb.grad_norm(grads)) - norm64(grads)) <= 2.0 ** -23 * norm64(grads)
    check_clip(sfb, grads, max_norm)


@pytest.mark.parametrize("dtype,into", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_clip_into_others(sfb, dtype, into):
    grads = some(SIZES, dtype, 1, 100.0)
    kept = [x.clone() for x in grads]
    out = [torch.full(x.shape, 9.0, dtype=DTYPES[into], device="cuda") for x in grads]
    check_clip(sfb, grads, 2.0, 1 / 1024, out)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    check_clip(sfb, grads, 1e6, 0.5, out)


def test_views_of_one_buffer_at_every_alignment(sfb):
    for dtype in ("f32", "bf16", "f16"):
        sizes = [1, 2, 3, 5, 17, 33, 16400, 7, 1, 40001, 9]
        flat = some([(sum(sizes),)], dtype, 3)[0]
        master = torch.empty(sum(sizes) + 3, device="cuda")[3:]
        check_clip(sfb, list(flat.split(sizes)), 0.5, 1.0, list(master.split(sizes)))
        before = flat.clone()
        check_clip(sfb, list(flat.split(sizes))[::2], 0.5)
        parts, old = flat.split(sizes), before.split(sizes)
        assert all(torch.equal(a, b) for a, b in zip(parts[1::2], old[1::2]))          # the neighbours stay


def test_clip_of_types_together_and_many_tensors(sfb):
    grads = some([(i % 7 + 1, 3) for i in range(900)], "f32") + some([(5, i % 11 + 1) for i in range(900)], "bf16") + some([(33,)] * 200, "f16")
    check_clip(sfb, grads, 3.0)
    out = [torch.empty(x.shape, device="cuda") for x in grads]
    check_clip(sfb, grads, 1.0, 0.25, out)


def test_other_layouts_of_elements(sfb):
    a, b = some([(30, 50), (4, 6, 8)], "f32", 5)
    check_clip(sfb, [a.t(), b.permute(2, 0, 1)], 1.0)
    out = [torch.empty(30, 50, device="cuda").t(), torch.empty(4, 6, 8, device="cuda").permute(2, 0, 1)]
    check_clip(sfb, [a.t(), b.permute(2, 0, 1)], 0.1, 1.0, out)


@pytest.mark.parametrize("value", [1e-30, 1e25, 3e38])
def test_squares_beyond_fp32(sfb, value):
    grads = [torch.full((1000,), value, device="cuda") / 40, torch.zeros(5, device="cuda")]
    norm = norm64(grads)
    assert abs(float(sfb.grad_norm(grads)) - norm) <= 2.0 ** -23 * norm
    check_clip(sfb, grads, 1.0)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_norms_that_are_not_finite(sfb, value):
    grads = some(SIZES, "f32")
    grads[-1][3, 5] = value
    kept, out = [x.clone() for x in grads], [torch.full_like(x, 4.0) for x in grads]
    assert not math.isfinite(float(sfb.clip_grad_norm(grads, 1.0)))
    assert not math.isfinite(float(sfb.clip_grad_norm(grads, 1.0, out=out)))
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(grads, kept)) and all((x == 4).all() for x in out)


def test_all_zeros(sfb):
    grads = [torch.zeros(100, device="cuda")]
    assert float(sfb.clip_grad_norm(grads, 1.0)) == 0.0 and (grads[0] == 0).all()


def test_large_list_and_its_bits(sfb):
    """More chunks than CTAs; the same bits every time."""
    grads = some([(5_000_001,), (1024, 4099), (3, 7)], "bf16", 2)
    first = sfb.grad_norm(grads)
    assert abs(float(first) - norm64(grads)) <= 2.0 ** -23 * norm64(grads)
    for _ in range(3):
        assert torch.equal(sfb.grad_norm(grads), first)
    check_clip(sfb, grads, 1.0)


def test_tables_and_lists_in_graphs_and_streams(sfb):
    g = torch.Generator().manual_seed(4)
    sets = []
    for i in range(2):
        ids = torch.randint(0, 400, (3, 100), generator=g, dtype=torch.int32).cuda()
        sets.append((torch.randn(3, 100, 64, generator=g).cuda(), ids))

    def step(dout, ids):
        dtable, dpos, _ = sfb.embedding_grad(dout, ids, 400, positions=True)
        return dtable, dpos, sfb.clip_grad_norm([dtable, dpos], 1.0)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in sets], [], []
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*x))
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


# ---- a step -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_training_step(sfb, dtype):
    """Embedding, attention over itself, logits over the tied table, loss; its gradients back to the tables, clipped: against autograd in 64 bits
    on the same rounded parameters."""
    t = DTYPES[dtype]
    B, nb, H, d, vocab = 2, 4, 4, 64, 512
    L, hidden, scale = nb * 64, H * d, math.sqrt(H * d)
    g = torch.Generator().manual_seed(8)
    table, pos = (torch.randn(vocab, hidden, generator=g) / hidden ** 0.5 / 4).to(t), (0.1 * torch.randn(L, hidden, generator=g)).to(t)
    ids = torch.randint(0, vocab, (B, L), generator=g, dtype=torch.int32)
    targets = torch.randint(0, vocab, (B, L), generator=g, dtype=torch.int32)
    blocks = layout("stride", nb)
    lay = plan(sfb, blocks, 64)
    up = 64.0                                                # the loss is scaled up

    x, _ = sfb.embedding(table.cuda(), ids.cuda(), pos.cuda(), scale=scale)
    heads = x.view(B, L, H, d)
    o, lse = sfb.fused_attention_stats(heads, heads, heads, lay)
    logits = sfb.linear_nt(o.view(B, L, hidden), table.cuda())
    logp, stats, _, _, _, _ = sfb.token_logprobs(logits, targets.cuda())
    dlogits = sfb.token_logprobs_grad(logits, targets.cuda(), stats, torch.full((B, L), -up / (B * L), device="cuda"))
    do = sfb.linear(dlogits, table.cuda())
    dq, dk, dv = sfb.attention_backward_recompute(heads, heads, heads, o, do.view(B, L, H, d), lse, lay)
    dx = (dq.float() + dk.float() + dv.float()).view(B, L, hidden)
    # the tied table's gradient from the logits, onto which the embedding's is added
    dtable = torch.matmul(dlogits.view(-1, vocab).t().float(), o.view(-1, hidden).float())
    dpos = torch.zeros(L, hidden, device="cuda")
    sfb.embedding_grad(dx, ids.cuda(), vocab, scale=scale, positions=True, out=(dtable, dpos))
    norm = sfb.clip_grad_norm([dtable, dpos], 0.5, scale=1 / up)

    tab, ps = table.double().requires_grad_(), pos.double().requires_grad_()
    y = (scale * tab[ids.long()] + ps).view(B, L, H, d)
    out, _ = attend(y, y, y, blocks_to_elements(blocks, 64), 1 / math.sqrt(d))
    lp = torch.log_softmax(out.reshape(B, L, hidden) @ tab.t(), -1)
    loss = -lp.gather(2, targets.long()[..., None]).mean()
    loss.backward()
    total = math.sqrt(float(tab.grad.square().sum() + ps.grad.square().sum()))
    factor = min(1.0, 0.5 / (total + 1e-6))
    # about ten roundings to 16 bits in a row, of independent entries: their norm
    tol = 12 * half_step(t)
    loss = float(loss.detach())
    assert abs(float(-logp.mean()) - loss) <= tol * loss
    assert abs(float(norm) - total) <= tol * total
    for got, want in ((dtable, tab.grad), (dpos, ps.grad)):
        assert float((got.cpu().double() - factor * want).norm()) <= tol * float(factor * want.norm())
