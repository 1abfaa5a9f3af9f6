"""What the operators of a training step refuse, without a GPU: the host side's checks come before anything is launched (a call that
passes all of them on CPU tensors is refused for being there), and so do those of the C ABI."""
import ctypes as C
import math
import re
import types

import pytest

torch = pytest.importorskip("torch")


def z(*size, dtype=torch.float32):
    return torch.zeros(*size, dtype=dtype)


def i32(*size):
    return z(*size, dtype=torch.int32)


def lay(nb=2, bs=32, heads=1):
    return types.SimpleNamespace(heads=heads, nb=nb, block_size=bs, blocks=nb, nn_max=1, nt_lut=i32(heads, nb, 2), nn_lut=i32(heads, 2 * nb, 2), tn_lut=i32(heads, 2 * nb, 2),
                                 tn_max=1, mask_np=None)


X = z(1, 64, 2, 16)
S = z(1, 2, 64)
PACKED = z(1, 64, 3, 2, 16)
G, T = z(2, 5, 16), i32(2, 5)
ODD = z(40)
CALLS = [
    ("attention", lambda s: s.fused_attention_stats(X, X, X, lay()), "CUDA device"),
    ("three dimensions", lambda s: s.fused_attention_stats(X[0], X[0], X[0], lay()), "[B, L, H, d]"),
    ("another length", lambda s: s.fused_attention_stats(X[:, :40], X[:, :40], X[:, :40], lay()), "sequence length"),
    ("heads of the layout", lambda s: s.fused_attention_stats(X, X, X, lay(heads=3)), "heads"),
    ("k of another type", lambda s: s.fused_attention_stats(X, X.half(), X, lay()), "alike"),
    ("v of another size", lambda s: s.fused_attention_stats(X, X, z(1, 64, 2, 8), lay()), "alike"),
    ("two pitches", lambda s: s.fused_attention_stats(X, PACKED[:, :, 0], X, lay()), "pitches"),
    ("heads apart", lambda s: s.fused_attention_stats(*[z(1, 64, 16, 2).transpose(2, 3)] * 3, lay()), "head slice"),
    ("batch elements apart", lambda s: s.fused_attention_stats(*[z(4, 64, 2, 16)[::2]] * 3, lay()), "head slice"),
    ("wide heads", lambda s: s.fused_attention_stats(*[z(1, 64, 1, 129)] * 3, lay()), "128"),
    ("backward", lambda s: s.attention_backward_recompute(X, X, X, X, X, S, lay()), "CUDA device"),
    ("o of another size", lambda s: s.attention_backward_recompute(X, X, X, X[:, :, :1], X, S, lay()), "o and dO"),
    ("do of another type", lambda s: s.attention_backward_recompute(X, X, X, X, X.half(), S, lay()), "o and dO"),
    ("lse of another order", lambda s: s.attention_backward_recompute(X, X, X, X, X, z(1, 64, 2), lay()), "lse"),
    ("lse in 64 bits", lambda s: s.attention_backward_recompute(X, X, X, X, X, S.double(), lay()), "lse"),
    ("lse apart", lambda s: s.attention_backward_recompute(X, X, X, X, X, z(1, 2, 128)[:, :, ::2], lay()), "lse"),
    ("table's gradient", lambda s: s.embedding_grad(G, T, 9), "CUDA device"),
    ("dout of two dimensions", lambda s: s.embedding_grad(G[0], T[0], 9), "[B, L, hidden]"),
    ("ids of another shape", lambda s: s.embedding_grad(G, i32(5, 2), 9), "[B, L, hidden]"),
    ("ids int64", lambda s: s.embedding_grad(G, T.long(), 9), "int32"),
    ("dout apart", lambda s: s.embedding_grad(z(2, 5, 32)[:, :, ::2], T, 9), "contiguous"),
    ("no vocabulary", lambda s: s.embedding_grad(G, T, 0), "vocab"),
    ("a vocabulary too large", lambda s: s.embedding_grad(G, T, (1 << 27) + 1), "vocab"),
    ("hidden 12", lambda s: s.embedding_grad(z(2, 5, 12), T, 9), "multiple of 8"),
    ("hidden 0", lambda s: s.embedding_grad(z(2, 5, 0), T, 9), "multiple of 8"),
    ("gradients of a third type", lambda s: s.embedding_grad(G, T, 9, dtype=torch.float16), "dout's type"),
    ("norm", lambda s: s.grad_norm([z(3)]), "CUDA device"),
    ("clipping", lambda s: s.clip_grad_norm([z(3)], 1.0), "CUDA device"),
    ("no gradients", lambda s: s.grad_norm([]), "at least one"),
    ("max_norm -1", lambda s: s.clip_grad_norm([z(3)], -1.0), "max_norm"),
    ("max_norm nan", lambda s: s.clip_grad_norm([z(3)], math.nan), "max_norm"),
    ("scale 0", lambda s: s.clip_grad_norm([z(3)], 1.0, scale=0.0), "scale"),
    ("scale inf", lambda s: s.clip_grad_norm([z(3)], 1.0, scale=math.inf), "scale"),
    ("scale nan", lambda s: s.grad_norm([z(3)], scale=math.nan), "scale"),
    ("elements apart", lambda s: s.grad_norm([z(6)[::2]]), "dense"),
    ("elements repeated", lambda s: s.clip_grad_norm([z(1).expand(5)], 1.0), "dense"),
    ("out too short", lambda s: s.clip_grad_norm([z(3), z(3)], 1.0, out=[z(3)]), "per gradient"),
    ("out of another shape", lambda s: s.clip_grad_norm([z(3)], 1.0, out=[z(4)]), "laid out"),
    ("out of another order", lambda s: s.clip_grad_norm([z(3, 4)], 1.0, out=[z(4, 3).t()]), "laid out"),
    ("fp32 into fp16", lambda s: s.clip_grad_norm([z(3)], 1.0, out=[z(3).half()]), "laid out"),
]


@pytest.mark.parametrize("name,call,text", CALLS, ids=[c[0] for c in CALLS])
def test_refused_by_the_host(sfb, name, call, text):
    with pytest.raises(AssertionError, match=re.escape(text)):
        call(sfb)


def test_types_that_are_none_of_the_three(sfb):
    for t in (torch.float64, torch.int32):
        with pytest.raises(KeyError):
            sfb.grad_norm([z(3, dtype=t)])
        with pytest.raises(KeyError):
            sfb.fused_attention_stats(X.to(t), X.to(t), X.to(t), lay())
        with pytest.raises(KeyError):
            sfb.embedding_grad(G.to(t), T, 9)
    with pytest.raises(KeyError):
        sfb.embedding_grad(G, T, 9, dtype=torch.float64)
    with pytest.raises(TypeError):
        sfb.grad_norm([1.0])
    with pytest.raises(TypeError):
        sfb.grad_norm(3)


one, null = C.c_void_p(64), None           # never dereferenced: the checks come first
BACK = dict(dtype=1, bs=64, blocks=4, B=1, nb=2, H=2, d=64, lh=1, ld=4, mh=1, scale=0.125, nn=2, tn=2, ip=0, op=0, dp=0, gp=0, ws=one, size=1 << 40)


def back(pointers=(one,) * 13, **changed):
    a = dict(BACK, **changed)
    p = list(pointers)
    return (null,) + tuple(p[:9]) + (null,) + tuple(p[9:12]) + tuple(a[n] for n in ("dtype", "bs", "blocks", "B", "nb", "H", "d", "lh", "ld", "mh", "scale", "nn", "tn", "ip", "op",
                                                                                   "dp", "gp", "ws", "size"))


def arr(kind, *values):
    return (kind * len(values))(*values)


PTR, N, D = arr(C.c_void_p, 64), arr(C.c_uint64, 5), arr(C.c_int32, 0)
ABI = [
    ("sfb_fused_attention_stats", (null, one, one, one, one, one, null, null, 1, 64, 4, 1, 2, 2, 64, 1, 4, 1, 0.125, 2, 0, 0), "NULL"),
    ("sfb_fused_attention_stats", (null, one, one, one, one, one, one, null, 1, 48, 4, 1, 2, 2, 64, 1, 4, 1, 0.125, 2, 0, 0), "block_size"),
    ("sfb_fused_attention_stats", (null, one, one, one, one, one, one, null, 1, 64, 4, 1, 2, 2, 64, 1, 4, 1, 0.125, 2, 100, 0), "pitch"),
    ("sfb_attention_backward_recompute", back((one, one, null) + (one,) * 9), "NULL"),
    ("sfb_attention_backward_recompute", back((one,) * 8 + (null,) + (one,) * 3), "NULL"),
    ("sfb_attention_backward_recompute", back(dtype=5), "dtype"),
    ("sfb_attention_backward_recompute", back(bs=16), "block_size"),
    ("sfb_attention_backward_recompute", back(d=129), "state_dim"),
    ("sfb_attention_backward_recompute", back(lh=3), "lut_heads"),
    ("sfb_attention_backward_recompute", back(mh=3), "mask_heads"),
    ("sfb_attention_backward_recompute", back(lh=2, ld=3), "lut_dim"),
    ("sfb_attention_backward_recompute", back(ip=127), "pitch"),
    ("sfb_attention_backward_recompute", back(gp=127), "pitch"),
    ("sfb_attention_backward_recompute", back(ws=null), "workspace"),
    ("sfb_attention_backward_recompute", back(ws=C.c_void_p(72)), "workspace"),
    ("sfb_attention_backward_recompute", back(size=100), "workspace"),
    ("sfb_embedding_scaled", (null, null, one, one, null, 1, 1, 8, 1, 0, 1.0, null), "NULL"),
    ("sfb_embedding_grad", (null, null, null, one, one, 1, 1, 8, 5, 0, 0, 1.0, 0, null, one), "NULL"),
    ("sfb_embedding_grad", (null, one, null, one, one, 1, 1, 12, 5, 0, 0, 1.0, 0, null, one), "multiple of 8"),
    ("sfb_embedding_grad", (null, one, null, one, one, 1, 1, 8, 0, 0, 0, 1.0, 0, null, one), "vocab"),
    ("sfb_embedding_grad", (null, one, null, one, one, 1, 1, 8, 5, 0, 1, 1.0, 0, null, one), "dtype"),
    ("sfb_embedding_grad", (null, one, null, one, one, 1, 1, 8, 5, 0, 0, 1.0, 0, null, null), "NULL"),
    ("sfb_embedding_grad", (null, one, null, C.c_void_p(72), one, 1, 1, 8, 5, 0, 0, 1.0, 0, null, one), "aligned"),
    ("sfb_embedding_grad", (null, one, null, one, one, 1 << 16, 1 << 16, 8, 5, 0, 0, 1.0, 0, null, one), "tokens"),
    ("sfb_clip_grad_norm", (null, 1, PTR, null, N, D, null, 1.0, 1.0, null, one), "NULL"),
    ("sfb_clip_grad_norm", (null, 1, PTR, null, N, D, null, -1.0, 1.0, one, one), "max_norm"),
    ("sfb_clip_grad_norm", (null, 1, PTR, null, N, D, null, 1.0, 0.0, one, one), "scale"),
    ("sfb_clip_grad_norm", (null, 1, PTR, null, N, arr(C.c_int32, 3), null, 1.0, 1.0, one, one), "dtype"),
    ("sfb_clip_grad_norm", (null, 1, PTR, PTR, N, D, arr(C.c_int32, 1), 1.0, 1.0, one, one), "dtype"),
    ("sfb_clip_grad_norm", (null, 1, PTR, PTR, N, D, null, 1.0, 1.0, one, one), "NULL"),
    ("sfb_clip_grad_norm", (null, 1, arr(C.c_void_p, 66), null, N, D, null, 1.0, 1.0, one, one), "aligned"),
    ("sfb_grad_norm", (null, 1, arr(C.c_void_p, 0), N, D, 1.0, one, one), "NULL"),
    ("sfb_grad_norm", (null, 1, PTR, arr(C.c_uint64, 1 << 60), D, 1.0, one, one), "elements"),
]


@pytest.mark.parametrize("name,args,text", ABI, ids=["%s-%s-%d" % (n[4:], t, i) for i, (n, _, t) in enumerate(ABI)])
def test_refused_by_the_library(sfb, name, args, text):
    assert getattr(sfb.lib, name)(*args) != 0
    assert text in sfb.lib.sfb_last_error().decode()


def test_workspaces(sfb):
    f = sfb.lib.sfb_attention_backward_workspace
    rows = 2 * 2 * 4 * 128 * 4
    assert f(1, 64, 4, 2, 2, 4, 64, 2, 2, 1) >= rows and f(0, 32, 8, 2, 4, 4, 64, 2, 2, 1) >= rows + 2 * 8 * 32 * 32 * 4
    assert f(9, 64, 4, 2, 2, 4, 64, 2, 2, 1) == 0
    # P and dS go through it a few heads at a time: in 512 MB, beside two numbers per row
    assert f(0, 32, 1 << 12, 64, 64, 16, 64, 64, 64, 1) <= (512 << 20) + 2 * 64 * 2048 * 16 * 4
    g = sfb.lib.sfb_embedding_grad_workspace
    assert g(0, 5, 16, 9) >= 40 and g(8, 4096, 768, 30522) >= 32768 * 16 + 30523 * 4 + 1024 * 2 * 768 * 4
    assert sfb.lib.sfb_clip_grad_norm_workspace(1) >= 8


def test_tensors_that_share_memory(sfb):
    """Found on the host, before the device is: what is written shares memory with nothing but the gradient that it takes the place of."""
    flat = z(100)
    for grads, out in (([flat, flat], None), ([flat[:60], flat[50:]], None), ([flat[10:20], flat], None), ([flat[:50], z(50)], [z(50), flat[40:90]]),
                       ([flat[:50], flat[50:]], [flat[50:], flat[:50]])):
        with pytest.raises(AssertionError, match="shares memory"):
            sfb.clip_grad_norm(grads, 1.0, out=out)
    for grads, out in (([flat[:50], flat[50:]], None), ([flat, flat], [z(100), z(100)]), ([flat], [flat]), ([flat[:50], flat[50:]], [flat[:50], z(50)])):
        with pytest.raises(AssertionError, match="CUDA device"):
            sfb.clip_grad_norm(grads, 1.0, out=out)
    with pytest.raises(AssertionError, match="CUDA device"):
        sfb.grad_norm([flat, flat])                          # nothing is written
