"""What the operators of a training step refuse beside test_host_training.py's list, without a GPU: a call that passes all checks on CPU tensors
is refused for being there."""
import re

import pytest

torch = pytest.importorskip("torch")

from test_host_training import i32, lay, z                # noqa: E402


IDS, TABLE = i32(2, 5), z(9, 16)
EMBEDDING = [
    ("a lookup", (TABLE, IDS), "CUDA device"),
    ("with positions", (TABLE, IDS, z(5, 16)), "CUDA device"),
    ("with a longer table of positions", (TABLE, IDS, z(512, 16)), "CUDA device"),
    ("with a batch dimension", (TABLE, IDS, z(1, 5, 16)), "CUDA device"),
    ("positions too few", (TABLE, IDS, z(4, 16)), "pos must"),
    ("positions of another width", (TABLE, IDS, z(10, 8)), "pos must"),
    ("positions of another type", (TABLE, IDS, z(5, 16, dtype=torch.bfloat16)), "pos must"),
    ("positions apart", (TABLE, IDS, z(10, 16)[::2]), "pos must"),
    ("positions elsewhere", (TABLE, IDS, torch.zeros(5, 16, device="meta")), "pos must"),
    ("ids elsewhere", (TABLE, torch.zeros(2, 5, dtype=torch.int32, device="meta")), "ids must be on"),
    ("ids of one dimension", (TABLE, IDS[0]), "[B, L]"),
    ("ids int64", (TABLE, IDS.long()), "int32"),
]


@pytest.mark.parametrize("name,args,text", EMBEDDING, ids=[c[0] for c in EMBEDDING])
def test_lookups_refused(sfb, name, args, text):
    with pytest.raises(AssertionError, match=re.escape(text)):
        sfb.embedding(*args, scale=2.0)


X, S = z(1, 64, 2, 16), z(1, 2, 64)
HEADS = z(1, 64, 6, 16)                          # six heads side by side
ROWS = z(65 * 96)
FLAT = z(4 * 64 * 2 * 16)


def head(i, n=2):
    return HEADS[:, :, i:i + n]


def at(first):
    return FLAT[first:first + X.numel()].view(X.shape)


def row(first):                                  # heads that begin there in rows of 96
    return ROWS.as_strided(X.shape, (64 * 96, 96, 16, 1), first)


def stats(out, q=X, k=X, v=X):
    return lambda s: s.fused_attention_stats(q, k, v, lay(), out=out)


def back(*out, q=X, k=X, v=X, o=X, do=X, lse=S):
    return lambda s: s.attention_backward_recompute(q, k, v, o, do, lse, lay(), out=out)


N = X.numel()
ATTENTION = [
    ("output", stats(z(1, 64, 2, 16)), "CUDA device"),
    ("output beside its operands' heads elsewhere", stats(head(2)), "CUDA device"),
    ("output of another size", stats(z(1, 64, 2, 8)), "out must be like q"),
    ("output of another type", stats(X.half()), "out must be like q"),
    ("output elsewhere", stats(torch.zeros(1, 64, 2, 16, device="meta")), "out must be like q"),
    ("heads of the output apart", stats(z(1, 64, 16, 2).transpose(2, 3)), "head slice"),
    ("output is q", stats(X), "out must not share"),
    ("output is v", stats(X, z(1, 64, 2, 16), z(1, 64, 2, 16)), "out must not share"),
    ("output over the end of k", stats(at(N - 1), z(1, 64, 2, 16), at(0), z(1, 64, 2, 16)), "out must not share"),
    ("output behind k", stats(at(N), z(1, 64, 2, 16), at(0), z(1, 64, 2, 16)), "CUDA device"),
    ("output between the operands' heads", stats(head(2), head(0), head(0), head(4)), "out must not share"),
    ("gradients", back(*(z(1, 64, 2, 16) for _ in range(3))), "CUDA device"),
    ("gradients side by side", back(head(4), head(0), head(2)), "CUDA device"),
    ("gradients one after another", back(at(0), at(N), at(2 * N)), "CUDA device"),
    ("two gradients", back(z(1, 64, 2, 16), z(1, 64, 2, 16)), "three tensors"),
    ("a gradient of another size", back(at(0), at(N), z(1, 64, 1, 16)), "out's tensors must be like q"),
    ("a gradient of another type", back(at(0), at(N), X.bfloat16()), "out's tensors must be like q"),
    ("gradients of two pitches", back(at(0), at(N), head(0)), "different row pitches"),
    ("a gradient twice", back(at(0), at(N), at(N)), "out's tensors must not share"),
    ("gradients that share a head", back(head(0), head(1), head(4)), "out's tensors must not share"),
    ("gradients that share a head across rows", back(row(0), row(32), row(80)), "out's tensors must not share"),
    ("gradients that fill a row", back(row(0), row(32), row(64)), "CUDA device"),
    ("gradients that share an element", back(at(0), at(N - 1), at(2 * N)), "out's tensors must not share"),
    ("a gradient is o", back(at(0), at(N), at(2 * N), o=at(2 * N)), "out must not share memory with the operands"),
    ("a gradient is dO", back(at(0), at(N), at(2 * N), do=at(0)), "out must not share memory with the operands"),
    ("gradients between the operands' heads", back(head(0), head(2), head(4), q=head(1), k=head(1), v=head(1)), "out must not share memory with the operands"),
    ("a gradient over the log-sums", back(at(0), at(N), at(2 * N), lse=FLAT[N:N + 128].view(1, 2, 64)), "out must not share memory with the operands"),
]
G = z(2, 5, 16)
ROOM = z(9 * 16 + 5 * 16 + 2 * 5 * 16)
TABLES = [
    ("a table", dict(out=z(9, 16)), "CUDA device"),
    ("tables", dict(out=(z(9, 16), z(5, 16)), positions=True), "CUDA device"),
    ("a list of tables", dict(out=[z(9, 16), z(5, 16)], positions=True), "CUDA device"),
    ("one table with positions", dict(out=z(9, 16), positions=True), "out must be"),
    ("three tables", dict(out=(z(9, 16), z(5, 16), z(5, 16)), positions=True), "out must be"),
    ("tables in the other order", dict(out=(z(5, 16), z(9, 16)), positions=True), "out must be"),
    ("a table of another size", dict(out=z(10, 16)), "out must be"),
    ("a table of another type", dict(out=z(9, 16).half()), "out must be"),
    ("a table apart", dict(out=z(9, 32)[:, ::2]), "out must be"),
    ("a table elsewhere", dict(out=torch.zeros(9, 16, device="meta")), "out must be"),
    ("tables that share memory", dict(out=(ROOM[:144].view(9, 16), ROOM[143:223].view(5, 16)), positions=True), "share memory"),
    ("a table over dout", dict(out=ROOM[:144].view(9, 16), dout=ROOM[140:300].view(2, 5, 16)), "share memory"),
    ("positions over dout", dict(out=(z(9, 16), ROOM[:80].view(5, 16)), positions=True, dout=ROOM[79:239].view(2, 5, 16)), "share memory"),
    ("tables beside dout", dict(out=(ROOM[:144].view(9, 16), ROOM[144:224].view(5, 16)), positions=True, dout=ROOM[224:384].view(2, 5, 16)), "CUDA device"),
]


@pytest.mark.parametrize("name,call,text", ATTENTION, ids=[c[0] for c in ATTENTION])
def test_results_of_the_attention_refused(sfb, name, call, text):
    with pytest.raises(AssertionError, match=text):
        call(sfb)


@pytest.mark.parametrize("name,args,text", TABLES, ids=[c[0] for c in TABLES])
def test_results_of_the_tables_refused(sfb, name, args, text):
    args = dict(args)
    with pytest.raises(AssertionError, match=text):
        sfb.embedding_grad(args.pop("dout", G), IDS, 9, **args)


def test_what_is_not_a_sequence_of_tensors(sfb):
    for out in (3, (1.0, 2.0, 3.0)):
        with pytest.raises(TypeError):
            sfb.attention_backward_recompute(X, X, X, X, X, S, lay(), out=out)


def test_workspaces_of_large_heads(sfb):
    """8 bytes per row where nothing of the scores is in memory; otherwise P and dS of some (batch, head) pairs, up to 512 MB, or of one where that is more."""
    f = sfb.lib.sfb_attention_backward_workspace
    mb = 1 << 20

    def asked(dtype, bs, nb, blocks, d, B=1, H=12, nn=None, tn=None, aligned=1):
        return f(dtype, bs, blocks, B, nb, H, d, nb if nn is None else nn, nb if tn is None else tn, aligned) - 8 * B * H * nb * bs

    def causal(nb):
        return nb * (nb + 1) // 2

    assert asked(1, 64, 256, causal(256), 64) == 0                                         # the tensor-core kernels up to 256 block-rows
    assert asked(1, 64, 257, causal(257), 64) == 4 * causal(257) * 4096                    # one pair: 518 MB
    assert asked(1, 64, 4096, 4096 * 20, 64, nn=128, tn=128) == 0                          # any number of short rows and columns
    assert 0 < asked(1, 64, 4096, 4096 * 20, 64, nn=129, tn=128) <= 1280 * mb
    assert 0 < asked(1, 64, 256, causal(256), 64, aligned=0) <= 514 * mb
    assert asked(1, 64, 512, causal(512), 64) == 4 * causal(512) * 4096 > 2000 * mb        # 32768 positions
    assert asked(2, 64, 1024, causal(1024), 128) == 4 * causal(1024) * 4096                # 65536
    assert asked(0, 32, 512, causal(512), 64) == 12 * causal(512) * 1024 > 1500 * mb
    for dtype, bs, nb, blocks, d in ((1, 32, 64, 64 * 20, 64), (2, 64, 32, 300, 128), (0, 32, 64, 2080, 64), (0, 64, 16, 256, 128)):
        for H in (1, 12, 400):
            assert 0 < asked(dtype, bs, nb, blocks, d, 8, H) <= 512 * mb


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("bs,d", [(32, 40), (64, 64)])
def test_workspaces_of_nothing(sfb, dtype, bs, d):
    """A sequence without blocks, a batch without elements, positions that no call takes: no memory, and no division by their number."""
    f = sfb.lib.sfb_attention_backward_workspace
    for blocks, B, nb, H in ((0, 2, 0, 4), (5, 2, 0, 4), (0, 0, 3, 4), (0, 2, 3, 0), (4, 1, 1 << 26, 1)):
        for aligned in (0, 1):
            assert f(dtype, bs, blocks, B, nb, H, d, 0, 0, aligned) == 0
    assert f(dtype, bs, 0, 2, 3, 4, d, 0, 0, 0) == 2 * 4 * 2 * 3 * bs * 4                  # rows without blocks: two numbers each
    assert sfb.lib.sfb_embedding_grad_workspace(0, 0, 0, 0) >= 0 and sfb.lib.sfb_clip_grad_norm_workspace(0) >= 8
