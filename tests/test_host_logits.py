"""What the operators on logits refuse, without a GPU: the host side's checks come before anything is launched (a call that passes
all of them on CPU tensors is refused for being there), and so do those of the C ABI."""
import ctypes as C
import math
import os
import re

import pytest

torch = pytest.importorskip("torch")


def z(*size, dtype=torch.float32):
    return torch.zeros(*size, dtype=dtype)


def i32(*size):
    return z(*size, dtype=torch.int32)


X = z(3, 50)
CALLS = [
    ("token_logprobs", lambda s: s.token_logprobs(X, i32(3)), "CUDA device"),
    ("no dimension", lambda s: s.token_logprobs(z(()), i32(1)), "last dimension"),
    ("no columns", lambda s: s.token_logprobs(z(3, 0), i32(3)), "1 to 2"),
    ("columns apart", lambda s: s.token_logprobs(z(50, 3).t(), i32(3)), "contiguous"),
    ("rows repeated", lambda s: s.token_logprobs(z(50).expand(3, 50), i32(3)), "pitch"),
    ("rows that overlap", lambda s: s.token_logprobs(z(100).as_strided((3, 50), (10, 1)), i32(3)), "pitch"),
    ("rows at two pitches", lambda s: s.token_logprobs(z(4, 3, 50)[::2, :2], i32(2, 2)), "pitch"),
    ("targets int64", lambda s: s.token_logprobs(X, z(3, dtype=torch.int64)), "targets"),
    ("targets of another shape", lambda s: s.token_logprobs(X, i32(4)), "targets"),
    ("targets apart", lambda s: s.token_logprobs(X, i32(6)[::2]), "targets"),
    ("vocab 0", lambda s: s.token_logprobs(X, i32(3), vocab=0), "vocab"),
    ("vocab beyond the columns", lambda s: s.token_logprobs(X, i32(3), vocab=51), "vocab"),
    ("scale 0", lambda s: s.token_logprobs(X, i32(3), scale=0.0), "scale"),
    ("scale -1", lambda s: s.token_logprobs(X, i32(3), scale=-1.0), "scale"),
    ("scale nan", lambda s: s.token_logprobs(X, i32(3), scale=math.nan), "scale"),
    ("scale inf", lambda s: s.token_logprobs(X, i32(3), scale=math.inf), "scale"),
    ("top_k -1", lambda s: s.token_logprobs(X, i32(3), top_k=-1), "top_k"),
    ("top_k beyond vocab", lambda s: s.token_logprobs(X, i32(3), vocab=10, top_k=11), "top_k"),
    ("top_k 129", lambda s: s.token_logprobs(z(3, 500), i32(3), top_k=129), "top_k"),
    ("alternatives of too many tokens", lambda s: s.token_logprobs(z(1, (1 << 19) + 1), i32(1), top_k=1), "2^19"),
    ("gradient", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 2), z(3)), "CUDA device"),
    ("stats of another shape", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 3), z(3)), "stats"),
    ("stats fp64", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 2).double(), z(3)), "stats"),
    ("dlogp expanded", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 2), z(1).expand(3)), "float tensor"),
    ("entropy alone", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 2), z(3), entropy=z(3)), "go together"),
    ("dentropy alone", lambda s: s.token_logprobs_grad(X, i32(3), z(3, 2), z(3), dentropy=z(3)), "go together"),
    ("lists", lambda s: s.distill_topk(X, i32(3, 4), z(3, 4)), "CUDA device"),
    ("lists of none", lambda s: s.distill_topk(X, i32(3, 0), z(3, 0)), "1 to 128"),
    ("lists of 129", lambda s: s.distill_topk(X, i32(3, 129), z(3, 129)), "1 to 128"),
    ("lists of two lengths", lambda s: s.distill_topk(X, i32(3, 4), z(3, 5)), "ids and teacher"),
    ("teacher bf16", lambda s: s.distill_topk(X, i32(3, 4), z(3, 4, dtype=torch.bfloat16)), "ids and teacher"),
    ("lists of other rows", lambda s: s.distill_topk(X, i32(2, 4), z(2, 4)), "ids and teacher"),
    ("remainder of too many tokens", lambda s: s.distill_topk(z(1, (1 << 20) + 1), i32(1, 4), z(1, 4), tail=True), "2^20"),
    ("gradient of lists", lambda s: s.distill_topk_grad(X, i32(3, 4), z(3, 4), z(3, 2), z(3)), "CUDA device"),
    ("stats without the remainder", lambda s: s.distill_topk_grad(X, i32(3, 4), z(3, 4), z(3, 2), z(3), tail=True), "stats"),
    ("stats with a remainder", lambda s: s.distill_topk_grad(X, i32(3, 4), z(3, 4), z(3, 3), z(3)), "stats"),
    ("a hard label without its stats", lambda s: s.distill_topk_grad(X, i32(3, 4), z(3, 4), z(3, 2), z(3), targets=i32(3), dlogp=z(3)), "go together"),
    ("scores", lambda s: s.linear_logprobs(z(3, 16), z(50, 16), i32(3)), "CUDA device"),
    ("table of another width", lambda s: s.linear_logprobs(z(3, 16), z(50, 24), i32(3)), "x and table"),
    ("table of another type", lambda s: s.linear_logprobs(z(3, 16), z(50, 16, dtype=torch.float16), i32(3)), "x and table"),
    ("a table that is no matrix", lambda s: s.linear_logprobs(z(3, 16), z(16), i32(3)), "x and table"),
    ("x apart", lambda s: s.linear_logprobs(z(3, 32)[:, :16], z(50, 16), i32(3)), "x and table"),
    ("vocab beyond the table", lambda s: s.linear_logprobs(z(3, 16), z(50, 16), i32(3), vocab=51), "vocab"),
    ("bias too short", lambda s: s.linear_logprobs(z(3, 16), z(50, 16), i32(3), bias=z(49)), "bias"),
]


@pytest.mark.parametrize("name,call,text", CALLS, ids=[c[0] for c in CALLS])
def test_refused_by_the_host(sfb, name, call, text):
    with pytest.raises(AssertionError, match=re.escape(text)):
        call(sfb)


def test_types_that_are_none_of_the_three(sfb):
    for t in (torch.float64, torch.int32):
        with pytest.raises(KeyError):
            sfb.token_logprobs(z(3, 50, dtype=t), i32(3))
    with pytest.raises(TypeError):
        sfb.token_logprobs([1.0, 2.0], i32(1))


one, null = C.c_void_p(64), None           # never dereferenced: the checks come first
ABI = [
    ("sfb_token_logprobs", (null, null, 50, one, 3, 50, 0, 1.0, one, one, null, null, null, 0, null), "logits"),
    ("sfb_token_logprobs", (null, C.c_void_p(66), 50, one, 3, 50, 0, 1.0, one, one, null, null, null, 0, null), "aligned"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 7, 1.0, one, one, null, null, null, 0, null), "dtype"),
    ("sfb_token_logprobs", (null, one, 49, one, 3, 50, 0, 1.0, one, one, null, null, null, 0, null), "pitch"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 0, 0, 1.0, one, one, null, null, null, 0, null), "vocab"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 0, 0.0, one, one, null, null, null, 0, null), "scale"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 0, 1.0, null, one, null, null, null, 0, null), "go together"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 0, 1.0, one, null, null, null, null, 0, null), "NULL"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 0, 1.0, one, one, null, one, one, 51, null), "top_k"),
    ("sfb_token_logprobs", (null, one, 50, one, 3, 50, 0, 1.0, one, one, null, null, one, 5, null), "NULL"),
    ("sfb_token_logprobs", (null, one, 1 << 20, one, 3, 1 << 20, 0, 1.0, one, one, null, one, one, 5, null), "alternatives"),
    ("sfb_token_logprobs_grad", (null, one, 50, null, one, one, null, null, one, 50, 3, 50, 50, 0, 1.0), "NULL"),
    ("sfb_token_logprobs_grad", (null, one, 50, one, one, one, one, null, one, 50, 3, 50, 50, 0, 1.0), "go together"),
    ("sfb_token_logprobs_grad", (null, one, 50, one, one, one, null, null, one, 49, 3, 50, 50, 0, 1.0), "overlap"),
    ("sfb_token_logprobs_grad", (null, one, 50, one, one, one, null, null, one, 50, 3, 51, 50, 0, 1.0), "vocab"),
    ("sfb_distill_topk", (null, one, 50, one, one, 3, 50, 0, 0, 1.0, 0, one, one, null), "entries"),
    ("sfb_distill_topk", (null, one, 50, one, one, 3, 50, 129, 0, 1.0, 0, one, one, null), "entries"),
    ("sfb_distill_topk", (null, one, 50, one, null, 3, 50, 4, 0, 1.0, 0, one, one, null), "NULL"),
    ("sfb_distill_topk", (null, one, 1 << 21, one, one, 3, 1 << 21, 4, 0, 1.0, 1, one, one, null), "remainder"),
    ("sfb_distill_topk_grad", (null, one, 50, one, one, one, one, one, null, one, one, 50, 3, 50, 50, 4, 0, 1.0, 0), "go together"),
    ("sfb_distill_topk_grad", (null, one, 50, one, one, null, one, null, null, null, one, 50, 3, 50, 50, 4, 0, 1.0, 0), "NULL"),
    ("sfb_linear_logprobs", (null, one, one, null, one, 3, 50, 16, 0, 1.0, one, one, null, null, one), "bf16 or fp16"),
    ("sfb_linear_logprobs", (null, one, one, null, one, 3, 50, 12, 1, 1.0, one, one, null, null, one), "multiple of 8"),
    ("sfb_linear_logprobs", (null, one, one, null, one, 3, 0, 16, 1, 1.0, one, one, null, null, one), "vocab"),
    ("sfb_linear_logprobs", (null, C.c_void_p(72), one, null, one, 3, 50, 16, 1, 1.0, one, one, null, null, one), "aligned"),
    ("sfb_linear_logprobs", (null, one, one, null, one, 3, 50, 16, 1, 1.0, one, one, null, null, null), "NULL"),
    ("sfb_linear_logprobs", (null, one, one, null, one, 3, 50, 16, 1, -1.0, one, one, null, null, one), "scale"),
]


@pytest.mark.parametrize("name,args,text", ABI)
def test_refused_by_the_library(sfb, name, args, text):
    assert getattr(sfb.lib, name)(*args) != 0
    assert text in sfb.lib.sfb_last_error().decode()


def test_workspace_of_the_scores(sfb):
    """It covers two parts per tile of 256 columns and row, never more rows than go through it at a time."""
    f = sfb.lib.sfb_linear_logprobs_workspace
    assert f(1, 1) >= 36 and f(0, 30522) == 0
    assert f(4096, 30522) >= 4096 * (120 * 32 + 4)
    assert f(1 << 20, 30522) == f(32768, 30522) < 1 << 28


def test_order_of_the_candidates_counter():
    """CTAs of a cluster add to CTA 0's counter once they have waited for its arrival: the counter has to be cleared before that arrival,
    which has to release the store, and the wait has to acquire it.  Nothing but the order in the source can show a missing one: a whole
    pass over the row lies between, so results are right all the same, nearly always."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sf-bert_b200", "csrc", "logits.cu")
    with open(path) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index("row_stats_kernel(const StatParams p)"):]
    clear, arrive, wait, add = (body.index(x) for x in ("top_s->cnt = 0", "barrier.cluster.arrive.", "barrier.cluster.wait.", "atomicAdd(&join->cnt"))
    assert clear < arrive < wait < add
    assert "if (TOP) asm volatile(\"barrier.cluster.arrive.release.aligned" in body[arrive - 60:arrive + 80]
    assert not re.search(r"barrier\.cluster\.wait\.(?!acquire)", body[:add])
