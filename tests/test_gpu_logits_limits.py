"""GPU tests of the operators on logits where their arithmetic or their order could go wrong: against 64 bits, within derived bounds."""
import math

import pytest

torch = pytest.importorskip("torch")
import logits_reference as R  # noqa: E402

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
