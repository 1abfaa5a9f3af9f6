"""What the operators of a training step refuse beside test_host_training.py's list, without a GPU: a call that passes all checks on CPU tensors
is refused for being there."""
import re

import pytest

torch = pytest.importorskip("torch")

from test_host_training import i32, z                     # noqa: E402


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
