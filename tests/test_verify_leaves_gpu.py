"""Verification with drafted logits: rows without children were drawn from for nothing, whatever stands there."""
import pytest
import torch

import tree_plain as plain
from test_verify_tree_gpu import SHAPES, either_way, make, run  # noqa: F401  (the fixture: both forms)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [257, 20000])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_rows_without_children_hold_anything(dtype, vocab, value):
    b = make(SHAPES + [(6, 1)] * 20, vocab, dtype, 41, True, [0.9] * 26)
    b["draft"][:60] = b["logits"][:60]                    # (these drafts are taken: walks end at leaves)
    leaves = [b["firsts"][i] + r for i, tree in enumerate(b["parents"]) for r in range(len(tree)) if r not in tree]
    want, ends = [], 0
    clean = b["draft"].float().cpu().numpy().copy()
    clean[leaves] = 0.0
    b["draft"][leaves] = value
    logits = b["logits"].float().cpu().numpy()
    path, accepted, following = run(b)
    for i, tree in enumerate(b["parents"]):
        a, e = b["firsts"][i], b["firsts"][i + 1]
        if tree:
            kept, token = plain.verify(logits[a:e], b["tokens"][a:e].tolist(), tree, b["uniform"][a:e].numpy(), 0.9, clean[a:e])
            assert path[a:e] == kept + [-1] * (e - a - len(kept)) and (accepted[i], following[i]) == (len(kept), token), f"request {i}"
            ends += kept[-1] not in tree
    assert ends > 3
