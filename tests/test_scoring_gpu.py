"""Scoring texts beside serving: what it refuses, and what it leaves behind in the engine."""
import random

import numpy as np
import pytest
import torch

import glassbox_b200

pytestmark = pytest.mark.gpu


def load(model_dirs, **kw):
    return glassbox_b200.load(model_dirs("D", "bfloat16"), "bfloat16", **{"blocks": 64, "budget": 64, **kw})


@pytest.mark.parametrize("cache_bits", [None, 4])
def test_scoring_leaves_room_for_serving(model_dirs, cache_bits):
    """Texts of every length, each twice: recorded steps are kept for good, a bounded number of them and of bytes."""
    llm = load(model_dirs, cache_bits=cache_bits)
    rng = random.Random(1)
    texts = [[rng.randrange(300) for _ in range(n)] for n in range(2, 300, 7)]
    first = llm.score(texts)
    torch.cuda.synchronize()
    held, graphs = torch.cuda.memory_allocated(), len(llm.engine._graphs)
    again = llm.score(texts + texts)
    torch.cuda.synchronize()
    # (portions are recorded at one size, 64 rows, for each width of the block tables, 8, 16 and 32 pages here, and single tokens likewise)
    assert graphs <= len(llm.engine._graphs) <= 2 * 3
    assert torch.cuda.memory_allocated() - held <= 3 * 64 * 300 * 4 + (1 << 20)
    replays = llm.engine.graph_replays
    llm.score(texts[:4])
    assert llm.engine.graph_replays == replays + 4               # (and short texts do replay them)
    for a, b in zip(first + first, again):
        assert np.abs(a.logprobs - b.logprobs).max() < 1e-3 and a.top_ids.shape == b.top_ids.shape


def test_tokens_outside_the_vocabulary_are_refused(model_dirs):
    llm = load(model_dirs)
    free = llm.engine.cache.free_pages(0)
    for text in ([1, 2, 300], [1, -1, 2], [300], [1, 2, 1 << 40]):
        with pytest.raises(ValueError, match="prompt 1.*vocabulary"):
            llm.score([[5, 6, 7], text])
    assert llm.engine.cache.free_pages(0) == free
    assert np.isfinite(llm.score([1, 2, 299]).logprobs).all()


def test_room_is_for_steps_with_portions_of_prompts(model_dirs):
    """Single tokens, one of which wants no logits, are recorded at their own size whatever room is asked for, and come out the same."""
    from glassbox_b200.engine.engine import StepEntry
    got = []
    for room in (0, 64):
        eng = load(model_dirs).engine
        for r in "ab":
            eng.add_request(r)
            eng.step([StepEntry(r, list(range(1, 30)), [])])
        for t in range(4):
            got.append(eng.step([StepEntry("a", [t], []), StepEntry("b", [t + 7], [0])], room=room).clone())
        eng.check()
        assert all(key[1] == 8 for key in eng._graphs if key[0] == "step" and key[3] == 0) and eng.graph_replays > 0
    assert all(torch.equal(x, y) for x, y in zip(got[:4], got[4:]))
