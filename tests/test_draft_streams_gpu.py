"""Sampled generation with a drafting model, seeds alike: the first token against the model's probabilities."""
import numpy as np
import pytest

import tree_plain as plain
from plain import llama_plain

pytestmark = pytest.mark.gpu


def test_first_tokens_have_the_models_distribution(model_dirs, runs=2000):
    """A chi-square over twelve groups of tokens (11 degrees: 45 is passed once in 2e5), from those that the model likes more than the drafting one to the others."""
    import glassbox_b200
    from glassbox_b200.engine.drafts import DraftModel
    from glassbox_b200.engine.engine import Engine
    folder, other, prompt = model_dirs("D", "float32"), model_dirs("D", "float32", 12), [5, 7, 9]
    x, y = (llama_plain.forward_logits(f, prompt)[-1] for f in (folder, other))
    heat = float(np.float32(x.std() / 1.5))
    p, q = plain.softmax(x, heat), plain.softmax(y, heat)
    assert np.minimum(p, q).sum() < 0.7                    # (drafts are refused often enough to see what follows)
    order = np.argsort(p / q)
    group = np.empty(len(p), dtype=int)
    group[order] = np.minimum(np.cumsum(p[order]) * 12, 11).astype(int)
    llm = glassbox_b200.load(folder, "float32", blocks=32, budget=64, max_seqs=2)
    small = Engine(other, "float32", cache_tokens=256, max_batch_tokens=64, max_requests=2)
    tokens = [llm.generate(prompt, 2, temperature=heat, seed=s, drafts=DraftModel(small, tokens=3, seed=s))[0] for s in range(runs)]
    want = np.bincount(group, weights=p, minlength=12) * runs
    chi = ((np.bincount(group[tokens], minlength=12) - want) ** 2 / want).sum()
    assert chi < 45, chi
