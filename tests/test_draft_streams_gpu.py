"""Sampled generation with a drafting model, seeds alike: the first token against the model's probabilities."""
import numpy as np
import pytest
import torch

import tree_plain as plain
from conftest import TINY
from glassbox_b200.models.llama import make_llama_raw_config
from plain import llama_plain

pytestmark = pytest.mark.gpu


def test_first_tokens_have_the_models_distribution(tmp_path, runs=3000):
    """A chi-square over sixteen tokens (15 degrees: 55 is passed once in 5e5). Where a draft and what is drawn in its place came from one number, it would be
    0.024 larger a run."""
    import glassbox_b200
    from glassbox_b200.engine.drafts import DraftModel
    from glassbox_b200.engine.engine import Engine
    folders, prompt = [], [5, 7, 9]
    for seed in (11, 12):
        folders.append(str(tmp_path / str(seed)))
        glassbox_b200.write_random_model(folders[-1], make_llama_raw_config(**dict(TINY["D"], vocab_size=16)), seed, torch.float32)
    x, y = (llama_plain.forward_logits(f, prompt)[-1] for f in folders)
    heat = float(np.float32(x.std()))
    p, q = plain.softmax(x, heat), plain.softmax(y, heat)
    assert np.minimum(p, q).sum() < 0.6                    # (drafts are refused often enough to see what follows)
    llm = glassbox_b200.load(folders[0], "float32", blocks=32, budget=64, max_seqs=2)
    small = Engine(folders[1], "float32", cache_tokens=256, max_batch_tokens=64, max_requests=2)
    tokens = [llm.generate(prompt, 2, temperature=heat, seed=s, drafts=DraftModel(small, tokens=3, seed=s))[0] for s in range(runs)]
    chi = ((np.bincount(tokens, minlength=16) - p * runs) ** 2 / (p * runs)).sum()
    assert chi < 55, chi
