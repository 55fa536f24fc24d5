"""Recorded steps of trees and of prompts."""
import random

import pytest

import tree_plain as plain
from conftest import TINY

pytestmark = pytest.mark.gpu


def test_trees_leave_prompts_room_to_be_recorded(model_dirs):
    from glassbox_b200.engine.engine import Engine, StepEntry
    rng, vocab = random.Random(1), TINY["D"]["vocab_size"]
    eng = Engine(model_dirs("D", "float32"), "float32", cache_tokens=1024, max_batch_tokens=256)
    eng.max_graphs = 4
    eng.add_request("x")
    for rows in (3, 12, 20, 28, 40, 60):
        for _ in range(3):
            eng.step([StepEntry("x", [rng.randrange(vocab) for _ in range(rows)], [0], plain.random_tree(rng, rows, 3))], commit=False)
    before = eng.graph_replays
    assert before > 0
    for rid in range(4):
        eng.add_request(rid)
        eng.step([StepEntry(rid, [rng.randrange(vocab) for _ in range(50)], [49])])
    assert eng.graph_replays == before + 2                  # (seen, recorded, replayed twice)
    eng.check()
