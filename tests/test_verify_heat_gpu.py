"""Verification of drafted tokens at temperatures next to zero and next to infinity, against the plain walk in float64."""
import random

import numpy as np
import pytest
import torch

import tree_plain as plain
from test_verify_tree_gpu import SHAPES, check, either_way, make, run  # noqa: F401  (the fixture: both forms)

pytestmark = pytest.mark.gpu


def batch(heat, largest, drafted, masked, dtype=torch.float32, vocab=5001):
    """Drafts are the model's most likely token, the drafting model's, or one that neither gives a probability; largest logits are about ``largest``."""
    rng = random.Random(int(largest) + 2 * drafted + masked)
    b = make(SHAPES, vocab, torch.float32, 21, drafted, [1.0] * 6, agree=0.0, masked=masked)
    for name in ("logits", "draft"):
        if b[name] is not None:
            b[name] = (b[name] * (largest / 10 if largest < 100 else 1.0) + (largest - 8 if largest >= 100 else 0)).to(dtype)
    b["temps"] = torch.full((6,), heat)
    for i, tree in enumerate(b["parents"]):
        for r, p in enumerate(tree):
            if p >= 0:
                row, kind = b["firsts"][i] + p, rng.random()
                x = b["draft"] if drafted and kind > 0.6 else b["logits"]
                b["tokens"][b["firsts"][i] + r] = int(x[row].argmax() if kind < 0.8 else x[row].argmin())
    return b


TINY = [1e-3, 1e-6, 3e-8, 1e-8, 2e-9, 1e-9, 1e-12, 1e-20, 1e-30, 1e-40]


@pytest.mark.parametrize("heat", TINY)
@pytest.mark.parametrize("largest", [5.0, 20.0, 100.0, 1e4])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("drafted", [False, True])
def test_next_to_zero(heat, largest, masked, drafted):
    b = batch(1e-5 if drafted and heat == 1e-3 else heat, largest, drafted, masked)      # (at 1e-3 some drafts have probabilities of 1e-300)
    check(b)
    best = b["logits"].argmax(-1).tolist()
    path, accepted, following = run(b)
    for i, (a, n) in enumerate(zip(b["firsts"], accepted)):
        if n and heat <= 1e-20 and not drafted:           # greedy but for equal logits
            x = b["logits"][a + path[a + n - 1]]
            assert x[following[i]] == x[best[a + path[a + n - 1]]]


@pytest.mark.parametrize("heat", [1e-8, 1e-20])
@pytest.mark.parametrize("drafted", [False, True])
def test_next_to_zero_in_bfloat16(heat, drafted):
    check(batch(heat, 20.0, drafted, False, torch.bfloat16))


@pytest.mark.parametrize("heat", [1e6, 1e30, 4e35, 6e35, 1e37, 3e38])
@pytest.mark.parametrize("drafted", [False, True])
def test_next_to_infinity(heat, drafted):
    """Every token that is not masked is as likely as any other; the masked ones have no probability."""
    b = make(SHAPES, 5001, torch.float32, 22, drafted, [1.0] * 6, agree=0.0, masked=True)
    b["temps"] = torch.full((6,), heat)
    check(b)
    path, accepted, following = run(b)
    for i, (a, n) in enumerate(zip(b["firsts"], accepted)):
        if n:
            assert b["logits"][a + path[a + n - 1], following[i]] > -np.inf


def test_an_infinite_temperature():
    b = make([(3, 1)] * 40, 4097, torch.float32, 23, False, [float("inf")] * 40, agree=0.0)
    b["logits"][:, 1000:] = -float("inf")
    _, accepted, following = run(b)
    assert all(0 <= t < 1000 for t in following)
    for i, (a, n) in enumerate(zip(b["firsts"], accepted)):
        if n == 1:
            assert following[i] == int(float(b["uniform"][a, 1]) * 1000)
