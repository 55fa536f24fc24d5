"""Trees of drafted tokens as the host lays them out, and drafts that the text itself gives."""
import random

import numpy as np
import pytest

import tree_plain as plain
from glassbox_b200.engine.drafts import PromptLookup
from glassbox_b200.engine.engine import tree_layout


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 64, 100])
def test_layout(rows):
    parents = plain.random_tree(random.Random(rows), rows, 3)
    depths, bits, chain = tree_layout(tuple(parents))
    assert depths.tolist() == plain.depths(parents)
    assert np.array_equal(bits.view(np.int32), plain.words(plain.ancestors(parents), -(-rows // 32)))
    assert chain == (parents == list(range(-1, rows - 1)))


@pytest.mark.parametrize("parents", [(), (0,), (-1, -1), (-1, 1), (-1, 0, 2), (-1, 0, -2)])
def test_what_is_no_tree(parents):
    with pytest.raises(ValueError):
        tree_layout(parents)


def paths(tokens, parents):
    """The texts of the leaves."""
    out = []
    for i in range(len(tokens)):
        if i not in parents:
            at, text = i, []
            while at > 0:
                text.append(tokens[at])
                at = parents[at]
            out.append(text[::-1])
    return out


def test_lookup_takes_what_followed_before():
    text = [1, 2, 3, 7, 8, 9, 5, 1, 2, 3, 7, 6, 4, 1, 2, 3]
    tokens, parents = PromptLookup(tokens=3, match=3, branches=1).propose(text, 10)
    assert tokens == [3, 7, 6, 4] and parents == [-1, 0, 1, 2]
    tokens, parents = PromptLookup(tokens=3, match=3, branches=2).propose(text, 10)
    assert tokens[0] == 3 and paths(tokens, parents) == [[7, 6, 4], [7, 8, 9]]      # (7 is shared)
    tree_layout(tuple(parents))
    for room in range(6):
        tokens, parents = PromptLookup(tokens=3, match=3, branches=2).propose(text, room)
        assert len(tokens) <= room + 1
        tree_layout(tuple(parents))


def test_lookup_without_anything_to_find():
    assert PromptLookup().propose([4], 5) == ([4], [-1])
    assert PromptLookup().propose([1, 2, 3, 4], 5) == ([4], [-1])
    assert PromptLookup().propose([4, 4], 5) == ([4, 4], [-1, 0])
    for bad in (dict(tokens=0), dict(match=0), dict(branches=0)):
        with pytest.raises(ValueError):
            PromptLookup(**bad)
