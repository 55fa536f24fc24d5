"""Verification of drafted tokens against a plain walk in float64."""
import random

import numpy as np
import pytest
import torch

import tree_plain as plain
from glassbox_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True, params=[False, True], ids=["all rows", "the walk's rows"])
def either_way(request, monkeypatch):
    monkeypatch.setattr(kernels, "verify_walks", lambda *sizes: request.param)


def make(shapes, vocab, dtype, seed, drafted, temps, agree=0.7, odd=0, masked=False):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    firsts, parents = [0], []
    for rows, width in shapes:
        parents.append(plain.random_tree(rng, rows, width) if rows else [])
        firsts.append(firsts[-1] + rows)
    n = firsts[-1]
    logits = torch.randn(n, vocab, generator=g) * 2
    if masked:
        logits[torch.rand(n, vocab, generator=g) < 0.7] = -float("inf")
        logits[:, vocab // 3] = 1.0
    tokens = torch.randint(0, vocab, (n,), generator=g)
    draft = None
    if drafted:
        draft = (logits + torch.randn(n, vocab, generator=g)).to(dtype)
        for i, tree in enumerate(parents):
            for r, p in enumerate(tree):
                if p >= 0:
                    t = temps[i] if temps[i] > 0 else 1.0
                    q = torch.softmax(draft[firsts[i] + p].double() / t, -1)
                    tokens[firsts[i] + r] = torch.multinomial(q, 1, generator=g)
    else:
        for i, tree in enumerate(parents):
            for r, p in enumerate(tree):
                if p >= 0 and rng.random() < agree:       # one of the children is what the model likes
                    logits[firsts[i] + p, tokens[firsts[i] + r]] = 8.0 + rng.random()
    if odd:                                               # rows that start `odd` numbers behind a multiple of 16 bytes
        place = lambda x: torch.cat([torch.zeros(n, odd, dtype=dtype), x.to(dtype), torch.zeros(n, 1, dtype=dtype)], 1).to(DEV)[:, odd:odd + vocab]
    else:
        place = lambda x: x.to(dtype).to(DEV)
    uniform = torch.rand(n, 2, generator=g)
    return dict(firsts=firsts, parents=parents, tokens=tokens, logits=place(logits), draft=None if draft is None else place(draft), uniform=uniform,
                temps=torch.tensor(temps, dtype=torch.float32), vocab=vocab)


def run(b):
    n, s = len(b["tokens"]), len(b["temps"])
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    flat = [p for tree in b["parents"] for p in tree]
    path, accepted, following = torch.full((n,), 99, dtype=torch.int32, device=DEV), as_int([99] * s), as_int([99] * s)
    kernels.verify_tree(b["logits"], b["tokens"].to(torch.int32).to(DEV), as_int(flat), as_int(b["firsts"]), b["uniform"].to(DEV), b["temps"].to(DEV), path, accepted,
                        following, b["draft"])
    return path.tolist(), accepted.tolist(), following.tolist()


def check(b):
    path, accepted, following = run(b)
    logits = b["logits"].float().cpu().numpy()
    draft = None if b["draft"] is None else b["draft"].float().cpu().numpy()
    total = 0
    for i, tree in enumerate(b["parents"]):
        a, e = b["firsts"][i], b["firsts"][i + 1]
        if not tree:
            assert accepted[i] == 0 and following[i] == -1
            continue
        kept, token = plain.verify(logits[a:e], b["tokens"][a:e].tolist(), tree, b["uniform"][a:e].numpy(), float(b["temps"][i]), None if draft is None else draft[a:e])
        assert path[a:e] == kept + [-1] * (e - a - len(kept)), f"request {i}"
        assert (accepted[i], following[i]) == (len(kept), token), f"request {i}"
        total += len(kept)
    return total


SHAPES = [(8, 3), (1, 1), (5, 1), (0, 1), (33, 4), (2, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 4096, 49152, 100003])
@pytest.mark.parametrize("temps", [[0.0] * 6, [0.8] * 6, [1.0, 0.0, 0.3, 1.0, 2.0, -1.0]])
@pytest.mark.parametrize("drafted", [False, True])
def test_against_the_walk(dtype, vocab, temps, drafted):
    check(make(SHAPES, vocab, dtype, vocab + len(SHAPES), drafted, temps))


@pytest.mark.parametrize("dtype,odd", [(torch.float32, 1), (torch.float32, 3), (torch.bfloat16, 1), (torch.bfloat16, 5), (torch.bfloat16, 7)])
@pytest.mark.parametrize("drafted", [False, True])
def test_rows_at_odd_places(dtype, odd, drafted):
    check(make(SHAPES, 5001, dtype, odd, drafted, [0.7] * 6, odd=odd))
    check(make(SHAPES, 5001, dtype, odd, drafted, [0.0] * 6, odd=odd))


@pytest.mark.parametrize("seqs", [1, 19, 40, 80, 200, 310])
@pytest.mark.parametrize("drafted", [False, True])
def test_batches(seqs, drafted):
    """Clusters of every size."""
    rng = random.Random(seqs)
    kept = check(make([(rng.randint(1, 7), rng.choice([1, 3])) for _ in range(seqs)], 33000 if seqs < 50 else 9000, torch.float32, seqs, drafted,
                      [rng.choice([0.0, 0.5, 1.0]) for _ in range(seqs)]))
    assert kept > seqs or seqs == 1


@pytest.mark.parametrize("drafted", [False, True])
def test_parts_that_have_no_probability(drafted):
    check(make(SHAPES, 7001, torch.float32, 5, drafted, [0.9] * 6, masked=True))
    check(make(SHAPES, 7001, torch.float32, 5, drafted, [0.0] * 6, masked=True))


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24])
@pytest.mark.parametrize("drafted", [False, True])
def test_the_ends_of_the_random_numbers(u, drafted):
    b = make(SHAPES, 3001, torch.float32, 6, drafted, [0.9] * 6, masked=True)
    b["uniform"][:] = u
    check(b)


def test_flat_and_steep_rows():
    b = make([(6, 2)] * 4, 50000, torch.float32, 7, False, [1.0, 1e-3, 100.0, 1.0], agree=0.0)
    b["logits"][:6] = 0.0
    b["logits"][18:, 1000:] = -80.0
    check(b)


def test_equal_logits_take_the_lowest_id():
    b = make([(4, 3)] * 2, 2000, torch.bfloat16, 8, False, [0.0, 0.0])
    b["logits"][:] = b["logits"].round().clamp(-2, 2)
    b["logits"][4, 5] = 0.0
    check(b)


def test_rows_that_are_no_distribution():
    for drafted in (False, True):
        b = make([(3, 1)] * 6, 3000, torch.float32, 9, drafted, [1.0, 1.0, 1.0, 0.0, 0.0, 0.0])
        x = b["logits"]
        x[0, 77], x[3, 2999], x[6] = float("nan"), float("inf"), -float("inf")
        x[9, 77], x[12], x[15] = float("nan"), float("nan"), -float("inf")
        check(b)
        path, accepted, following = run(b)
        assert following[:3] == [-1] * 3 and following[4] == -1 and accepted[:3] == [1] * 3
    b = make([(3, 1)] * 2, 3000, torch.float32, 9, True, [1.0, 1.0])
    b["draft"][0] = -float("inf")
    b["draft"][3, 5] = float("nan")
    check(b)
    assert run(b)[2] == [-1, -1]


def test_drafts_equal_to_the_model_are_taken():
    """Every row's first child, so that the walk ends at a leaf."""
    b = make([(6, 1)] * 8, 5000, torch.float32, 10, True, [1.0] * 8)
    b["draft"] = b["logits"].clone()
    check(b)
    walks = []
    for tree in b["parents"]:
        walks.append([0])
        while walks[-1][-1] in tree:
            walks[-1].append(tree.index(walks[-1][-1]))
    assert run(b)[1] == [len(w) for w in walks]


def test_the_same_child_twice_and_tokens_outside():
    b = make([(5, 4)], 1000, torch.float32, 11, False, [0.0])
    b["parents"] = [[-1, 0, 0, 0, 2]]
    top = int(b["logits"][0].argmax())
    b["tokens"][:] = torch.tensor([3, top + 1, top, top, 4])
    check(b)
    assert run(b)[0][:2] == [0, 2]
    for temps in ([0.0], [1.0]):
        for drafted in (False, True):
            b = make([(4, 3)], 1000, torch.float32, 12, drafted, temps)
            b["parents"] = [[-1, 0, 0, 0]]
            b["tokens"][1:3] = torch.tensor([-5, 1000])
            check(b)


def test_what_comes_out_is_distributed_as_the_model(seqs=20000):
    """The first token behind a row, whatever was drafted: frequencies against the model's probabilities (a chi-square of 11 degrees: 45 is passed once in 2e5)."""
    g = torch.Generator().manual_seed(13)
    vocab = 12
    x, y = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    for parents in ([-1, 0], [-1, 0, 0, 0]):
        rows = len(parents)
        n = rows * seqs
        draft = y.repeat(n, 1)
        b = dict(firsts=list(range(0, n + 1, rows)), parents=[parents] * seqs, tokens=torch.multinomial(torch.softmax(y.double(), -1), n, True, generator=g), vocab=vocab,
                 logits=x.repeat(n, 1).to(DEV), draft=draft.to(DEV), uniform=torch.rand(n, 2, generator=g), temps=torch.ones(seqs))
        path, accepted, following = run(b)
        first = [int(b["tokens"][i * rows + path[i * rows + 1]]) if accepted[i] > 1 else following[i] for i in range(seqs)]
        want = torch.softmax(x.double(), -1).numpy() * seqs
        chi = ((np.bincount(first, minlength=vocab) - want) ** 2 / want).sum()
        assert chi < 45, chi


def test_recorded():
    b = make(SHAPES, 20000, torch.float32, 14, True, [0.9] * 6)
    want = run(b)
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    n, s = len(b["tokens"]), 6
    args = [b["logits"], b["tokens"].to(torch.int32).to(DEV), as_int([p for tree in b["parents"] for p in tree]), as_int(b["firsts"]), b["uniform"].to(DEV), b["temps"].to(DEV)]
    path, accepted, following = as_int([9] * n), as_int([9] * s), as_int([9] * s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.verify_tree(*args, path, accepted, following, b["draft"])
    for _ in range(3):
        path.fill_(9), accepted.fill_(9), following.fill_(9)
        graph.replay()
        assert (path.tolist(), accepted.tolist(), following.tolist()) == want
