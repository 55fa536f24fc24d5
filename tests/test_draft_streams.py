"""The random numbers of drafted generation, on the CPU: what is drafted, whether it is taken, and what is drawn in its place depend on numbers that have nothing
to do with one another, whatever the seeds."""
import numpy as np
import pytest

import draft_fakes as fakes
from glassbox_b200.engine import drafts
from glassbox_b200.sampling.sampler import SamplerConfig

VOCAB = 12


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(drafts.kernels, "sample", fakes.sample)


def engines(**kw):
    g = np.random.default_rng(13)
    x, y = g.standard_normal(VOCAB), g.standard_normal(VOCAB)
    return x, fakes.FakeEngine(VOCAB, lambda text: x, **kw), fakes.FakeEngine(VOCAB, lambda text: y, **kw)


def chi_square(tokens, x):
    p = np.exp(x - x.max())
    want = p / p.sum() * len(tokens)
    return (((np.bincount(tokens, minlength=VOCAB) - want) ** 2) / want).sum()


@pytest.mark.parametrize("draft_seed", ["the run's", "default", "another"])
def test_sampled_text_has_the_models_distribution(draft_seed, runs=3000):
    """Chi-squares of 11 degrees: 45 is passed once in 2e5."""
    x, target, small = engines()
    first, second = [], []
    for seed in range(runs):
        model = drafts.DraftModel(small, tokens=4, **({} if draft_seed == "default" else dict(seed=seed if draft_seed == "the run's" else seed + 10 ** 6)))
        (tokens,), _, _ = drafts.generate(target, [[1]], 2, model, SamplerConfig(temperature=1.0, seed=seed))
        first.append(tokens[0])
        second.append(tokens[1])
    assert chi_square(first, x) < 45 and chi_square(second, x) < 45


def test_requests_of_a_run_under_default_seeds(requests=3000):
    x, target, small = engines()
    outs, _, counts = drafts.generate(target, [[1]] * requests, 2, drafts.DraftModel(small), SamplerConfig(temperature=1.0))
    assert counts.drafted > counts.accepted > 0
    assert chi_square([o[0] for o in outs], x) < 45 and chi_square([o[1] for o in outs], x) < 45


def test_a_run_begins_anew_and_a_request_has_numbers_of_its_own():
    x, target, small = engines()
    model = drafts.DraftModel(small, tokens=3, seed=5)
    cfg = lambda seed: SamplerConfig(temperature=1.0, seed=seed)
    many, _, _ = drafts.generate(target, [[1], [2], [3]], 9, model, cfg(5))
    assert drafts.generate(target, [[1], [2], [3]], 9, model, cfg(5))[0] == many
    for i, prompt in enumerate([[1], [2], [3]]):
        assert drafts.generate(target, [prompt], 9, model, cfg(5 + i))[0] == [many[i]]
    assert drafts.generate(target, [[1], [2], [3]], 9, model, cfg(77))[0] != many
    drafts.generate(target, [[1]], 3, drafts.DraftModel(small, seed=-7), cfg(-3))


def test_the_numbers_of_any_two_uses_have_nothing_to_do_with_one_another():
    """Means, and products of what two streams give, over seeds and places that differ by little: within six deviations."""
    streams = {}
    for what in (1, 2):
        for seeds in ((0, 0), (0, 1), (1, 0), (2 ** 32, 0), (0, -1)):
            for at in (1, 2, 3):
                x = drafts._numbers(what, seeds, at, 4000)
                assert x.dtype == np.float32 and 0 <= x.min() and x.max() < 1
                streams[what, seeds, at] = (x.astype(np.float64) - 0.5) * 12 ** 0.5
    all_of = np.array(list(streams.values()))
    assert abs(all_of.mean(1)).max() < 6 / 4000 ** 0.5 and abs((all_of ** 2).mean(1) - 1).max() < 6 * 0.8 ** 0.5 / 4000 ** 0.5
    products = all_of @ all_of.T / 4000 - np.eye(len(all_of)) * (all_of ** 2).mean(1)
    assert abs(products).max() < 6 / 4000 ** 0.5
    for shift in (1, 2, 5):
        assert abs(all_of[:, shift:] @ all_of[:, :-shift].T / (4000 - shift)).max() < 6 / (4000 - shift) ** 0.5
