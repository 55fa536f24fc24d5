"""Drafted generation on the CPU, with stand-ins for the engines: drafting models of other kinds than the model they draft for, and what happens when something
runs out."""
import numpy as np
import pytest

import draft_fakes as fakes
import tree_plain as plain
from glassbox_b200.engine import drafts
from glassbox_b200.sampling.sampler import Sampler, SamplerConfig

VOCAB = 11


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(drafts.kernels, "sample", fakes.sample)


def likes(text):
    return (sum(text) * 7 + len(text) * 3 + text[-1]) % VOCAB


def logits_of(text):
    x = np.cos(np.arange(VOCAB) * (1 + likes(text)))
    x[likes(text)] = 2.0
    return x


def nearly(text):
    """A drafting model that is wrong behind every third text or so."""
    x = logits_of(text)
    if (sum(text) + len(text)) % 3 == 0:
        x[(likes(text) + 1) % VOCAB] = 3.0
    return x


def alone(prompt, count, temperature, seed, most=64):
    """The text that comes token by token."""
    text, rng = list(prompt), Sampler(SamplerConfig(seed=seed)).rng
    while len(text) < len(prompt) + count and (len(text) < most or len(text) == len(prompt)):
        x = logits_of(text).astype(np.float32)
        text.append(plain.draw(plain.softmax(x, temperature), rng.next_f32()) if temperature > 0 else int(x.argmax()))
    return text[len(prompt):]


PROMPTS = [[1, 2, 3, 4, 5], [6], [7, 8, 9, 1, 2, 3, 4, 5, 6]]


def run(model, target=None, prompts=PROMPTS, count=30, temperature=0.0, **kw):
    target = target or fakes.FakeEngine(VOCAB, logits_of)
    outs, reasons, counts = drafts.generate(target, prompts, count, model, SamplerConfig(temperature=temperature, seed=3), **kw)
    assert not target.cache.request_ids()
    if isinstance(model, drafts.DraftModel):
        assert not model.engine.cache.request_ids()
    return outs, counts


def small(**kw):
    return drafts.DraftModel(fakes.FakeEngine(VOCAB, nearly, **kw), tokens=4)


@pytest.mark.parametrize("kind", [dict(state=True), dict(window=3, page_size=2), dict(window=3, page_size=2, state=True)])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_models_that_cannot_go_back_draft_alike(kind, temperature):
    """What was drafted and not kept is no part of what comes next, whatever the drafting model carries along."""
    want, plain_counts = run(small(), temperature=temperature)
    got, counts = run(small(**kind), temperature=temperature)
    assert got == want and counts == plain_counts and 0 < counts.accepted < counts.drafted
    if not temperature:
        assert got == [alone(p, 30, 0.0, 0) for p in PROMPTS]


def test_a_drafting_model_of_a_shorter_context():
    got, counts = run(small(max_position=16))
    assert got == [alone(p, 30, 0.0, 0) for p in PROMPTS] and counts.accepted > 0
    got, counts = run(small(max_position=4))
    assert got == [alone(p, 30, 0.0, 0) for p in PROMPTS]
    assert drafts.generate(fakes.FakeEngine(VOCAB, logits_of), PROMPTS, 30, small(max_position=16), SamplerConfig(temperature=0.7))[0]


@pytest.mark.parametrize("budget", [1, 2, 3])
def test_a_drafting_model_of_a_small_budget(budget):
    want, plain_counts = run(small())
    assert run(small(budget=budget)) == (want, plain_counts)
    want = run(small(), temperature=0.7)
    assert run(small(budget=budget), temperature=0.7) == want


def test_a_drafting_model_holds_as_many_requests_as_run_at_once():
    two = fakes.FakeEngine(VOCAB, logits_of, max_requests=2)
    assert run(small(max_requests=2), two, max_seqs=8)[0] == [alone(p, 30, 0.0, 0) for p in PROMPTS]
    two = fakes.FakeEngine(VOCAB, logits_of, budget=2)
    assert run(small(max_requests=2), two)[0] == [alone(p, 30, 0.0, 0) for p in PROMPTS]
    with pytest.raises(ValueError, match="requests"):
        run(small(max_requests=2))


def test_pages_run_out_where_nothing_was_drafted():
    """The drafting model is at its last position; the last request waits and is read again."""
    prompts = [[1, 2, 3, 4, 5, 6, 7, 8, 9], [9, 8, 7, 6, 5, 4, 3, 2, 1]]
    few = fakes.FakeEngine(VOCAB, logits_of, pages=5, page_size=4)
    got, _ = run(small(max_position=9), few, prompts, 3, 0.7)
    assert got == [alone(p, 3, 0.7, 3 + i) for i, p in enumerate(prompts)]


@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_a_prompt_that_fills_the_context(temperature):
    """One token follows it, as without drafts."""
    prompts = [[1 + i % 9 for i in range(n)] for n in (16, 15, 14)]
    full = lambda: fakes.FakeEngine(VOCAB, logits_of, max_position=16)
    want = [alone(p, 30, temperature, 3 + i, most=16) for i, p in enumerate(prompts)]
    assert [len(w) for w in want] == [1, 1, 2]
    assert run(drafts.PromptLookup(), full(), prompts, temperature=temperature)[0] == want
    got = run(small(max_position=16), full(), prompts, temperature=temperature)[0]
    assert [len(o) for o in got] == [1, 1, 2] and got[0] == want[0]
    assert temperature or got == want                     # (what was drafted is drawn with other numbers)


@pytest.mark.parametrize("pages", [16, 17, 20, 24])
def test_a_request_that_waits_for_pages_is_not_read_over_and_over(pages):
    prompts = [[1 + (i * j) % 9 for i in range(32)] for j in (1, 2, 3)]
    few = fakes.FakeEngine(VOCAB, logits_of, pages=pages, page_size=4, budget=8)
    got, _ = run(drafts.PromptLookup(tokens=2), few, prompts, 24)
    assert got == [alone(p, 24, 0.0, 0) for p in prompts]
    assert sum(n for step in few.log for _, n in step) <= 3 * sum(32 + 24 for _ in prompts)


@pytest.mark.parametrize("pages", [3, 9, 14, 20])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_a_drafting_model_whose_pages_do_not_hold_every_text(pages, temperature):
    """The texts that fit are drafted for, the others go on without, and none is read in every step."""
    prompts = [[1 + (i * j) % 9 for i in range(20)] for j in (1, 2, 3, 4)]
    model = small(pages=pages, page_size=4, budget=8)
    got, counts = run(model, prompts=prompts, count=24, temperature=temperature)
    assert temperature or got == [alone(p, 24, 0.0, 0) for p in prompts]
    assert counts.accepted > 0 or pages < 7
    assert sum(n for step in model.engine.log for _, n in step if n > 1) <= 3 * sum(20 + 24 for _ in prompts)
