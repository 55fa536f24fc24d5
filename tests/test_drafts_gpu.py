"""Whole models with drafted tokens: steps of trees against the plain implementation, what the cache keeps, and generation against generation token by token."""
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

import tree_plain as plain
from conftest import ROOT, TINY, assert_logits_close
from plain import llama_plain

pytestmark = pytest.mark.gpu


def make_engine(folder, dtype, **kw):
    from glassbox_b200.engine.engine import Engine
    kw.setdefault("cache_tokens", 1024)
    kw.setdefault("max_batch_tokens", 256)
    return Engine(folder, dtype, **kw)


def text_of(text, tokens, parents, row):
    up = []
    while row >= 0:
        up.append(tokens[row])
        row = parents[row]
    return text + up[::-1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])          # (heads of 16, 32, 48 and 64)
@pytest.mark.parametrize("graphs", [True, False])
def test_logits_of_trees(model_dirs, name, dtype, graphs):
    """Every row's logits are those of the text that leads to it; steps of one shape are recorded and replayed."""
    from glassbox_b200.engine.engine import StepEntry
    folder, vocab = model_dirs(name, dtype), TINY[name]["vocab_size"]
    rng = random.Random(3)
    eng = make_engine(folder, dtype, use_graphs=graphs)
    texts = {"a": [rng.randrange(vocab) for _ in range(37)], "b": [rng.randrange(vocab) for _ in range(16)], "c": []}
    for rid, text in texts.items():
        eng.add_request(rid)
        if text:
            eng.step([StepEntry(rid, text)])
    for turn in range(3):
        entries, trees = [], {"a": plain.random_tree(rng, 9, 3), "b": None, "c": plain.random_tree(rng, 5, 2)}
        for rid, tree in trees.items():
            count = len(tree) if tree else 4
            entries.append(StepEntry(rid, [rng.randrange(vocab) for _ in range(count)], list(range(count)), tree))
        got = eng.step(entries, commit=False).cpu().numpy()
        at = 0
        for e in entries:
            tree = e.parents or list(range(-1, len(e.tokens) - 1))
            for r in range(len(e.tokens)):
                want = llama_plain.forward_logits(folder, text_of(texts[e.request], e.tokens, tree, r))[-1]
                assert_logits_close(got[at:at + 1], want[None], dtype, f"{name} {e.request} row {r} turn {turn}")
                at += 1
    assert (eng.graph_replays > 0) == graphs
    eng.check()


@pytest.mark.parametrize("name", ["A", "D"])
def test_what_is_kept_is_as_if_decoded(model_dirs, name):
    """Trees around what a greedy model writes: its own tokens are kept, the cache then gives the logits of that text."""
    from glassbox_b200.engine.engine import StepEntry
    folder, vocab = model_dirs(name, "float32"), TINY[name]["vocab_size"]
    rng = random.Random(4)
    eng = make_engine(folder, "float32")
    text = [rng.randrange(vocab) for _ in range(20)]
    eng.add_request("x")
    eng.step([StepEntry("x", text[:-1])])
    for turn in range(5):
        ahead, own = [], list(text)
        for _ in range(4):
            ahead.append(int(llama_plain.forward_logits(folder, own)[-1].argmax()))
            own.append(ahead[-1])
        # wrong turns beside the right way, which lies at rows 2, 4 and 7; its fourth token is not drafted
        parents = [-1, 0, 0, 1, 2, 2, 3, 4, 4]
        tokens = [text[-1]] + [(ahead[d - 1] + 1 + r) % vocab for r, d in enumerate(plain.depths(parents)[1:])]
        for row, t in zip((2, 4, 7), ahead):
            tokens[row] = t
        for r in range(1, 9):
            if r not in (2, 4, 7) and tokens[r] == ahead[plain.depths(parents)[r] - 1]:
                tokens[r] = (tokens[r] + 1) % vocab
        kept, = eng.verify_step([StepEntry("x", tokens, parents=parents)])
        assert kept.rows == [0, 2, 4, 7] and kept.tokens == ahead[:3] and kept.next_token == ahead[3]
        text = own
        assert eng.cache.tokens("x") == text[:-1]
        eng.cache.check_invariants()
        logits = eng.step([StepEntry("x", [text[-1]], [0])], commit=False).cpu().numpy()
        assert_logits_close(logits, llama_plain.forward_logits(folder, text)[-1:], "float32", f"turn {turn}")
    eng.check()


def test_forks_write_their_own_pages(model_dirs):
    from glassbox_b200.engine.engine import StepEntry
    folder, vocab = model_dirs("D", "float32"), TINY["D"]["vocab_size"]
    rng = random.Random(5)
    eng = make_engine(folder, "float32")
    text = [rng.randrange(vocab) for _ in range(21)]
    eng.add_request("x")
    eng.step([StepEntry("x", text[:-1])])
    eng.fork("x", "y")
    trees = [[-1, 0, 0, 1, 2], [-1, 0, 0, 0, 1]]
    entries = [StepEntry(rid, [text[-1]] + [rng.randrange(vocab) for _ in range(4)], parents=t) for rid, t in zip("xy", trees)]
    kept = eng.verify_step(entries, [1.0, 1.0], np.full((10, 2), 0.4, dtype=np.float32))
    for rid, k in zip("xy", kept):
        own = text + k.tokens + [k.next_token]
        got = eng.step([StepEntry(rid, [k.next_token], [0])], commit=False).cpu().numpy()
        assert_logits_close(got, llama_plain.forward_logits(folder, own)[-1:], "float32", rid)
    eng.cache.check_invariants()
    eng.check()


def repeating(rng, vocab, count):
    """A text that repeats itself, as code and quotations do."""
    part = [rng.randrange(vocab) for _ in range(7)]
    text = []
    while len(text) < count:
        text += part[:rng.randint(3, 7)]
    return text[:count]


@pytest.mark.parametrize("name", ["A", "D"])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_generation_is_the_models_own(model_dirs, name, temperature):
    """With drafts from the text: the tokens that come one by one, also for requests that draw (the same random numbers in the same places)."""
    import glassbox_b200
    from glassbox_b200.engine.drafts import PromptLookup
    vocab = TINY[name]["vocab_size"]
    rng = random.Random(6)
    prompts = [repeating(rng, vocab, n) for n in (30, 5, 1, 44, 16)]
    llm = glassbox_b200.load(model_dirs(name, "float32"), "float32", blocks=128, budget=64, max_seqs=3)
    want = llm.generate(prompts, 24, temperature=temperature, seed=7)
    for drafts in (PromptLookup(), PromptLookup(tokens=3, match=1, branches=5)):
        assert llm.generate(prompts, 24, temperature=temperature, seed=7, drafts=drafts) == want
        assert llm.draft_counts.drafted > 0
    assert llm.generate(prompts[0], 24, temperature=temperature, seed=7, drafts=PromptLookup()) == want[0]
    stop = want[0][3]
    assert llm.generate(prompts, 24, temperature=temperature, seed=7, stop=[stop], drafts=PromptLookup(), return_reasons=True) == \
        llm.generate(prompts, 24, temperature=temperature, seed=7, stop=[stop], return_reasons=True)
    assert not llm.engine.cache.request_ids()
    llm.engine.cache.check_invariants()


def test_a_model_that_drafts_for_its_twin(model_dirs):
    """The same weights in another engine: greedy drafts are all accepted, drawn ones nearly all; another model's text does not change the model's."""
    import glassbox_b200
    from glassbox_b200.engine.drafts import DraftModel
    folder, vocab = model_dirs("D", "float32"), TINY["D"]["vocab_size"]
    rng = random.Random(8)
    prompts = [[rng.randrange(vocab) for _ in range(n)] for n in (12, 3, 40)]
    llm = glassbox_b200.load(folder, "float32", blocks=128, budget=64, max_seqs=2)
    want = llm.generate(prompts, 20)
    twin = DraftModel(make_engine(folder, "float32", max_requests=2, max_batch_tokens=64), tokens=4)
    assert llm.generate(prompts, 20, drafts=twin) == want
    c = llm.draft_counts
    assert c.accepted == c.drafted and c.steps <= 3 * 5
    llm.generate(prompts, 20, temperature=1.0, drafts=twin)
    c = llm.draft_counts
    assert c.accepted >= 0.95 * c.drafted                  # (float32 logits of two kernels, one in thousands of which tips a coin)
    assert not twin.engine.cache.request_ids()
    other = DraftModel(make_engine(model_dirs("D", "float32", 12), "float32", max_requests=2, max_batch_tokens=64), tokens=3)
    assert llm.generate(prompts, 20, drafts=other) == want
    assert [len(o) for o in llm.generate(prompts, 20, temperature=0.7, drafts=other)] == [20] * 3


def test_when_pages_run_out(model_dirs):
    import glassbox_b200
    from glassbox_b200.engine.drafts import DraftModel, PromptLookup
    folder, vocab = model_dirs("D", "float32"), TINY["D"]["vocab_size"]
    rng = random.Random(9)
    prompts = [repeating(rng, vocab, n) for n in (40, 30, 20)]
    want = glassbox_b200.load(folder, "float32", blocks=128, budget=64, max_seqs=3).generate(prompts, 40)
    small = glassbox_b200.load(folder, "float32", blocks=9, budget=64, max_seqs=3, prefix_cache=False)
    assert small.generate(prompts, 40, drafts=PromptLookup()) == want
    few = DraftModel(make_engine(folder, "float32", num_pages=4, max_requests=3, max_batch_tokens=64), tokens=4)
    assert small.generate(prompts, 40, drafts=few) == want
    tiny = glassbox_b200.load(folder, "float32", blocks=3, budget=64, max_seqs=3, prefix_cache=False)
    outs, reasons = tiny.generate(prompts[2:], 40, drafts=PromptLookup(), return_reasons=True)
    assert reasons == ["length"] and outs[0] == want[2][:len(outs[0])] and 20 <= len(outs[0]) + 20 <= 49
    small.engine.cache.check_invariants()


def test_to_the_last_position(model_dirs):
    import glassbox_b200
    from glassbox_b200.engine.drafts import PromptLookup
    vocab, most = TINY["A"]["vocab_size"], TINY["A"]["max_position_embeddings"]
    prompt = repeating(random.Random(10), vocab, most - 10)
    llm = glassbox_b200.load(model_dirs("A", "float32"), "float32", blocks=32, budget=64, max_seqs=2)
    assert llm.generate(prompt, 50, drafts=PromptLookup(), return_reasons=True) == llm.generate(prompt, 50, return_reasons=True)
    assert llm.generate(prompt, 0, drafts=PromptLookup()) == []


def test_refusals(model_dirs):
    import glassbox_b200
    from glassbox_b200.engine.drafts import DraftModel, PromptLookup
    from glassbox_b200.engine.engine import StepEntry
    folder = model_dirs("D", "bfloat16")
    eng = make_engine(folder, "bfloat16")
    eng.add_request("x")
    ok = StepEntry("x", [1, 2, 3], parents=[-1, 0, 0])
    with pytest.raises(ValueError, match="commit"):
        eng.step([ok])
    with pytest.raises(ValueError, match="sampl"):
        eng.step([ok], commit=False, sampling=[])
    for bad in ([-1, 0], [0, 0, 0], [-1, 0, 2]):
        with pytest.raises(ValueError):
            eng.verify_step([StepEntry("x", [1, 2, 3], parents=bad)])
    with pytest.raises(ValueError, match="vocabulary"):
        eng.verify_step([StepEntry("x", [1, 300, 3])])
    with pytest.raises(ValueError, match="random"):
        eng.verify_step([ok], [0.5])
    with pytest.raises(ValueError):
        eng.verify_step([ok], [0.5], np.zeros((2, 2), np.float32))
    with pytest.raises(ValueError):
        eng.verify_step([ok], [0.5, 0.5])
    with pytest.raises(ValueError):
        eng.verify_step([ok], draft_logits=torch.zeros(3, 5, device="cuda"))
    assert eng.length("x") == 0 and eng.verify_step([ok])[0].rows[0] == 0
    eng.check()
    four = make_engine(folder, "bfloat16", cache_bits=4)
    four.add_request("x")
    with pytest.raises(ValueError, match="4 bits"):
        four.verify_step([ok])
    llm = glassbox_b200.load(folder, blocks=64, budget=64, max_seqs=2)
    with pytest.raises(ValueError, match="top_k"):
        llm.generate([1, 2], 3, temperature=1.0, top_k=5, drafts=PromptLookup())
    with pytest.raises(ValueError, match="itself"):
        llm.generate([1, 2], 3, drafts=DraftModel(llm.engine))
    with pytest.raises(ValueError, match="tokens"):
        llm.generate([1, 2], 3, drafts=DraftModel(make_engine(model_dirs("A", "bfloat16"), "bfloat16")))
    with pytest.raises(ValueError):
        DraftModel(eng, tokens=0)


def test_models_that_carry_something_from_row_to_row_are_refused(tmp_path):
    import felovik_util as fu
    from glassbox_b200.engine.engine import StepEntry
    cfg = fu.CONFIGS["even"]()
    eng = make_engine(fu.write_model(str(tmp_path / "m"), cfg, fu.random_weights(cfg, 1)), "bfloat16")
    eng.add_request("x")
    with pytest.raises(ValueError, match="drafted"):
        eng.verify_step([StepEntry("x", [1, 2, 3])])


def test_command_line(model_dirs):
    folder = model_dirs("D", "float32")
    base = [sys.executable, "-m", "glassbox_b200", "generate", "--model", folder, "--dtype", "f32", "--prompt", "5 6 7 8 5 6 7 8 5 6", "-n", "12", "--blocks", "64"]
    runs = [subprocess.run(base + extra, capture_output=True, text=True, cwd=ROOT) for extra in ([], ["--draft-lookup", "6"], ["--draft-model", folder, "--draft-tokens", "3"])]
    for r in runs:
        assert r.returncode == 0, r.stderr
    assert runs[0].stdout == runs[1].stdout == runs[2].stdout
    assert "drafted tokens accepted" in runs[1].stderr and "drafted tokens accepted" in runs[2].stderr


@pytest.mark.parametrize("held", ["pages", "slots", "pages later"])
def test_beside_requests_that_hold_the_cache(model_dirs, held):
    """What does not fit because of others is an error, and no text that ends early."""
    from glassbox_b200.cache.manager import OutOfPages
    from glassbox_b200.engine.drafts import PromptLookup, generate
    from glassbox_b200.engine.engine import StepEntry
    from glassbox_b200.sampling.sampler import SamplerConfig
    eng = make_engine(model_dirs("A", "float32"), "float32", cache_tokens=128, max_requests=1 if held == "slots" else 4)
    page = eng.page_size
    total = sum(eng.cache.free_pages(g) for g in range(1)) * page
    other = [1 + i % 7 for i in range(total - {"pages": 1, "slots": total - 3, "pages later": 2 * page + 1}[held])]
    eng.add_request("other")
    for a in range(0, len(other), 64):
        eng.step([StepEntry("other", other[a:a + 64])])
    with pytest.raises(OutOfPages):
        generate(eng, [[3, 4, 5, 3, 4]], 100, PromptLookup(3), SamplerConfig(temperature=0.0))
    assert eng.cache.request_ids() == ["other"] and eng.length("other") == len(other)
    eng.free_request("other")
    tokens, reasons, _ = generate(eng, [[3, 4, 5, 3, 4]], 5, PromptLookup(3), SamplerConfig(temperature=0.0))
    assert len(tokens[0]) == 5 and reasons == ["length"]
