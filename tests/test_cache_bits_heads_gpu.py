"""Whole models with the cache in 4 bits at the head sizes whose prompts take other kernels: against the plain implementation, and single tokens
beside portions of prompts against the same tokens alone."""
import random

import numpy as np
import pytest
import torch

import glassbox_b200
from glassbox_b200 import kernels
from glassbox_b200.models.llama import make_llama_raw_config
from plain import llama_plain
from test_cache_bits_gpu import ELSE, SHARE, make_engine, plain_logits

pytestmark = pytest.mark.gpu

VOCAB = 300


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    made = {}

    def get(hd, dtype, heads=3, kv_heads=1):
        key = (hd, dtype, heads, kv_heads)
        if key not in made:
            folder = str(tmp_path_factory.mktemp(f"heads{heads}_{hd}_{dtype}"))
            raw = make_llama_raw_config(hidden_size=128, intermediate_size=208, num_hidden_layers=2, num_attention_heads=heads,
                                        num_key_value_heads=kv_heads, head_dim=hd, vocab_size=VOCAB, rope_theta=100000.0, rms_norm_eps=1e-5, tie_word_embeddings=True,
                                        max_position_embeddings=320)
            glassbox_b200.write_random_model(folder, raw, 11, torch.float32 if dtype == "float32" else torch.bfloat16)
            made[key] = folder
        return made[key]

    return get


def step(eng, *entries):
    from glassbox_b200.engine.engine import StepEntry
    return eng.step([StepEntry(*e) for e in entries])


# (what is allowed: as for heads of 32 and 64, beside SHARE and ELSE)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [96, 128, 256])
def test_logits(folders, monkeypatch, hd, dtype):
    folder = folders(hd, dtype)
    toks = [random.Random(2).randrange(VOCAB) for _ in range(150)]
    want = plain_logits(folder, toks, monkeypatch)
    eng, rows = make_engine(folder, dtype), []
    eng.add_request("a")
    for a, b in ((0, 70), (70, 100), (100, 101), (101, 140)):
        rows.append(step(eng, ("a", toks[a:b], list(range(b - a)))).cpu().numpy())
    for t in toks[140:]:
        rows.append(step(eng, ("a", [t], [0])).cpu().numpy())
    eng.check()
    got = np.concatenate(rows)
    effect = np.abs(want - llama_plain.forward_logits(folder, toks))
    spread, diff = want.std(), np.abs(got - want)
    assert diff.max() <= SHARE[dtype] * effect.max() + ELSE[dtype][0] * spread, (diff.max() / spread, effect.max() / spread)
    assert diff.mean() <= SHARE[dtype] * effect.mean() + ELSE[dtype][1] * spread, (diff.mean() / spread, effect.mean() / spread)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads, kv_heads, hd", [(3, 1, 32), (24, 24, 32), (3, 1, 64), (3, 1, 96), (24, 24, 96), (3, 1, 128), (3, 1, 256)])
def test_single_tokens_beside_prompts(folders, heads, kv_heads, hd, dtype):
    """Three times, so that the later ones replay what was recorded; every row of the mixed step is compared with the request's own."""
    folder = folders(hd, dtype, heads, kv_heads)
    rng = random.Random(4)
    toks = {r: [rng.randrange(VOCAB) for _ in range(120)] for r in "abcd"}
    alone = {}
    for r in "abcd":
        eng = make_engine(folder, dtype, use_graphs=False)
        eng.add_request(r)
        step(eng, (r, toks[r][:40], []))
        alone[r] = step(eng, (r, toks[r][40:41], [0]) if r in "ab" else (r, toks[r][40:110], [0, 35, 69])).clone()
    eng = make_engine(folder, dtype)
    for again in range(3):
        for r in "abcd":
            eng.add_request(r)
        step(eng, *[(r, toks[r][:40], []) for r in "abcd"])
        got = step(eng, *[(r, toks[r][40:41], [0]) for r in "ab"], *[(r, toks[r][40:110], [0, 35, 69]) for r in "cd"]).clone()
        eng.check()
        for r, a, b in (("a", 0, 1), ("b", 1, 2), ("c", 2, 5), ("d", 5, 8)):
            eng.free_request(r)
            spread = float(alone[r].std())
            # (in bfloat16 another order of a sum moves a rounding of the activations, and with it now and then a code)
            assert float((got[a:b] - alone[r]).abs().max()) <= (1e-3 if dtype == "float32" else 0.12) * spread, (r, again)
    assert eng.graph_replays > 0


@pytest.mark.parametrize("hd", [32, 96])
def test_prompts_of_many_rows_and_heads_work_on_tiles_of_rows(folders, monkeypatch, hd):
    """... of the engine's own queries, which are columns of wider rows; few rows and heads are faster row by row."""
    calls = []
    exact = kernels.sink_attention_tiles
    monkeypatch.setattr(kernels, "sink_attention_tiles", lambda *a, **k: (calls.append(a[0].shape[0]), exact(*a, **k))[1])
    for heads, rows, want in ((24, 130, [130, 130]), (24, 16, []), (3, 130, [])):
        eng = make_engine(folders(hd, "bfloat16", heads, heads), "bfloat16", use_graphs=False)
        eng.add_request("a")
        calls.clear()
        step(eng, ("a", [1 + i % 200 for i in range(rows)], [rows - 1]))
        eng.check()
        assert calls == want
