"""Drafting models that carry a state or give pages back behind a window: what was drafted and not kept is no part of what they draft next."""
import random

import pytest

import felovik_util
import tagenex_util

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("util,name", [(felovik_util, "even"), (tagenex_util, "odd")], ids=["state", "window"])
def test_drafts_follow_from_the_text_alone(tmp_path, util, name):
    from glassbox_b200.engine.drafts import DraftModel
    from glassbox_b200.engine.engine import Engine
    cfg = util.CONFIGS[name]()
    eng = Engine(util.write_model(str(tmp_path / "m"), cfg, util.random_weights(cfg, 1)), "float32", cache_tokens=512, max_batch_tokens=64, max_requests=2)
    rng, model = random.Random(2), DraftModel(eng, tokens=6)
    text = [rng.randrange(cfg["vocab"]) for _ in range(50)]
    for kept in (0, 3, 1, 0, 6, 2):
        ((drafts, parents),), _ = model.propose_all(["a"], [text], [6], [0.0], [0])
        ((again, _),), _ = model.propose_all(["b"], [text], [6], [0.0], [0])
        model.drop("b")
        assert drafts == again and len(drafts) == 7 and parents == list(range(-1, 6))
        text = text + drafts[1:1 + kept] + [(drafts[min(kept + 1, 6)] + 1) % cfg["vocab"]]
    model.drop("a")
    eng.cache.check_invariants()
    eng.check()
