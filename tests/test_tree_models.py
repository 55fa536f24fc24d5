"""Which models take trees of drafted tokens, and what the others' refusal says."""
import pytest

import felovik_util
import tagenex_util
from conftest import tiny_raw
from glassbox_b200.config.registry import parse_config
from glassbox_b200.config.specs import with_cache_bits
from glassbox_b200.engine.model import DecoderModel


def test_grouped_query_attention_takes_them():
    assert DecoderModel(parse_config(tiny_raw("D"))).takes_trees
    four = DecoderModel(with_cache_bits(parse_config(tiny_raw("D")), 4))
    assert not four.takes_trees and four.why_no_trees() == "not built for GqaAttention over a cache in 4 bits"


@pytest.mark.parametrize("raw,part,other", [(felovik_util.CONFIGS["even"], "StateSpace", "BranchNormBlock"), (tagenex_util.CONFIGS["odd"], "BranchNormBlock", "StateSpace")])
def test_the_refusal_names_the_parts(raw, part, other):
    model = DecoderModel(parse_config(raw()))
    assert not model.takes_trees
    said = model.why_no_trees()
    assert part in said and other not in said and "GqaAttention" not in said and "4 bits" not in said
