"""When an engine with its cache in 4 bits allocates what grows with the cache: all of it when it is made."""
import pytest
import torch

import glassbox_b200
from glassbox_b200.models.llama import make_llama_raw_config

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads, hd, dtype", [(2, 64, "bfloat16"), (2, 128, "float32"), (24, 32, "bfloat16")])
def test_the_first_prompt_needs_no_memory_that_grows_with_the_cache(tmp_path, heads, hd, dtype):
    from glassbox_b200.engine.engine import Engine, StepEntry
    raw = make_llama_raw_config(hidden_size=128, intermediate_size=208, num_hidden_layers=2, num_attention_heads=heads, num_key_value_heads=heads,
                                head_dim=hd, vocab_size=300, rope_theta=100000.0, rms_norm_eps=1e-5, tie_word_embeddings=True, max_position_embeddings=320)
    glassbox_b200.write_random_model(str(tmp_path), raw, 3, torch.bfloat16)
    tokens = 100_000
    eng = Engine(str(tmp_path), dtype, cache_tokens=tokens, max_batch_tokens=256, max_requests=8, cache_bits=4)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    eng.add_request("a")
    eng.step([StepEntry("a", [1 + i % 200 for i in range(200)], [199])])
    eng.check()
    grown = torch.cuda.memory_allocated() - before
    unpacked = 2 * tokens * heads * hd * (2 if dtype == "bfloat16" else 4)
    # (activations of 256 + 8 + 128 rows: some thirty buffers of at most 3 heads hd numbers each)
    assert grown < unpacked / 2 and grown < 30 * 392 * 4 * (3 * heads * hd + 700), (grown, unpacked)
