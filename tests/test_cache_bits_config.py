"""Which models' caches can be kept in 4 bits, as configurations say it."""
import dataclasses
from types import SimpleNamespace

import pytest

from conftest import tiny_raw
from glassbox_b200.config import ConfigError
from glassbox_b200.config.registry import parse_config
from glassbox_b200.config.specs import with_cache_bits


def config():
    return parse_config(tiny_raw("D"))


def test_every_layer_keeps_4_bits():
    before = config()
    after = with_cache_bits(before, 4)
    assert [layer.mixer.cache_bits for layer in after.layers] == [4] * len(before.layers)
    assert all(layer.mixer.cache_bits is None for layer in before.layers)


@pytest.mark.parametrize("layer", [SimpleNamespace(arrangement="of its own"), SimpleNamespace(mixer=None), SimpleNamespace(mixer=SimpleNamespace(kind="mingru"))], ids=str)
def test_layers_without_such_attention_are_refused(layer):
    """... with a configuration's error, also where a layer has no mixer at all."""
    before = config()
    with pytest.raises(ConfigError, match="layer 1"):
        with_cache_bits(dataclasses.replace(before, layers=(before.layers[0], layer)), 4)
