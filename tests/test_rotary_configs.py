"""rotary_inv_freq with what configurations hold beside the scaling's dict
(each value from the formula, in Python's 64 bits)."""

import math

import pytest
import torch

from lmcache_amd import formats


def _inv(dim, base=10000.0):
    return base ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)


def test_longrope_without_factor():
    """Frequencies' factors in the dict, both contexts beside it."""
    cfg = {"type": "longrope", "short_factor": [1.0, 1.5], "long_factor": [2.0, 5.0]}
    inv, scale = formats.rotary_inv_freq(4, scaling=cfg, seq_len=4097, max_position_embeddings=131072,
                                         original_max_position_embeddings=4096)
    assert torch.equal(inv, _inv(4) / torch.tensor([2.0, 5.0], dtype=torch.float64))
    assert abs(scale - math.sqrt(1 + math.log(32) / math.log(4096))) < 1e-14
    # The dict's own entries come first.
    own = dict(cfg, original_max_position_embeddings=8192)
    inv, scale = formats.rotary_inv_freq(4, scaling=own, seq_len=8192, max_position_embeddings=131072,
                                         original_max_position_embeddings=4096)
    assert torch.equal(inv, _inv(4) / torch.tensor([1.0, 1.5], dtype=torch.float64))
    assert abs(scale - math.sqrt(1 + math.log(16) / math.log(8192))) < 1e-14
    assert formats.rotary_inv_freq(4, scaling=dict(own, factor=4.0), max_position_embeddings=131072)[1] == \
        math.sqrt(1 + math.log(4) / math.log(8192))
    assert formats.rotary_inv_freq(4, scaling=dict(own, attention_factor=1.25))[1] == 1.25
    # A context that is no longer than the original one.
    assert formats.rotary_inv_freq(4, scaling=own, max_position_embeddings=8192)[1] == 1.0


def test_dynamic_without_original_context():
    cfg = {"rope_type": "dynamic", "factor": 4.0}
    inv, scale = formats.rotary_inv_freq(8, 10000.0, cfg, 6000, max_position_embeddings=2048)
    base = 10000.0 * (4.0 * 6000 / 2048 - 3.0) ** (8 / 6)
    assert scale == 1.0 and torch.allclose(inv, _inv(8, base), rtol=1e-14)
    assert torch.equal(formats.rotary_inv_freq(8, 10000.0, cfg, 2048, max_position_embeddings=2048)[0], _inv(8))


def test_yarn_without_original_context():
    cfg = {"rope_type": "yarn", "factor": 4.0}
    given = formats.rotary_inv_freq(64, 1e6, dict(cfg, original_max_position_embeddings=32768))
    beside = formats.rotary_inv_freq(64, 1e6, cfg, max_position_embeddings=32768)
    assert torch.equal(given[0], beside[0]) and given[1] == beside[1]
    other = formats.rotary_inv_freq(64, 1e6, cfg, max_position_embeddings=131072, original_max_position_embeddings=32768)
    assert torch.equal(given[0], other[0])


@pytest.mark.parametrize("scaling,more", [
    ({"rope_type": "dynamic", "factor": 2.0}, {}),
    ({"rope_type": "yarn", "factor": 2.0}, {}),
    ({"rope_type": "longrope", "short_factor": [1.0] * 4, "long_factor": [1.0] * 4}, {}),
    ({"rope_type": "longrope", "short_factor": [1.0] * 4, "long_factor": [1.0] * 4}, {"original_max_position_embeddings": 64}),
    ({"rope_type": "dynamic"}, {"max_position_embeddings": 64}),
])
def test_what_is_nowhere_is_refused(scaling, more):
    with pytest.raises(ValueError, match="scaling needs"):
        formats.rotary_inv_freq(8, 10000.0, scaling, **more)
