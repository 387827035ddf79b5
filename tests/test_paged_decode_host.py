"""What the paged decoder and its tables decide on the host (no GPU)."""

import pytest
import torch


@pytest.mark.parametrize("keys", [{"mscale": 0.707, "mscale_all_dim": 0.707}, {"mscale": 1.0, "mscale_all_dim": 0.5},
                                  {"mscale": 0.7}, {"mscale_all_dim": 0.7}, {"mscale": 0.0, "mscale_all_dim": 1.0},
                                  {"mscale": 1.0, "mscale_all_dim": 0.4, "attention_factor": 1.2}, {"truncate": False}])
@pytest.mark.parametrize("factor", [8.0, 1.0])
def test_yarn_keys_match_transformers(keys, factor):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from turbopress_amd.paged import rotary_frequencies
    scaling = dict({"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": 4096}, **keys)
    cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=64, max_position_embeddings=int(4096 * factor),
                      rope_theta=1e4, rope_scaling=dict(scaling, rope_theta=1e4))
    want, want_factor = ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    got, got_factor = rotary_frequencies(64, 1e4, scaling)
    assert abs(got_factor - want_factor) < 1e-6
    assert ((got - want.double()).abs() <= 2.0 ** -21 * want.double()).all()
