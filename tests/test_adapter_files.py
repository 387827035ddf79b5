"""Adapters' files that mean more than two products added to the model's own
weights are refused."""

import pytest
import torch

from test_serving_decode import _pair, _write

NAME = "model.layers.0.self_attn.q_proj"


@pytest.mark.parametrize("config", [
    {"init_lora_weights": "pissa"}, {"init_lora_weights": "pissa_niter_16"}, {"init_lora_weights": "olora"},
    {"init_lora_weights": "corda"}, {"init_lora_weights": "loftq"}, {"init_lora_weights": "lora_ga"}, {"lora_bias": True}, {"use_qalora": True},
    {"layer_replication": [[0, 4], [2, 5]]}, {"alora_invocation_tokens": [5, 6]}, {"trainable_token_indices": [1]},
    {"target_parameters": ["mlp.experts"]}])
def test_adapters_of_other_weights_are_refused(tmp_path, config):
    from turbopress_amd.lora import LoraAdapters
    with pytest.raises(ValueError, match=next(iter(config))):
        LoraAdapters.load([_write(tmp_path / "a", {NAME: _pair(torch.Generator().manual_seed(0), 4, 6, 10)}, config)], torch.float16, "cpu")


@pytest.mark.parametrize("config", [{}, {"init_lora_weights": True}, {"init_lora_weights": False}, {"init_lora_weights": "gaussian"},
                                    {"init_lora_weights": None, "lora_bias": False, "layer_replication": None, "alora_invocation_tokens": None}])
def test_plain_adapters_are_loaded(tmp_path, config):
    from turbopress_amd.lora import LoraAdapters
    pair = _pair(torch.Generator().manual_seed(0), 4, 6, 10)
    got = LoraAdapters.load([_write(tmp_path / "a", {NAME: pair}, config)], torch.float16, "cpu")
    assert torch.equal(got.stacks[NAME][0][0], pair[0]) and torch.equal(got.stacks[NAME][1][0], pair[1])
