"""Rotary settings of Hugging Face configs, where they stand in one dict."""

import pytest
import torch

from nibble_amd import model_checkpoint as mc
from nibble_amd.llama import LlamaDecoder

BASE = dict(vocab_size=256, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
            max_position_embeddings=4096)
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 512}


@pytest.mark.parametrize("parameters,scaled", [({**LLAMA3, "rope_theta": 5e5}, True),
                                               ({"rope_type": "default", "rope_theta": 5e5}, False)])
def test_theta_beside_the_scaling(parameters, scaled):
    cfg = mc.decoder_config({**BASE, "rope_parameters": parameters}, 64, rope_scaling=True)
    assert cfg.rope_theta == 5e5 and (cfg.rope_scaling is not None) is scaled
    split = {**BASE, "rope_theta": 5e5, **({"rope_scaling": LLAMA3} if scaled else {})}
    want = LlamaDecoder(mc.decoder_config(split, 64, rope_scaling=True), device="cpu")
    got = LlamaDecoder(cfg, device="cpu")
    assert torch.equal(got.cos, want.cos) and torch.equal(got.inv_freq, want.inv_freq)
    # an entry of its own comes first; without rope_scaling configs keep what they gave
    assert mc.decoder_config({**BASE, "rope_theta": 2e4, "rope_parameters": parameters}, 64,
                             rope_scaling=True).rope_theta == 2e4
    assert mc.decoder_config({**BASE, "rope_parameters": parameters}, 64).rope_theta == 10000.0
    assert mc.decoder_config({**BASE, "rope_parameters": None}, 64, rope_scaling=True).rope_theta == 10000.0


def test_theta_of_an_installed_config():
    transformers = pytest.importorskip("transformers")
    config = transformers.LlamaConfig(hidden_size=256, num_attention_heads=4, rope_theta=5e5)
    assert mc.decoder_config(config.to_dict(), 64, rope_scaling=True).rope_theta == 5e5
