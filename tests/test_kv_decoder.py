"""LlamaDecoder over an 8-bit key/value cache and with scaled rotary positions."""

import dataclasses

import pytest
import torch

from nibble_amd import kv_reference, rope_tables
from nibble_amd import model_checkpoint as mc
from nibble_amd.llama import LlamaConfig, LlamaDecoder
from tests import _kv


def _cfg(**changes):
    base = LlamaConfig(vocab_size=512, hidden_size=512, intermediate_size=1280, num_layers=2, num_heads=8,
                       num_kv_heads=2, head_dim=64, max_seq_len=96, kv_cache="int8", kv_block=32)
    return dataclasses.replace(base, **changes)


def _prompt(n, seed=1):
    return torch.randint(0, 512, (n,), generator=_kv.gen(seed))


# -------------------------------------------------------------------------------- CPU

@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_cpu_decoder_is_near_the_fp16_cache(codes):
    """Two tokens after a prompt. A code is off by at most half a step: int8
    2^-8 of its block's largest value or less, e4m3 2^-4 of itself; the logits,
    whose attention part averages such errors, are asked for 5% of their size."""
    cfg = _cfg(kv_cache=codes, head_dim=32, num_heads=16, num_kv_heads=4)
    model = LlamaDecoder(cfg, device="cpu", seed=3)
    exact = LlamaDecoder(dataclasses.replace(cfg, kv_cache="fp16"), device="cpu", seed=3)
    assert model.k_cache.numel() == 0 and model.kv_caches[0].k_codes.dtype == _kv.CODES[codes]
    prompt = _prompt(9)
    with torch.inference_mode():
        for m in (model, exact):
            m.prefill(prompt)
            m.token.fill_(7)
            m.step()
    diff = (model.logits.float() - exact.logits.float()).norm() / exact.logits.float().norm()
    assert diff < 0.05
    assert int(model.position) == 10


def test_cpu_decoder_recomputes_the_same_prefix():
    """A restart reuses the cache without clearing it."""
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    first = model.generate(_prompt(5), 4, use_graph=False)
    assert torch.equal(model.generate(_prompt(5), 4, use_graph=False), first)


def test_configs():
    with pytest.raises(ValueError, match="kv_cache"):
        LlamaDecoder(_cfg(kv_cache="int4"), device="cpu")
    with pytest.raises(ValueError, match="block_size"):
        LlamaDecoder(_cfg(kv_block=24), device="cpu")
    with pytest.raises(ValueError, match="unknown rope scaling"):
        LlamaDecoder(_cfg(rope_scaling={"rope_type": "other"}), device="cpu")
    with pytest.raises(IndexError, match="longer"):
        LlamaDecoder(_cfg(max_seq_len=8), device="cpu").prefill(_prompt(9))
    plain = LlamaDecoder(_cfg(kv_cache="fp16"), device="cpu")
    assert plain.kv_caches is None and plain.k_cache.shape[2] == 96


def test_checkpoint_configs():
    base = dict(vocab_size=256, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                max_position_embeddings=4096)
    assert mc.decoder_config(base).rope_scaling is None and mc.decoder_config(base).kv_cache == "fp16"
    assert mc.decoder_config(base, 64, kv_cache="fp8").kv_cache == "fp8"
    scaled = lambda config, slots=2048: mc.decoder_config(config, slots, rope_scaling=True).rope_scaling
    assert scaled(base) is None
    assert scaled({**base, "rope_parameters": {"rope_type": "default", "rope_theta": 1e4}}) is None
    llama = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 512}
    assert scaled({**base, "rope_scaling": llama}) == llama
    assert mc.decoder_config({**base, "rope_scaling": llama}).rope_scaling is None
    assert scaled({**base, "rope_scaling": {"type": "dynamic", "factor": 2.0}}, 8192)[
        "original_max_position_embeddings"] == 4096
    with pytest.raises(ValueError, match="longrope"):
        LlamaDecoder(mc.decoder_config({**base, "rope_scaling": {"type": "longrope"}}, 64, rope_scaling=True), device="cpu")


def test_scaled_positions_reach_the_tables():
    scaling = {"rope_type": "linear", "factor": 4.0}
    model = LlamaDecoder(_cfg(kv_cache="fp16", rope_scaling=scaling), device="cpu", seed=3)
    cos, sin = rope_tables(64, 96, 1e4, scaling)
    assert torch.equal(model.cos, cos) and torch.equal(model.sin, sin)
    assert torch.allclose(model.inv_freq, LlamaDecoder(_cfg(kv_cache="fp16"), device="cpu").inv_freq / 4, rtol=2.0 ** -22)


# -------------------------------------------------------------------------------- GPU

gpu_only = pytest.mark.gpu


@gpu_only
@pytest.mark.parametrize("codes,changes", [("int8", {}), ("fp8", {}), ("int8", dict(num_heads=4, head_dim=128)),
                                           ("fp8", dict(num_heads=2, num_kv_heads=1, head_dim=256)),
                                           ("int8", dict(rope_scaling={"rope_type": "yarn", "factor": 2.0,
                                                                       "original_max_position_embeddings": 48})),
                                           ("int8", dict(max_seq_len=1500))])
@pytest.mark.parametrize("length", [1, 12, 70])
def test_fused_step_matches_torch_step(gpu, codes, changes, length):
    """Prompt and step through the fused launches against the torch-op path
    around the same cache operators, on the logits: |err| <= 2e-2 (1 + |ref|),
    the bar of the fp16 decoder's test."""
    model = LlamaDecoder(_cfg(kv_cache=codes, **changes), device=gpu, seed=0)
    assert model.fused and not model.attn_o
    prompt = _prompt(length).to(gpu)
    logits = []
    for fused in (False, True):
        model.fused = fused
        model.prefill(prompt)
        model.token.fill_(3)
        if fused:
            model.x_buf.copy_(model.embed[3])
        model.step()
        logits.append(model.logits.float().cpu())
        assert int(model.position) == length + 1
    assert torch.isfinite(logits[1]).all()
    assert torch.all((logits[1] - logits[0]).abs() <= 2e-2 * (1 + logits[0].abs()))


@gpu_only
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("max_seq_len", [96, 2048])
def test_graph_generation(gpu, codes, max_seq_len):
    """Captured steps and a captured prompt give the eager tokens, twice."""
    model = LlamaDecoder(_cfg(kv_cache=codes, max_seq_len=max_seq_len), device=gpu, seed=2)
    prompt = _prompt(20).to(gpu)
    want = model.generate(prompt, 40, use_graph=False).cpu()
    model.capture(tokens_per_replay=4)
    assert torch.equal(model.generate(prompt, 40).cpu(), want)
    model.capture_prefill(20)
    for _ in range(2):
        assert torch.equal(model.generate(prompt, 40).cpu(), want)


@gpu_only
def test_gpu_prompt_matches_cpu(gpu):
    """The first layer's cache after a prompt against the CPU path on the same
    weights: its keys and values come from projections whose fp32 sums differ
    in their order, an fp16 step at most, which moves a code by one where it
    lies at a border."""
    model = LlamaDecoder(_cfg(), device=gpu, seed=0)
    ref = LlamaDecoder(_cfg(), device="cpu", init="empty")
    ref.load_state_dict({k: v.detach().cpu() for k, v in model.state_dict().items()})
    prompt = _prompt(12)
    model.prefill(prompt.to(gpu))
    ref.prefill(prompt)
    a, b = model.kv_caches[0], ref.kv_caches[0]
    for x, y in ((a.k_codes, b.k_codes), (a.v_codes, b.v_codes)):
        assert (x[:, :, :12].cpu().int() - y[:, :, :12].int()).abs().max() <= 1
    assert int(model.position) == int(ref.position) == 12


@gpu_only
def test_gpu_refuses_other_head_dims(gpu):
    with pytest.raises(ValueError, match="head_dim"):
        LlamaDecoder(_cfg(head_dim=32, num_heads=16), device=gpu)


@gpu_only
@pytest.mark.parametrize("length", [10, 300])
def test_scaled_fp16_decoder(gpu, length):
    """A factor on the tables keeps the steps that rotate by inv_freq alone off."""
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
    model = LlamaDecoder(_cfg(kv_cache="fp16", max_seq_len=512, rope_scaling=yarn), device=gpu, seed=0)
    assert model.fused and not model.attn_o
    prompt = _prompt(length).to(gpu)
    logits = []
    for fused in (False, True):
        model.fused = fused
        model.prefill(prompt)
        model.token.fill_(3)
        if fused:
            model.x_buf.copy_(model.embed[3])
        model.step()
        logits.append(model.logits.float().cpu())
    assert torch.all((logits[1] - logits[0]).abs() <= 2e-2 * (1 + logits[0].abs()))
    assert kv_reference.block_size(512, 8) == 64
