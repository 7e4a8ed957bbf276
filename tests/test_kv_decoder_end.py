"""LlamaDecoder at the end of its 8-bit key/value cache."""

import pytest
import torch

from nibble_amd.llama import LlamaDecoder
from tests.test_kv_decoder import _cfg, _prompt


@pytest.mark.parametrize("kv_cache", ["int8", "fp8", "fp16"])
def test_generation_past_the_cache_is_refused(kv_cache):
    """Where the fp16 cache raises, at the latest at the step that has no slot;
    a cache that is exactly full works."""
    model = LlamaDecoder(_cfg(max_seq_len=16, kv_cache=kv_cache), device="cpu", seed=0)
    full = model.generate(_prompt(10), 7, use_graph=False)
    assert full.numel() == 7 and int(model.position) == 16 and torch.isfinite(model.logits).all()
    assert model.generate(_prompt(16), 1, use_graph=False).numel() == 1
    for prompt, tokens in ((10, 8), (16, 2), (1, 17), (10, 20)):
        with pytest.raises(IndexError):
            model.generate(_prompt(prompt), tokens, use_graph=False)
    assert torch.equal(model.generate(_prompt(10), 7, use_graph=False), full)


@pytest.mark.parametrize("kv_cache", ["int8", "fp8"])
def test_step_past_the_cache_is_refused(kv_cache):
    model = LlamaDecoder(_cfg(max_seq_len=16, kv_cache=kv_cache), device="cpu", seed=0)
    model.prefill(_prompt(15))
    model.step()
    caches = [t.clone() for c in model.kv_caches for t in c.tensors()]
    state = [model.token.clone(), model.position.clone()]
    with pytest.raises(IndexError, match="longer than the key/value cache"):
        model.step()
    assert model.host_position == 16
    assert all(torch.equal(a, b) for a, b in zip(state, (model.token, model.position)))
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(caches, (t for c in model.kv_caches for t in c.tensors())))
    model.prefill(_prompt(3))
    model.step()


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache", ["int8", "fp8"])
def test_graphs_past_the_cache_are_refused(gpu, kv_cache):
    model = LlamaDecoder(_cfg(max_seq_len=32, kv_cache=kv_cache), device=gpu, seed=2)
    prompt = _prompt(20).to(gpu)
    want = model.generate(prompt, 13, use_graph=False)
    model.capture()
    model.capture_prefill(20)
    assert torch.equal(model.generate(prompt, 13), want) and int(model.position) == 32
    for call in (model.replay, model.step, model.replay_tokens, lambda: model.generate(prompt, 14),
                 lambda: model.prefill(_prompt(33).to(gpu)), lambda: model.capture_prefill(33)):
        with pytest.raises(IndexError, match="longer than the key/value cache"):
            call()
    assert torch.equal(model.generate(prompt, 13), want)   # the captured prompt is the one of before
