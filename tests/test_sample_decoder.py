"""``LlamaDecoder.sample``: one sequence, several that share a prompt, and their end."""

import dataclasses

import pytest
import torch

from nibble_amd import llama
from nibble_amd.llama import LlamaConfig, LlamaDecoder
from nibble_amd.sampling import sample
from tests import _kv


def _cfg(**changes):
    base = LlamaConfig(vocab_size=512, hidden_size=512, intermediate_size=1280, num_layers=2, num_heads=8,
                       num_kv_heads=2, head_dim=64, max_seq_len=160, kv_cache="int8", kv_block=32)
    return dataclasses.replace(base, **changes)


def _prompt(n, seed=1, device="cpu"):
    return torch.randint(0, 512, (n,), generator=_kv.gen(seed)).to(device)


def _numbers(n, steps, seed=2, device="cpu"):
    return torch.rand((n, steps), generator=_kv.gen(seed)).to(device)


# -------------------------------------------------------------------------------- CPU

@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_greedy_is_generate(cache):
    model = LlamaDecoder(_cfg(kv_cache=cache), device="cpu", seed=3)
    want = model.generate(_prompt(9), 6, use_graph=False)
    assert torch.equal(model.sample(_prompt(9), 6, temperature=0.0)[0], want)


@pytest.mark.parametrize("shared", [False, True])
def test_greedy_sequences_are_generate(shared, monkeypatch):
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    want = model.generate(_prompt(9), 5, use_graph=False)
    got = model.sample(_prompt(9), 5, sequences=3, temperature=0.0)
    assert got.shape == (3, 5) and torch.equal(got, want.expand(3, -1))
    assert int(model.position) == 9      # the decoder's own state stays behind the prompt


def test_first_tokens_are_drawn_from_the_prompts_logits():
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers = _numbers(40, 2)
    got = model.sample(_prompt(9), 2, sequences=40, temperature=1.5, top_k=30, random=numbers)
    model.prefill(_prompt(9))
    want = sample(model.logits.unsqueeze(0).expand(40, -1), numbers[:, 0].contiguous(), temperature=1.5, top_k=30)
    assert torch.equal(got[:, 0], want) and len(set(want.tolist())) > 3


@pytest.mark.parametrize("shared", [False, True])
def test_sequences_do_not_depend_on_each_other(shared, monkeypatch):
    """The same numbers give the same sequence, whatever the others draw."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers = _numbers(4, 5)
    first = model.sample(_prompt(9), 5, sequences=4, top_p=0.9, random=numbers)
    other = numbers.flip(0).contiguous()
    assert torch.equal(model.sample(_prompt(9), 5, sequences=4, top_p=0.9, random=other), first.flip(0))


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("sequences", [1, 6])
def test_eos(shared, sequences, monkeypatch):
    """Sequences end at their first eos; the others move up and go on as before."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    monkeypatch.setattr(llama, "EOS_STRIDE", 2)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers = _numbers(sequences, 12)
    calls = []
    reorder = llama.QuantizedKVCache.reorder
    monkeypatch.setattr(llama.QuantizedKVCache, "reorder", lambda self, *a: (calls.append(a), reorder(self, *a))[1])
    free = model.sample(_prompt(9), 12, sequences=sequences, top_k=3, random=numbers)
    eos = int(free.flatten().mode().values)       # a token that comes often
    got = model.sample(_prompt(9), 12, sequences=sequences, top_k=3, random=numbers, eos=eos)
    for row, want in zip(got.tolist(), free.tolist()):
        end = want.index(eos) if eos in want else len(want)
        assert row[:end] == want[:end] and all(t == eos for t in row[end:])
    assert sequences == 1 or calls


def test_eos_of_more_sequences_than_a_cache_is_reordered_with(monkeypatch):
    """The ended ones run on beside the others."""
    monkeypatch.setattr(llama, "EOS_STRIDE", 2)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers = _numbers(6, 12)
    free = model.sample(_prompt(9), 12, sequences=6, top_k=3, random=numbers)
    eos = int(free.flatten().mode().values)
    want = model.sample(_prompt(9), 12, sequences=6, top_k=3, random=numbers, eos=eos)
    monkeypatch.setattr(llama, "REORDER_VALUES_MAX", 5 * model.cfg.head_dim)
    monkeypatch.setattr(llama.QuantizedKVCache, "reorder", None)
    assert torch.equal(model.sample(_prompt(9), 12, sequences=6, top_k=3, random=numbers, eos=eos), want)


def test_refusals():
    model = LlamaDecoder(_cfg(max_seq_len=16), device="cpu")
    plain = LlamaDecoder(_cfg(kv_cache="fp16", max_seq_len=16), device="cpu")
    for error, call in [(ValueError, lambda: plain.sample(_prompt(4), 2, sequences=2)),
                        (ValueError, lambda: model.sample(_prompt(4), 0)),
                        (ValueError, lambda: model.sample(_prompt(4), 2, sequences=0)),
                        (ValueError, lambda: model.sample(_prompt(4), 2, random=torch.zeros(2, 2))),
                        (ValueError, lambda: model.sample(_prompt(4), 2, temperature=-1.0)),
                        (IndexError, lambda: model.sample(_prompt(4), 14)),
                        (IndexError, lambda: plain.sample(_prompt(4), 14))]:
        with pytest.raises(error):
            call()
    assert model.sample(_prompt(4), 13).shape == (1, 13)
    assert model.sample(_prompt(4), 1, sequences=3).shape == (3, 1)


# -------------------------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_gpu_one_sequence(gpu, cache):
    """Eager and captured steps draw the same tokens; greedy ones are generate's."""
    model = LlamaDecoder(_cfg(kv_cache=cache), device="cuda", seed=3)
    prompt, numbers = _prompt(9, device="cuda"), _numbers(1, 20, device="cuda")
    assert torch.equal(model.sample(prompt, 8, temperature=0.0)[0], model.generate(prompt, 8, use_graph=False))
    eager = model.sample(prompt, 20, top_p=0.95, random=numbers, use_graph=False)
    model.prefill(prompt)
    model.capture()
    assert torch.equal(model.sample(prompt, 20, top_p=0.95, random=numbers), eager)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [2, 5, 17, 40])
@pytest.mark.parametrize("codes,dim", [("int8", 64), ("fp8", 128)])
@pytest.mark.parametrize("shared", [False, True])
def test_gpu_sequences(gpu, shared, codes, dim, sequences, monkeypatch):
    """Captured steps draw what eager ones draw; equal numbers give equal sequences."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(kv_cache=codes, head_dim=dim, num_heads=512 // dim, num_kv_heads=2), device="cuda", seed=3)
    prompt, numbers = _prompt(33, device="cuda"), _numbers(sequences, 12, device="cuda")
    numbers[1] = numbers[0]
    eager = model.sample(prompt, 12, sequences=sequences, temperature=0.9, top_k=100, top_p=0.9, random=numbers,
                         use_graph=False)
    assert torch.equal(eager[0], eager[1])
    assert torch.equal(model.sample(prompt, 12, sequences=sequences, temperature=0.9, top_k=100, top_p=0.9,
                                    random=numbers), eager)


@pytest.mark.gpu
def test_gpu_shared_and_forked_logits(gpu, monkeypatch):
    """The two ways of keeping the prompt give nearly the same logits: the codes of the
    tokens behind it differ by a step where they share a block's scale with its last
    tokens (asked for 5% of their size, as caches of different codes are)."""
    seen = []
    forward = LlamaDecoder._rows_forward
    monkeypatch.setattr(LlamaDecoder, "_rows_forward", lambda self, *a: (seen.append(forward(self, *a)), seen[-1])[1])
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    for limit in (0, 1 << 40):
        monkeypatch.setattr(llama, "FORK_BYTES_MAX", limit)
        model.sample(_prompt(50, device="cuda"), 3, sequences=4, temperature=0.0, use_graph=False)
    for a, b in zip(seen[:2], seen[2:]):
        assert (a.float() - b.float()).norm() <= 0.05 * b.float().norm()


@pytest.mark.gpu
def test_gpu_eos(gpu, monkeypatch):
    monkeypatch.setattr(llama, "EOS_STRIDE", 4)
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    prompt, numbers = _prompt(9, device="cuda"), _numbers(8, 24, device="cuda")
    free = model.sample(prompt, 24, sequences=8, top_k=3, random=numbers)
    eos = int(free.flatten().mode().values)
    got = model.sample(prompt, 24, sequences=8, top_k=3, random=numbers, eos=eos)
    for row in got.tolist():
        end = row.index(eos) if eos in row else len(row)
        assert all(t == eos for t in row[end:])
    # until the first ones have moved up the same launches run
    assert torch.equal(got[:, :4], torch.where((free[:, :4] == eos).cumsum(dim=1) > 0, eos, free[:, :4]))
