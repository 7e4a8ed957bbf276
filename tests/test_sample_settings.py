"""``LlamaDecoder.sample`` with a value of a setting for each sequence."""

import pytest
import torch

from nibble_amd import llama
from nibble_amd.llama import LlamaDecoder
from tests.test_sample_decoder import _cfg, _numbers, _prompt


def _settings(n, device="cpu"):
    """One value a sequence of each setting; greedy and unlimited ones among them."""
    spread = lambda *values: torch.tensor([values[i % len(values)] for i in range(n)], device=device)  # noqa: E731
    return dict(temperature=spread(0.9, 0.0, 1.3), top_k=spread(3, 0, 2, 5), top_p=spread(0.9, 1.0),
                min_p=spread(0.0, 0.0, 0.05, 0.0, 0.2))


def _check_eos(free, got, eos):
    for row, want in zip(got.tolist(), free.tolist()):
        end = want.index(eos) if eos in want else len(want)
        assert row[:end] == want[:end] and all(t == eos for t in row[end:])


@pytest.mark.parametrize("shared", [False, True])
def test_each_sequence_has_its_own(shared, monkeypatch):
    """A sequence is the one that its settings give where all have them."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers, settings = _numbers(6, 8), _settings(6)
    got = model.sample(_prompt(9), 8, sequences=6, random=numbers, **settings)
    for b in range(6):
        alike = model.sample(_prompt(9), 8, sequences=6, random=numbers, **{k: v[b].item() for k, v in settings.items()})
        assert torch.equal(got[b], alike[b])


@pytest.mark.parametrize("sequences", [1, 6])
def test_settings_move_up_with_the_sequences(sequences, monkeypatch):
    monkeypatch.setattr(llama, "EOS_STRIDE", 2)
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    numbers, settings = _numbers(sequences, 12), _settings(sequences)
    calls = []
    reorder = llama.QuantizedKVCache.reorder
    monkeypatch.setattr(llama.QuantizedKVCache, "reorder", lambda self, *a: (calls.append(a), reorder(self, *a))[1])
    free = model.sample(_prompt(9), 12, sequences=sequences, random=numbers, **settings)
    moved = 0
    for eos in sorted(set(free.flatten().tolist())):     # each token that comes
        calls.clear()
        _check_eos(free, model.sample(_prompt(9), 12, sequences=sequences, random=numbers, eos=eos, **settings), eos)
        moved += bool(calls)
    assert sequences == 1 or moved


@pytest.mark.parametrize("sequences", [1, 3])
@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
def test_other_lengths_are_refused_before_anything_runs(name, sequences):
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    whole = torch.int64 if name == "top_k" else torch.float32
    for n in (sequences + 1, 0):
        with pytest.raises(ValueError, match=name):
            model.sample(_prompt(9), 4, sequences=sequences, **{name: torch.ones((n,), dtype=whole)})
    with pytest.raises(ValueError, match=name):
        model.sample(_prompt(9), 4, sequences=sequences, **{name: torch.ones((), dtype=whole)})
    assert model.host_position == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
def test_gpu_settings(gpu, shared, monkeypatch):
    """Captured steps draw what eager ones draw, also once sequences have moved up."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    monkeypatch.setattr(llama, "EOS_STRIDE", 4)
    monkeypatch.setattr(llama, "MOVED_ROWS", 0)
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    prompt, numbers, settings = _prompt(33, device="cuda"), _numbers(7, 40, device="cuda"), _settings(7, "cuda")
    free = model.sample(prompt, 40, sequences=7, random=numbers, **settings)
    assert torch.equal(model.sample(prompt, 40, sequences=7, random=numbers, use_graph=False, **settings), free)
    eos = int(free.flatten().mode().values)
    kw = dict(sequences=7, random=numbers, eos=eos, **settings)
    assert torch.equal(model.sample(prompt, 40, **kw), model.sample(prompt, 40, use_graph=False, **kw))
