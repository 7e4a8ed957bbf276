"""``LlamaDecoder.sample`` once finished sequences have left the batch: those that move
up go on with their own keys, values and numbers."""

import pytest
import torch

from nibble_amd import llama
from nibble_amd.llama import LlamaDecoder
from tests.test_sample_decoder import _cfg, _numbers, _prompt

SEQUENCES, STEPS, EOS = 8, 26, 7
ENDS = [3, 99, 6, 99, 2, 17, 7, 14]      # the step at which a sequence draws eos: four leave at 8, two more at 20


def _forced(n, steps, device):
    """Numbers whose tokens, 512 times each, do not depend on the logits."""
    tokens = torch.randint(8, 512, (n, steps), generator=torch.Generator().manual_seed(5))
    for row, end in zip(tokens, ENDS):
        row[end:end + 1] = EOS
    return ((tokens + 0.5) / 512).to(device)


def _run(monkeypatch, model, device, most):
    """(tokens, the logits of each step, the sources of the sequences each time that some moved up);
    `most` sequences times head_dim are reordered."""
    logits, sources = [], []
    forward, reorder = LlamaDecoder._rows_forward, llama.QuantizedKVCache.reorder

    def spy_reorder(self, source, lengths):
        if self.k_codes.data_ptr() == first[0].k_codes.data_ptr():     # one layer's tell
            sources.append(source.tolist())
        return reorder(self, source, lengths)

    def spy_forward(self, tokens, caches, *rest):
        first[0] = caches[0]
        logits.append(forward(self, tokens, caches, *rest).float().cpu())
        return logits[-1].to(device, torch.float16)

    first = [None]
    with monkeypatch.context() as patch:
        patch.setattr(llama, "EOS_STRIDE", 4)
        patch.setattr(llama, "REORDER_VALUES_MAX", most)
        patch.setattr(llama, "MOVED_ROWS", 0)
        patch.setattr(llama, "sample", lambda x, random, **_: (random * 512).to(torch.int64))
        patch.setattr(LlamaDecoder, "_rows_forward", spy_forward)
        patch.setattr(llama.QuantizedKVCache, "reorder", spy_reorder)
        tokens = model.sample(_prompt(33, device=device), STEPS, sequences=SEQUENCES, eos=EOS, use_graph=False,
                              random=_forced(SEQUENCES, STEPS, device))
    return tokens.cpu(), logits, sources


def _check_moved(monkeypatch, device, shared, dim):
    """Against a run in which none moves up, with the same tokens whatever the logits are."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(head_dim=dim, num_heads=512 // dim), device=device, seed=3)
    tokens, logits, sources = _run(monkeypatch, model, device, 1 << 18)
    stayed, whole, none = _run(monkeypatch, model, device, 0)
    assert len(sources) == 2 and not none and torch.equal(tokens, stayed)
    rows, sizes = list(range(SEQUENCES)), []
    assert len(logits) == len(whole) == STEPS - 1
    for got, want in zip(logits, whole):
        if got.shape[0] != len(rows):
            rows = [rows[i] for i in sources.pop(0) if i >= 0]
        assert got.shape[0] == len(rows)
        sizes.append(len(rows))
        # Batches of another size round otherwise (2^-11 a value), and a key or value near the
        # middle of two codes may take the other one: a step, at most 2 / 127 of its block's
        # largest value, 5% of the values' size where the largest is three times that. (Planted
        # on the CPU: no reorder 0.44, the newest token left behind 0.16, another order 0.61.)
        for a, b in zip(got, want[rows]):
            assert (a - b).norm() <= 0.05 * b.norm()
    assert sizes == [8] * 7 + [4] * 12 + [2] * 6 and rows == [1, 3]


@pytest.mark.parametrize("shared", [False, True])
def test_moved_rows(shared, monkeypatch):
    _check_moved(monkeypatch, "cpu", shared, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_gpu_moved_rows(gpu, dim, shared, monkeypatch):
    _check_moved(monkeypatch, "cuda", shared, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("codes,dim", [("int8", 64), ("fp8", 128)])
def test_gpu_captured(gpu, codes, dim, shared, monkeypatch):
    """Steps captured anew once sequences have moved up draw what eager steps draw, to the end."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    monkeypatch.setattr(llama, "EOS_STRIDE", 4)
    monkeypatch.setattr(llama, "MOVED_ROWS", 0)
    moves = []
    reorder = llama.QuantizedKVCache.reorder
    monkeypatch.setattr(llama.QuantizedKVCache, "reorder", lambda self, *a: (moves.append(a), reorder(self, *a))[1])
    model = LlamaDecoder(_cfg(kv_cache=codes, head_dim=dim, num_heads=512 // dim), device="cuda", seed=3)
    prompt, numbers = _prompt(33, device="cuda"), _numbers(SEQUENCES, 60, device="cuda")
    free = model.sample(prompt, 60, sequences=SEQUENCES, top_k=3, random=numbers)
    # a token that about half of the sequences have drawn by the middle: they leave long before the end
    early = [int((free[:, :30] == t).any(dim=1).sum()) for t in range(512)]
    eos = min(range(512), key=lambda t: abs(early[t] - SEQUENCES // 2))
    assert SEQUENCES // 2 <= early[eos] < SEQUENCES
    kw = dict(sequences=SEQUENCES, top_k=3, random=numbers, eos=eos)
    captured = model.sample(prompt, 60, **kw)
    count = len(moves)
    assert count > 0 and torch.equal(captured, model.sample(prompt, 60, use_graph=False, **kw)) and len(moves) == 2 * count


def test_what_a_move_is_worth():
    """More than 16 sequences, or 12 GiB of keys and values that need not be read (2 layers of 256 bytes a token)."""
    model = LlamaDecoder(_cfg(), device="cpu", seed=3)
    assert model._moves_pay(17, 8, 1, 16) and not model._moves_pay(16, 8, 1, 16)
    left = (12 << 30) // (8 * 1024 * 2 * 2 * 128)
    assert model._moves_pay(16, 8, 1024, left) and not model._moves_pay(16, 8, 1024, left - 1)
    assert not model._moves_pay(16, 9, 1024, left)


@pytest.mark.gpu
def test_gpu_few_short_ones_stay(gpu, monkeypatch):
    """Eight sequences go on to their end, recorded or not: the draws are those of a run without eos."""
    monkeypatch.setattr(llama, "EOS_STRIDE", 4)
    monkeypatch.setattr(llama.QuantizedKVCache, "reorder", None)
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    prompt, kw = _prompt(33, device="cuda"), dict(sequences=SEQUENCES, top_k=3, random=_numbers(SEQUENCES, 40, device="cuda"))
    free = model.sample(prompt, 40, **kw)
    eos = int(free.flatten().mode().values)
    want = torch.where((free == eos).cumsum(dim=1) > 0, eos, free)
    for graph in (True, False):
        assert torch.equal(model.sample(prompt, 40, eos=eos, use_graph=graph, **kw), want)
