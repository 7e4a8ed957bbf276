"""When ``LlamaDecoder.sample`` records its step in a graph."""

import pytest
import torch

from nibble_amd import llama
from nibble_amd.llama import LlamaDecoder
from tests.test_sample_decoder import _cfg, _numbers, _prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("replays", [-1, 0, 1])
def test_recorded_for_enough_replays(gpu, replays, monkeypatch):
    """One step is drawn from the prompt, one runs eagerly, the others replay."""
    steps = 2 + llama.GRAPH_REPLAYS_MIN + replays
    recorded = []
    graph = torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: (recorded.append(graph()), recorded[-1])[1])
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    prompt, numbers = _prompt(9, device="cuda"), _numbers(3, steps, device="cuda")
    got = model.sample(prompt, steps, sequences=3, top_k=5, random=numbers)
    assert len(recorded) == (replays >= 0)
    assert torch.equal(got, model.sample(prompt, steps, sequences=3, top_k=5, random=numbers, use_graph=False))
    assert len(recorded) == (replays >= 0)
