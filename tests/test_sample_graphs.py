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


@pytest.mark.parametrize("shared", [False, True])
def test_side_stream_and_beside_the_decoders_graphs(gpu, shared, monkeypatch):
    """Calls on a stream of their own, one after the other without a wait, between greedy runs of the decoder's graphs."""
    monkeypatch.setattr(llama, "FORK_BYTES_MAX", 0 if shared else 1 << 40)
    model = LlamaDecoder(_cfg(), device="cuda", seed=3)
    prompt, numbers = _prompt(21, device="cuda"), _numbers(5, 24, device="cuda")
    model.prefill(prompt)
    model.capture()
    model.capture_prefill(21)
    greedy = model.generate(prompt, 12)
    kw = dict(sequences=5, temperature=0.9, top_p=0.9, random=numbers)
    want = model.sample(prompt, 24, **kw)
    one = model.sample(prompt, 24, random=numbers[:1])
    assert torch.equal(model.generate(prompt, 12), greedy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aside = [model.sample(prompt, 24, **kw), model.sample(prompt, 24, random=numbers[:1]),
                 model.generate(prompt, 12), model.sample(prompt, 24, **kw)]
    torch.cuda.current_stream().wait_stream(stream)
    for got, expected in zip(aside, (want, one, greedy, want)):
        assert torch.equal(got, expected)
