"""The documented example of several answers to a prompt, run as it stands on the CPU."""

import pathlib
import re

import torch

import nibble_amd
from nibble_amd import QuantizedKVCache
from tests import _kv


def _example() -> tuple[str, str]:
    """What the example does once, and what it does at each step."""
    text = (pathlib.Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    blocks = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "attend_shared(" in b]
    assert len(blocks) == 1
    once, step = re.split(r"(?=^q = )", blocks[0].replace('"cuda"', '"cpu"'), maxsplit=1, flags=re.M)
    return once, step


def test_beams_keep_every_token_of_theirs():
    """After each step a beam attends to what the beam that it goes on from has written, its newest token too."""
    once, step = _example()
    n, heads, kv, dim, length, steps = 4, 4, 2, 64, 20, 6
    rows = lambda batch, tokens, seed: _kv.rows((batch, tokens, heads + 2 * kv, dim), "fp16", seed).split([heads, kv, kv], dim=2)  # noqa: E731,E501
    cos, sin = _kv.tables(64, dim)
    prompt = QuantizedKVCache(1, kv, 32, dim, "fp8", 64)
    prompt.rotary_write(*rows(1, length, 1), cos, sin, torch.tensor([0]))
    names = dict(torch=torch, nibble_amd=nibble_amd, QuantizedKVCache=QuantizedKVCache, n=n, kv_heads=kv, head_dim=dim,
                 new_tokens=steps, length=length, cos=cos, sin=sin, prompt_cache=prompt,
                 prompt_lengths=torch.tensor([length]), held=torch.zeros((n,), dtype=torch.int64))
    exec(once, names)
    written = [[] for _ in range(n)]       # each beam's keys and values so far
    for i in range(steps):
        q, k, v = rows(n, 1, 10 + i)
        beams = torch.randint(n, (n,), generator=_kv.gen(50 + i))
        names.update(q=q, k=k, v=v, logits=_kv.rows((n, 50), "fp32", 30 + i), beams=beams)
        exec(step, names)
        written = [w + [(k[b:b + 1], v[b:b + 1])] for b, w in enumerate(written)]
        for b, w in enumerate(written):
            alone = QuantizedKVCache(1, kv, steps, dim, "fp8")
            for at, (kk, vv) in enumerate(w):
                turned = alone.rotary_write(q[b:b + 1], kk, vv, cos[length:], sin[length:], torch.tensor([at]))
            want = alone.attend_shared(turned, prompt, torch.tensor([length]), torch.tensor([i]))
            assert torch.equal(names["out"][b:b + 1], want)
        written = [written[int(b)] for b in beams]
