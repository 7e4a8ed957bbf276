"""LlamaDecoder over an 8-bit cache on the GPU: models that the fused step is not made for."""

import pytest
import torch

from nibble_amd.llama import LlamaDecoder
from tests.test_kv_decoder import _cfg, _prompt

pytestmark = pytest.mark.gpu


def _logits(model, prompt):
    """Of a prompt and of a token behind it."""
    model.prefill(prompt)
    first = model.token.clone()
    model.step()
    return first, model.logits.clone()


@pytest.mark.parametrize("kv_cache,changes", [("fp16", {}), ("int8", {}), ("fp8", dict(num_heads=4, head_dim=128)),
                                              ("int8", dict(num_heads=2, num_kv_heads=1, head_dim=256))])
@pytest.mark.parametrize("group_size", [32, 64, 256])
def test_other_group_sizes_run_the_torch_step(gpu, group_size, kv_cache, changes):
    """The fused step's GEMVs index scales of groups of 128: wrong ones, or past
    the tensor's end, with another size."""
    cfg = _cfg(kv_cache=kv_cache, group_size=group_size, **changes)
    model, plain = LlamaDecoder(cfg, device=gpu, seed=4), LlamaDecoder(cfg, device=gpu, seed=4, fused=False)
    assert not model.fused and not model.attn_o and not model.fused_prefill(9)
    for a, b in zip(_logits(model, _prompt(9).to(gpu)), _logits(plain, _prompt(9).to(gpu))):
        assert torch.isfinite(a.float()).all() and torch.equal(a, b)
    cpu = LlamaDecoder(cfg, device="cpu", init="empty")
    cpu.load_state_dict({k: v.cpu() for k, v in model.state_dict().items()})
    model.prefill(_prompt(9).to(gpu))
    cpu.prefill(_prompt(9))
    for m in (model, cpu):
        m.token.fill_(3)
        m.step()
    got, want = model.logits.float().cpu(), cpu.logits.float()
    # sums in another order, an fp16 step at most, move a code by one here and there; wrong scales give other logits
    assert (got - want).norm() <= 0.02 * want.norm()
    assert LlamaDecoder(_cfg(kv_cache=kv_cache, **changes), device=gpu, seed=4).fused is (
        kv_cache != "fp16" or changes == {})
