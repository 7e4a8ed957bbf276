"""Keys and values of an 8-bit cache in one buffer: layouts that interleave them
work, layouts that overlap are refused before a launch."""

import pytest
import torch

from nibble_amd import kv_attention_cuda, kv_read_cuda, kv_write_cuda, rotary_kv_write_cuda
from tests import _kv

pytestmark = pytest.mark.gpu


def _views(codes, scales, kind):
    """(k_codes, k_scales, v_codes, v_scales) [2, 3, slots, 64] in one buffer each."""
    if kind == "heads":          # keys behind values, head by head
        return codes[:, 0:6:2], scales[:, 0:6:2], codes[:, 1:6:2], scales[:, 1:6:2]
    if kind == "halves":
        return codes[:, :3], scales[:, :3], codes[:, 3:6], scales[:, 3:6]
    return codes[:, :3], scales[:, :3], codes[:, 2:5], scales[:, 2:5]   # share a head


@pytest.mark.parametrize("kind", ["heads", "halves"])
def test_write_into_one_buffer(gpu, kind):
    k, v = (_kv.rows((2, 40, 3, 64), "fp16", i).cuda() for i in (71, 72))
    start = torch.tensor([0, 5]).cuda()
    codes, scales = (t.cuda() for t in _kv.cache(2, 6, 50, 64, "int8", 16, 73))
    view = _views(codes, scales, kind)
    apart = [t.contiguous() for t in view]
    kv_write_cuda(k, v, *view, start)
    kv_write_cuda(k, v, *apart, start)
    for a, b in zip(view, apart):
        assert _kv.same(a, b)


def test_overlapping_views_are_refused(gpu):
    k = _kv.rows((2, 4, 3, 64), "fp16", 74).cuda()
    start = torch.zeros(2, dtype=torch.int64, device="cuda")
    cos, sin = (t.cuda() for t in _kv.tables(50, 64))
    codes, scales = (t.cuda() for t in _kv.cache(2, 6, 50, 64, "int8", 16, 73))
    before = codes.clone()
    view = _views(codes, scales, "overlap")
    other = codes.clone()[:, :3]
    for cache in (view, (view[0], view[1], other, view[3]), (view[0], view[1], view[2], scales.clone()[:, :3])):
        with pytest.raises(RuntimeError, match="must not share memory"):
            kv_write_cuda(k, k, *cache, start)
        with pytest.raises(RuntimeError, match="must not share memory"):
            rotary_kv_write_cuda(k, k, k, cos, sin, *cache, start)
    torch.cuda.synchronize()
    assert _kv.same(codes, before)


def test_codes_that_require_grad_are_refused(gpu):
    """e4m3 codes can: the attention would return outputs without a gradient."""
    k = _kv.rows((2, 4, 3, 64), "fp16", 75).cuda()
    start = torch.zeros(2, dtype=torch.int64, device="cuda")
    codes, scales = (t.cuda() for t in _kv.cache(2, 3, 50, 64, "fp8", 16, 76))
    other, own = codes.clone(), scales.clone()
    leaf = codes.clone().requires_grad_()
    for call in (lambda: kv_attention_cuda(k, codes, scales, leaf, own, start), lambda: kv_read_cuda(leaf, scales),
                 lambda: kv_write_cuda(k, k, leaf, scales, other, own, start)):
        with pytest.raises(RuntimeError, match="must not require grad"):
            call()
