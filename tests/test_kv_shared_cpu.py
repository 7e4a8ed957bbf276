"""Attention behind shared prefixes without a GPU: the torch form against the
oracle, and refusals of the C ABI."""

import ctypes

import pytest
import torch

from nibble_amd import QuantizedKVCache, _lib
from nibble_amd.kv_reference import kv_shared_attention_reference as shared
from tests import _kv, _shared


def _ints(values):
    return torch.tensor(values, dtype=torch.int64)


CASES = [
    (1, 3, 1, [40], [0, 5, 19], None),
    (2, 2, 4, [33, 50], [0, 7, 16, 2], [4, 0, 2, 9]),
    (3, 1, 2, [0, 1, 51], [3, 18, 0], None),              # an empty prefix, one slot, one that is too long
    (1, 2, 3, [-1], [0, 4], None),                        # no such length
    (1, 4, 2, [50], [-1, 19, 20, 1 << 60], [2, 2, 2, 0]),  # positions outside
]


@pytest.mark.parametrize("groups,per,tokens,lengths,start,counts", CASES)
@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
def test_torch_form(groups, per, tokens, lengths, start, counts, codes, dtype):
    q, prefix, own = _shared.case(groups, per, tokens, 6, 2, 64, 50, 20, codes, dtype)
    got = shared(q, *prefix, _ints(lengths), *own, _ints(start), None if counts is None else _ints(counts))
    ref, bound = _shared.attend(q, prefix, lengths, own, start, counts, 64, 32)
    _kv.close(got, ref, bound)


def test_refusals_of_the_torch_form():
    q, prefix, own = _shared.case(2, 2, 1, 4, 2, 64, 30, 20)
    lengths, start = _ints([30, 30]), _ints([0] * 4)
    for bad in (dict(q=q[:, :, :3]), dict(q=q[:3]), dict(prefix=[x[:, :1] for x in prefix]), dict(lengths=lengths[:1]),
                dict(prefix=[torch.cat((x, x[:1])) for x in prefix], lengths=_ints([1, 1, 1])), dict(scale=float("inf")),
                dict(start=start[:2])):
        a = {**dict(q=q, prefix=prefix, lengths=lengths, start=start, scale=None), **bad}
        with pytest.raises(ValueError):
            shared(a["q"], *a["prefix"], a["lengths"], *own, a["start"], None, a["scale"])
    with pytest.raises(TypeError):
        shared(q, *prefix, lengths.int(), *own, start)


def test_method():
    cache, prefix = QuantizedKVCache(4, 2, 20, 64, "int8", 32), QuantizedKVCache(2, 2, 50, 64, "int8", 64)
    q, p, own = _shared.case(2, 2, 1, 4, 2, 64, 50, 20)
    cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales = own
    prefix.k_codes, prefix.k_scales, prefix.v_codes, prefix.v_scales = p
    got = cache.attend_shared(q, prefix, _ints([50, 9]), _ints([3, 4, 5, 6]))
    ref, bound = _shared.attend(q, p, [50, 9], own, [3, 4, 5, 6], None, 64, 32)
    _kv.close(got, ref, bound)


def _cache(address, batch=4, heads=2, slots=40, dim=64, block=16, kind=0):
    blocks = -(-slots // block)
    side = lambda at: _lib.KVCodes(at, at + (1 << 24), heads * slots * dim, slots * dim, heads * blocks, blocks)  # noqa: E731
    return _lib.KVCache(side(address), side(address + (1 << 25)), batch, heads, slots, dim, block, kind)


def test_refusals_of_the_c_abi():
    rows = _lib.KVRows(1 << 40, 1024, 256, 64)

    def call(prefix=None, cache=None, tokens=1, heads=4, q=rows, out=1 << 41, lengths=1 << 42, start=1 << 43, scale=0.125,
             kind=0, workspace=1 << 44, size=1 << 30):
        p, c = prefix or _cache(1 << 30, batch=2), cache or _cache(1 << 32)
        return _lib.lib().w4a16_kv_shared_attention(
            None if q is None else ctypes.byref(q), out, tokens, heads, ctypes.byref(p), lengths, ctypes.byref(c), start,
            None, scale, kind, workspace, size, None)

    for other in (dict(heads=4), dict(dim=128), dict(kind=1), dict(batch=3), dict(batch=0)):
        assert call(prefix=_cache(1 << 30, **{"batch": 2, **other})) == _lib.W4A16_ERR_SHAPE
    assert call(heads=3) == call(heads=0) == call(tokens=-1) == _lib.W4A16_ERR_SHAPE
    assert call(kind=2) == call(scale=float("inf")) == _lib.W4A16_ERR_CONFIG
    assert call(q=None) == call(out=None) == call(lengths=None) == call(start=None) == _lib.W4A16_ERR_NULL
    assert call(out=(1 << 41) + 2) == call(q=_lib.KVRows((1 << 40) + 1, 0, 0, 0)) == _lib.W4A16_ERR_ALIGNMENT
    assert call(workspace=None) == call(size=4 * 4 * 64) == _lib.W4A16_ERR_CONFIG
    assert call(workspace=(1 << 44) + 8) == _lib.W4A16_ERR_ALIGNMENT
    assert call(tokens=1 << 25) == call(cache=_cache(1 << 32, batch=1 << 24), tokens=1 << 10) == _lib.W4A16_ERR_TOO_LARGE
    many = dict(prefix=_cache(1 << 30, batch=1 << 24), cache=_cache(1 << 32, batch=1 << 24))
    assert call(tokens=1 << 20, **many) == _lib.W4A16_ERR_TOO_LARGE
    assert call(tokens=0) == call(cache=_cache(1 << 32, batch=0)) == _lib.W4A16_OK
    size = _lib.lib().w4a16_kv_shared_attention_workspace_bytes
    assert size(1, 100, 8, 1, 4, 2, 40, 64) > 0 and size(3, 100, 8, 1, 4, 2, 40, 64) == 0
    assert size(0, 100, 8, 1, 4, 2, 40, 64) == size(1, 0, 8, 1, 4, 2, 40, 64) == size(1, 100, 0, 1, 4, 2, 40, 64) == 0
