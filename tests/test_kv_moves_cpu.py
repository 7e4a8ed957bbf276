"""Forking and reordering caches without a GPU: the torch form, and refusals of
the C ABI, which come before anything is launched."""

import ctypes

import pytest
import torch

from nibble_amd import QuantizedKVCache, _lib
from tests import _kv, _moves


@pytest.mark.parametrize("held,slots,batch,to_slots,block,source,lengths", _moves.FORKS)
def test_fork(held, slots, batch, to_slots, block, source, lengths):
    a = QuantizedKVCache(held, 2, slots, 64, "int8", block)
    b = QuantizedKVCache(batch, 2, to_slots, 64, "int8", block)
    a.k_codes, a.k_scales, a.v_codes, a.v_scales = _moves.tensors(held, 2, slots, 64, "int8", block, 1)
    b.k_codes, b.k_scales, b.v_codes, b.v_scales = _moves.tensors(batch, 2, to_slots, 64, "int8", block, 5)
    want = _moves.expected(a.tensors(), b.tensors(), source, lengths, block)
    b.fork_from(a, torch.tensor(source), torch.tensor(lengths))
    _moves.check(b.tensors(), want)


@pytest.mark.parametrize("batch,slots,block,source,lengths", _moves.REORDERS)
def test_reorder(batch, slots, block, source, lengths):
    a = QuantizedKVCache(batch, 3, slots, 64, "fp8", block)
    a.k_codes, a.k_scales, a.v_codes, a.v_scales = _moves.tensors(batch, 3, slots, 64, "fp8", block, 9)
    want = _moves.expected(a.tensors(), a.tensors(), source, lengths, block)
    a.reorder(torch.tensor(source), torch.tensor(lengths))
    _moves.check(a.tensors(), want)


def test_refusals_of_the_torch_form():
    cache = lambda batch=2, heads=2, slots=40, dim=64, dtype="int8", block=16: QuantizedKVCache(batch, heads, slots, dim, dtype, block)  # noqa: E731,E501
    a, source, lengths = cache(), torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    for other in (cache(heads=3), cache(dim=128), cache(dtype="fp8"), cache(block=32)):
        with pytest.raises(ValueError, match="same KV heads"):
            a.fork_from(other, source, lengths)
    with pytest.raises(ValueError, match="shape"):
        a.fork_from(cache(batch=3), source, lengths)
    with pytest.raises(TypeError):
        a.reorder(source.int(), lengths)
    with pytest.raises(ValueError, match="shape"):
        a.reorder(source, lengths[:1])
    # one scale for all slots: of the other cache's block
    a.fork_from(cache(slots=10, block=128), source, lengths)
    cache(slots=300, block=128).fork_from(cache(slots=10, block=32), source, lengths)


def _cache(address, batch=2, heads=2, slots=40, dim=64, block=16, kind=0):
    blocks = -(-slots // block)
    side = lambda at: _lib.KVCodes(at, at + (1 << 24), heads * slots * dim, slots * dim, heads * blocks, blocks)  # noqa: E731
    return _lib.KVCache(side(address), side(address + (1 << 25)), batch, heads, slots, dim, block, kind)


def test_refusals_of_the_c_abi():
    def fork(a, b, source=1 << 20, lengths=1 << 21):
        return _lib.lib().w4a16_kv_fork(ctypes.byref(a), ctypes.byref(b), source, lengths, None)

    def reorder(a, source=1 << 20, lengths=1 << 21):
        return _lib.lib().w4a16_kv_reorder(ctypes.byref(a), source, lengths, None)

    here, there = 1 << 30, 1 << 32
    for other in (dict(heads=3), dict(dim=128), dict(block=32), dict(kind=1)):
        assert fork(_cache(here), _cache(there, **other)) == _lib.W4A16_ERR_SHAPE
    assert fork(_cache(here), _cache(there), source=None) == fork(_cache(here), _cache(there), lengths=None) == _lib.W4A16_ERR_NULL
    assert reorder(_cache(here), source=None) == _lib.W4A16_ERR_NULL
    assert fork(_cache(here), _cache(here)) == _lib.W4A16_ERR_CONFIG and "share" in _lib.last_error()
    # the second sequence of one as the first of the other; the other's keys in this one's scales
    assert fork(_cache(here), _cache(here + 2 * 40 * 64)) == _lib.W4A16_ERR_CONFIG
    assert fork(_cache(here), _cache(here + (1 << 24) - (1 << 25))) == _lib.W4A16_ERR_CONFIG
    same = _cache(here)
    same.k.batch_stride = 0
    assert reorder(same) == fork(_cache(there), same) == _lib.W4A16_ERR_CONFIG
    assert reorder(_cache(here, batch=4097)) == _lib.W4A16_ERR_TOO_LARGE
    assert reorder(_cache(here, batch=1025, dim=256)) == _lib.W4A16_ERR_TOO_LARGE
    assert reorder(_cache(here, dim=96)) == fork(_cache(here, slots=0), _cache(there)) == _lib.W4A16_ERR_SHAPE
    assert reorder(_cache(here, batch=0)) == fork(_cache(here, batch=0), _cache(there)) == _lib.W4A16_OK
    assert _kv.same(torch.zeros(1), torch.zeros(1))
