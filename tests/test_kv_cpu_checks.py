"""The CPU path of the 8-bit key/value cache refuses what the GPU ops refuse."""

import pytest
import torch

from nibble_amd import QuantizedKVCache, rope_tables, rotary
from tests import _kv


@pytest.fixture
def parts():
    cache = QuantizedKVCache(2, 2, 40, 64, block_size=16, device="cpu")
    q, k, v = (_kv.rows((2, 3, h, 64), "fp16", i) for i, h in ((1, 4), (2, 2), (3, 2)))
    return cache, q, k, v, torch.tensor([0, 5])


def _calls(cache, q, k, v, start, counts=None):
    cos, sin = rope_tables(64, 40)
    return (lambda: cache.write(k, v, start, counts), lambda: cache.rotary_write(q, k, v, cos, sin, start, counts),
            lambda: cache.attend(q, start, counts))


@pytest.mark.parametrize("start,counts,error", [
    ([0], None, ValueError), ([0, 1, 2], None, ValueError), ([[0, 1]], None, ValueError), (0, None, ValueError),
    ([0.0, 1.0], None, TypeError), ([0, 1], [3], ValueError), ([0, 1], [3, 3, 3], ValueError),
    ([0, 1], [True, True], TypeError),
])
def test_lengths_of_another_batch_are_refused(parts, start, counts, error):
    """A short `start` used to leave sequences out without a word."""
    cache, q, k, v, _ = parts
    before = [t.clone() for t in cache.tensors()]
    for call in _calls(cache, q, k, v, torch.tensor(start), None if counts is None else torch.tensor(counts)):
        with pytest.raises(error, match="start must|counts must"):
            call()
    with pytest.raises(TypeError, match="start must"):
        cache.write(k, v, torch.tensor([0, 1], dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors()))


def test_rows_of_another_cache_are_refused(parts):
    cache, q, k, v, start = parts
    cos, sin = rope_tables(64, 40)
    before = [t.clone() for t in cache.tensors()]
    for bad in (k[:1], k[:, :2], k[:, :, :1], k[..., :32], k[0], q):
        with pytest.raises(ValueError, match="v must have shape"):
            cache.write(k, bad, start)
        with pytest.raises(ValueError, match="[kv] must have shape"):
            cache.rotary_write(q, bad, v, cos, sin, start)
    for bad in (q[:1], q[..., :32], q[0]):
        with pytest.raises(ValueError, match="q must have shape"):
            cache.attend(bad, start)
    for bad in (q[:, :, :3], q[:, :, :0]):
        with pytest.raises(ValueError, match="positive multiple"):
            cache.attend(bad, start)
    with pytest.raises(ValueError, match="finite"):
        cache.attend(q, start, scale=float("nan"))
    with pytest.raises(ValueError, match="a row for every slot"):
        cache.rotary_write(q, k, v, cos[:39], sin[:39], start)
    for call in _calls(cache, q.clone().requires_grad_(), k.clone().requires_grad_(), v, start):
        with pytest.raises(ValueError, match="must not require grad"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors()))


def test_rotary_positions_of_another_shape_are_refused():
    """[1] and [batch, 1] used to be taken for all tokens."""
    x = _kv.rows((2, 4, 3, 64), "fp16", 4)
    cos, sin = rope_tables(64, 10)
    good = torch.tensor([0, 9, 3, 3])
    assert _kv.same(rotary(x, good, cos, sin), rotary(x, good.expand(2, 4), cos, sin))
    assert _kv.same(rotary(x[0], good, cos, sin), rotary(x, good, cos, sin)[0])
    for rows, bad in ((x, good[:1]), (x, good[:2].unsqueeze(1)), (x, good.expand(1, 4)), (x, good[0]), (x[0], good.expand(2, 4)),
                      (x[0], good.unsqueeze(0))):
        with pytest.raises(ValueError, match="positions must have shape"):
            rotary(rows, bad, cos, sin)
    with pytest.raises(ValueError, match="x must have shape"):
        rotary(x[0, 0], good[0], cos, sin)
    for tables in ((cos, sin[:9]), (cos[0], sin[0])):
        with pytest.raises(ValueError, match="cos and sin"):
            rotary(x, good, *tables)


def test_rotary_without_table_rows():
    """Every position lies outside: NaN in the rotated dims, as on the GPU."""
    x = _kv.rows((4, 2, 64), "fp16", 5)
    cos, sin = rope_tables(16, 0)
    got = rotary(x, torch.tensor([0, 1, -1, 5]), cos, sin)
    assert torch.isnan(got[..., :16]).all() and torch.equal(got[..., 16:], x[..., 16:])
    assert rotary(x[:0], torch.zeros(0, dtype=torch.int64), cos, sin).shape == (0, 2, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient_is_the_rotation_back(interleaved):
    cos, sin = rope_tables(16, 10)
    x = _kv.rows((4, 2, 24), "fp32", 6).requires_grad_()
    weights, at = _kv.rows((4, 2, 24), "fp32", 7), torch.tensor([0, 9, 3, 3])
    (rotary(x, at, cos, sin, interleaved) * weights).sum().backward()
    assert torch.allclose(x.grad, rotary(weights, at, cos, -sin, interleaved), rtol=0, atol=4 * 2.0 ** -24 * 20)
