"""Refusals of the 8-bit key/value cache that need no GPU: memory that a write
would change twice."""

import ctypes
import random

import pytest

from nibble_amd import _lib

SLOTS, DIM, BLOCK = 16, 64, 16
ROW = SLOTS * DIM


def _write(k, v, batch, heads):
    """A write call's answer about the sides (codes address and strides, scales
    address and strides): its message, or '' where it goes on to the queries,
    which are misaligned (nothing is launched)."""
    sides = [_lib.KVCodes(c[0], s[0], c[1], c[2], s[1], s[2]) for c, s in (k, v)]
    cache = _lib.KVCache(*sides, batch, heads, SLOTS, DIM, BLOCK, 0)
    rows, queries = _lib.KVRows(1 << 40, 4096, 256, 64), _lib.KVRows((1 << 40) + 2, 4096, 256, 64)
    code = _lib.lib().w4a16_rotary_kv_write(ctypes.byref(queries), 1 << 42, 4, ctypes.byref(rows), ctypes.byref(rows), 3,
                                            1 << 43, 1 << 43, SLOTS, DIM, 0, ctypes.byref(cache), 1 << 41, None, 0, None)
    if code == _lib.W4A16_ERR_ALIGNMENT:
        return ""
    assert code == _lib.W4A16_ERR_CONFIG
    return _lib.last_error()


def _apart(batch, heads, address=1 << 30):
    return (address, heads, 1)


def test_overlapping_sides_are_refused():
    heads, batch = 4, 4
    far = [_apart(batch, heads), _apart(batch, heads, 1 << 31)]
    dense = lambda address, stride=heads * ROW: (address, stride, ROW)  # noqa: E731
    base = 1 << 20
    call = lambda k, v, s=far: _write((k, s[0]), (v, s[1]), batch, heads)  # noqa: E731
    assert call(dense(base), dense(base + batch * heads * ROW)) == ""
    assert "share memory" in call(dense(base), dense(base))
    assert "share memory" in call(dense(base), dense(base + ROW))                       # one row further
    assert "share memory" in call(dense(base), dense(base + batch * heads * ROW - 16))  # the last bytes
    assert "share memory" in call(dense(base + 16), dense(base))
    # heads 0 .. 3 and 3 .. 6 of one buffer of eight; heads 0 .. 3 and 4 .. 7
    assert "share memory" in call(dense(base, 8 * ROW), dense(base + 3 * ROW, 8 * ROW))
    assert call(dense(base, 8 * ROW), dense(base + 4 * ROW, 8 * ROW)) == ""
    # keys and values of a head in turn, and by slots of a longer row
    assert call((base, 2 * heads * ROW, 2 * ROW), (base + ROW, 2 * heads * ROW, 2 * ROW)) == ""
    assert "share memory" in call((base, 2 * heads * ROW, 2 * ROW), (base + ROW - 16, 2 * heads * ROW, 2 * ROW))
    # heads outside, sequences inside; backwards
    assert call((base, ROW, batch * ROW), dense(base + 64 * ROW)) == ""
    assert "share memory" in call((base, ROW, batch * ROW), dense(base + 15 * ROW))
    assert call((base + 15 * ROW, -heads * ROW, -ROW), dense(base + 16 * ROW)) == ""
    assert "share memory" in call((base + 15 * ROW, -heads * ROW, -ROW), dense(base))
    # scales: the same ones, and codes of one side in the other's scales
    assert "share memory" in call(dense(base), dense(base + 64 * ROW), [far[0], far[0]])
    assert "share memory" in call(dense(base), dense(base + 64 * ROW), [far[0], (far[0][0] + 60, heads, 1)])
    assert call(dense(base), dense(base + 64 * ROW), [far[0], (far[0][0] + 64, heads, 1)]) == ""
    assert "share memory" in call(dense(base), dense(base + 64 * ROW), [far[0], (base + 5 * ROW, heads, 1)])


def test_sides_that_overlap_themselves_are_refused():
    heads, batch = 4, 4
    far = [_apart(batch, heads), _apart(batch, heads, 1 << 31)]
    base, other = 1 << 20, (1 << 22, heads * ROW, ROW)
    for strides in ((0, ROW), (heads * ROW, 0), (heads * ROW - 16, ROW), (heads * ROW, ROW - 16), (ROW, ROW)):
        assert "overlap themselves" in _write(((base, *strides), far[0]), (other, far[1]), batch, heads)
    assert "overlap themselves" in _write(((base, heads * ROW, ROW), (1 << 30, 1, 1)), (other, far[1]), batch, heads)
    # a dimension of one has no step
    assert _write(((base, 0, ROW), (1 << 30, 0, 1)), (other, far[1]), 1, 16) == ""
    assert _write(((base, ROW, 0), (1 << 30, 1, 0)), (other, far[1]), 16, 1) == ""


@pytest.mark.parametrize("seed", range(40))
def test_overlap_against_counting(seed):
    """Random strides against the set of 16-byte pieces that each side holds."""
    rng = random.Random(seed)
    for _ in range(25):
        batch, heads = rng.choice([(2, 8), (4, 4), (8, 2), (16, 1), (1, 16), (3, 6)])
        unit = ROW // 16

        def side(address):
            inner = unit * rng.choice([1, 2, 3]) + rng.choice([0, 0, 5])
            outer_first = rng.random() < 0.7
            n = heads if outer_first else batch
            outer = inner * (n - 1) + unit + rng.choice([0, 0, unit, 7])
            strides = (outer, inner) if outer_first else (inner, outer)
            pieces = {address + b * strides[0] + h * strides[1] + i
                      for b in range(batch) for h in range(heads) for i in range(unit)}
            assert len(pieces) == batch * heads * unit
            return (16 * address, 16 * strides[0], 16 * strides[1]), pieces

        k, held = side(1 << 16)
        v, other = side((1 << 16) + rng.randrange(-3 * unit, (batch * heads + 3) * unit * 2))
        answer = _write((k, _apart(batch, heads)), (v, _apart(batch, heads, 1 << 31)), batch, heads)
        assert ("share memory" in answer) == bool(held & other), (k, v, batch, heads)
