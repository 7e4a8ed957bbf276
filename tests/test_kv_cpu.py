"""The 8-bit key/value cache on the CPU: the torch path against the 64-bit
oracle, the rotary tables, and the refusals of the C ABI (no GPU is touched)."""

import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

import nibble_amd
from nibble_amd import QuantizedKVCache, _lib, rope_frequencies, rope_tables, rotary
from nibble_amd import kv_reference as plain
from tests import _kv

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "w4a16_kv.h")


def test_header_symbols_bound():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(w4a16_\w+)\s*\(", text))
    assert names == set(_lib.KV_SIGNATURES)
    handle = _lib.lib()
    for name in names:
        assert getattr(handle, name)


# --------------------------------------------------------------- the oracle is pinned

def test_oracle_rounds_like_the_types():
    x = torch.linspace(-500, 500, 20011, dtype=torch.float64)
    assert np.array_equal(_kv.nearest(x.float().double().numpy(), torch.float8_e4m3fn),   # one number on both sides
                          x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy())
    small = torch.linspace(-0.03, 0.03, 4001, dtype=torch.float64)   # subnormals
    assert np.array_equal(_kv.nearest(small.float().double().numpy(), torch.float8_e4m3fn),
                          small.float().to(torch.float8_e4m3fn).double().numpy())
    assert _kv.nearest(np.array([0.5, 1.5, 2.5, -0.5, 300.0]), torch.int8).tolist() == [0, 2, 2, 0, 127]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_scale_is_the_smallest_that_fits(dtype):
    top = _kv.LARGEST[dtype]
    for e in (-39, -3, 0, 7, 39):
        amax = torch.tensor([top * 2.0 ** e, math.nextafter(top * 2.0 ** e, 1e30) * (1 + 2.0 ** -23)])
        got = plain.scale_of(amax, top)
        assert got.tolist() == [2.0 ** e, 2.0 ** min(e + 1, 40)]
        assert [_kv.scale(float(a), dtype) for a in amax] == got.tolist()
    assert plain.scale_of(torch.tensor([0.0, 1e-30, 1e30, float("inf")]), top).tolist() == [2.0 ** -40, 2.0 ** -40,
                                                                                              2.0 ** 40, 2.0 ** 40]


# ----------------------------------------------------------------------- the torch path

@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("block,start,counts", [(16, [0, 5], None), (64, [70, 3], [4, 0]), (32, [-2, 98], [9, 9]),
                                                (128, [0, 99], [11, 20])])
def test_write_matches_oracle(codes, dtype, block, start, counts):
    x = _kv.rows((2, 9, 3, 64), dtype, 1, spread=3.0)
    x[0, 2, 1, 5], x[1, 0, 0, 0], x[1, 1, 2, 3] = float("nan"), float("inf"), 0.0
    c, s = _kv.cache(2, 3, 100, 64, codes, block, 2)
    v, vs = _kv.cache(2, 3, 100, 64, codes, block, 3)
    first = torch.tensor(start)
    limits = None if counts is None else torch.tensor(counts)
    want = _kv.write(x, c, s, start, counts, block)
    nibble_amd.kv_reference.kv_write_reference(x, x, c, s, v, vs, first, limits)
    assert np.array_equal(_kv.numbers(c), want[0]) and np.array_equal(_kv.numbers(s), want[1])


def test_cache_object_runs_on_the_cpu():
    cache = QuantizedKVCache(2, 2, 40, 64, dtype="int8", block_size=16, device="cpu")
    cos, sin = rope_tables(64, 40)
    q, k, v = (_kv.rows((2, 7, h, 64), "fp16", i) for i, h in ((1, 4), (2, 2), (3, 2)))
    start, counts = torch.tensor([0, 20]), torch.tensor([7, 5])
    turned = cache.rotary_write(q, k, v, cos, sin, start, counts)
    out = cache.attend(turned, start, counts)
    positions = start.unsqueeze(1) + torch.arange(7)
    ref, size = _kv.rotate(q, cos, sin, positions, False)
    ref[1, 5:] = 0
    _kv.close(turned, ref, 3 * 2.0 ** -24 * size)
    want, bound = _kv.attend(turned, *cache.tensors(), start, counts, 16)
    _kv.close(out, want, bound)
    assert torch.equal(out[1, 5:], torch.zeros_like(out[1, 5:]))
    keys, values = cache.read(25)
    assert keys.shape == (2, 2, 25, 64)
    assert np.array_equal(_kv.numbers(values), _kv.values(cache.v_codes, cache.v_scales, 16)[:, :, :25])
    assert cache.nbytes() == 2 * (2 * 2 * 40 * 64 + 4 * 2 * 2 * 3)
    assert cache.read(0)[0].shape == (2, 2, 0, 64)


def test_one_token_at_a_time_stays_near_one_write():
    """Scales grow as tokens come; every code is then off by its own half step
    and at most half a step of each growth, in all less than one and a half of the last."""
    x = _kv.rows((1, 64, 2, 64), "fp16", 4) * torch.linspace(0.01, 4, 64).view(1, 64, 1, 1).half()
    cache = QuantizedKVCache(1, 2, 64, 64, device="cpu")
    for t in range(64):
        cache.write(x[:, t:t + 1], x[:, t:t + 1], torch.tensor([t]))
    got = _kv.values(cache.k_codes, cache.k_scales, 64)[0]
    step = _kv.numbers(cache.k_scales)[0].max(axis=1)[:, None, None]
    assert (np.abs(got - _kv.numbers(x)[0].transpose(1, 0, 2)) <= 1.5 * step).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot,dim", [(64, 64), (16, 64), (2, 6), (10, 33)])
def test_rotary_matches_oracle(interleaved, rot, dim):
    x = _kv.rows((2, 5, 3, dim), "bf16", 1)
    cos, sin = _kv.tables(50, rot)
    positions = torch.tensor([[0, 1, 49, 50, 7], [-1, 3, 3, 2, 48]])
    got = rotary(x, positions, cos, sin, interleaved)
    ref, size = _kv.rotate(x, cos, sin, positions, interleaved)
    _kv.close(got, ref, 3 * 2.0 ** -24 * size)


def test_cache_object_refuses():
    with pytest.raises(ValueError, match="int8"):
        QuantizedKVCache(1, 1, 8, 64, dtype="int4", device="cpu")
    with pytest.raises(ValueError, match="block_size"):
        QuantizedKVCache(1, 1, 8, 64, block_size=48, device="cpu")
    with pytest.raises(ValueError, match="greater than zero"):
        QuantizedKVCache(0, 1, 8, 64, device="cpu")
    cache = QuantizedKVCache(1, 1, 8, 64, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        cache.read(9)


# ------------------------------------------------------------------------- the tables

SCALINGS = [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
    {"type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048},
]


def test_rope_frequencies_ends():
    """The ends of each scaling, from its definition."""
    inv, one = rope_frequencies(128, 500000.0)
    assert one == 1.0 and inv[0] == 1.0
    assert torch.equal(rope_frequencies(128, 500000.0, SCALINGS[0])[0], inv / 4)
    llama, _ = rope_frequencies(128, 500000.0, SCALINGS[1])
    fast, slow = 8192 * inv / (2 * math.pi) > 4.0, 8192 * inv / (2 * math.pi) < 1.0
    assert torch.equal(llama[fast], inv[fast]) and torch.allclose(llama[slow], inv[slow] / 8, rtol=1e-15)
    assert (llama[1:] < llama[:-1]).all()
    yarn, factor = rope_frequencies(128, 500000.0, SCALINGS[2])
    assert yarn[0] == inv[0] and math.isclose(float(yarn[-1]), float(inv[-1]) / 4) and factor > 1.13
    assert torch.equal(rope_frequencies(128, 1e4, SCALINGS[3], 2048)[0], rope_frequencies(128, 1e4)[0])
    assert rope_frequencies(128, 1e4, SCALINGS[3], 8192)[0][-1] < rope_frequencies(128, 1e4)[0][-1]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s.get("rope_type", s.get("type")))
def test_rope_frequencies_match_transformers(scaling):
    utils = pytest.importorskip("transformers.modeling_rope_utils")
    transformers = pytest.importorskip("transformers")
    kind = scaling.get("rope_type", scaling.get("type"))
    original = 2048 if kind == "dynamic" else 32768
    cfg = transformers.LlamaConfig(hidden_size=2048, num_attention_heads=16, rope_theta=500000.0,
                                   max_position_embeddings=original,
                                   rope_scaling={**{k: v for k, v in scaling.items() if k != "type"}, "rope_type": kind})
    want, factor = utils.ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=8192)
    got, own = rope_frequencies(128, 500000.0, scaling, 8192)
    # theirs are formed in fp32: a power, a division and a blend of a few roundings
    assert torch.allclose(got, want.double(), rtol=8 * 2.0 ** -24, atol=0) and math.isclose(own, factor, rel_tol=1e-6)


def test_rope_tables():
    cos, sin = rope_tables(64, 200000, 1e4)
    assert cos.shape == (200000, 32) and cos.dtype == torch.float32
    assert math.isclose(float(cos[199999, 0]), math.cos(199999.0), abs_tol=2.0 ** -24)
    assert math.isclose(float(sin[199999, 31]), math.sin(199999.0 * 1e4 ** (-62 / 64)), abs_tol=2.0 ** -24)
    scaled = rope_tables(64, 10, 1e4, {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 8})
    assert math.isclose(float(scaled[0][0, 0]), 0.1 * math.log(2.0) + 1.0, rel_tol=1e-6)


@pytest.mark.parametrize("scaling,message", [
    ({"rope_type": "longrope", "factor": 2.0}, "unknown rope scaling"),
    ({"rope_type": "linear"}, "positive factor"),
    ({"rope_type": "linear", "factor": 0.0}, "positive factor"),
    ({"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
      "original_max_position_embeddings": 8}, "high_freq_factor"),
    ({"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 8, "mscale": 1.0}, "mscale"),
])
def test_rope_frequencies_refuse(scaling, message):
    with pytest.raises(ValueError, match=message):
        rope_frequencies(64, 1e4, scaling)


def test_rope_frequencies_refuse_sizes():
    for dims, theta in ((0, 1e4), (3, 1e4), (4, 0.0)):
        with pytest.raises(ValueError):
            rope_frequencies(dims, theta)


# ------------------------------------------------------------ refusals of the C ABI (host only)

def _side(address=1 << 20, batch_stride=2048, head_stride=1024):
    return _lib.KVCodes(address, address + (1 << 16), batch_stride, head_stride, 2, 1)


def _cache(**changes):
    args = dict(k=_side(), v=_side(1 << 21), batch=1, kv_heads=2, slots=16, head_dim=64, block=16, code_type=0)
    args.update(changes)
    return _lib.KVCache(**args)


def _rows(address=1 << 22):
    return _lib.KVRows(address, 4096, 256, 64)


def _write(cache, tokens=3, type_=0, k=None, start=1 << 24):
    rows = _rows() if k is None else k
    return _lib.lib().w4a16_kv_write(ctypes.byref(rows), ctypes.byref(rows), tokens, ctypes.byref(cache), start, None,
                                     type_, None)


def _attend(cache, tokens=1, heads=4, type_=0, out=1 << 23, q=None, workspace=None, nbytes=0, scale=0.125):
    rows = _rows() if q is None else q
    return _lib.lib().w4a16_kv_attention(ctypes.byref(rows), out, tokens, heads, ctypes.byref(cache), 1 << 24, None,
                                         scale, type_, workspace, nbytes, None)


@pytest.mark.parametrize("changes,code", [
    (dict(block=48), _lib.W4A16_ERR_GROUP_SIZE), (dict(block=0), _lib.W4A16_ERR_GROUP_SIZE),
    (dict(code_type=2), _lib.W4A16_ERR_CONFIG),
    (dict(head_dim=96), _lib.W4A16_ERR_SHAPE), (dict(kv_heads=0), _lib.W4A16_ERR_SHAPE),
    (dict(slots=0), _lib.W4A16_ERR_SHAPE), (dict(batch=-1), _lib.W4A16_ERR_SHAPE),
    (dict(slots=(1 << 30) + 1), _lib.W4A16_ERR_TOO_LARGE),
    (dict(k=_side(0)), _lib.W4A16_ERR_NULL), (dict(v=_side((1 << 20) + 8)), _lib.W4A16_ERR_ALIGNMENT),
    (dict(k=_side(head_stride=1032)), _lib.W4A16_ERR_ALIGNMENT),
])
def test_cache_refusals(changes, code):
    assert _write(_cache(**changes)) == code
    assert _attend(_cache(**changes)) == code
    assert _lib.last_error()


def test_write_refusals():
    assert _write(_cache(), tokens=-1) == _lib.W4A16_ERR_SHAPE
    assert _write(_cache(), type_=2) == _lib.W4A16_ERR_CONFIG
    assert _write(_cache(), k=_lib.KVRows(None, 0, 0, 0)) == _lib.W4A16_ERR_NULL
    assert _write(_cache(), k=_rows((1 << 22) + 1)) == _lib.W4A16_ERR_ALIGNMENT
    assert _write(_cache(), start=None) == _lib.W4A16_ERR_NULL
    assert _write(_cache(), tokens=0) == _lib.W4A16_OK
    assert _write(_cache(batch=0)) == _lib.W4A16_OK


def test_rotary_refusals():
    fn = _lib.lib().w4a16_rotary
    rows = _rows()

    def call(dim=64, rot=64, table=1 << 22, out=1 << 23, type_=0, batch=1, x=rows):
        return fn(ctypes.byref(x), out, batch, 2, 3, dim, table, table, 10, rot, 1 << 24, 0, 1, 0, type_, None)

    assert call(rot=63) == _lib.W4A16_ERR_SHAPE
    assert call(rot=0) == _lib.W4A16_ERR_SHAPE
    assert call(rot=66) == _lib.W4A16_ERR_SHAPE
    assert call(type_=2) == _lib.W4A16_ERR_CONFIG
    assert call(table=None) == _lib.W4A16_ERR_NULL
    assert call(out=None) == _lib.W4A16_ERR_NULL
    assert call(out=(1 << 23) + 1) == _lib.W4A16_ERR_ALIGNMENT
    assert call(batch=-1) == _lib.W4A16_ERR_SHAPE
    assert call(batch=0) == _lib.W4A16_OK


def test_calls_past_a_launch_are_refused():
    """2^32 threads or more, and products of sizes past 64 bits."""
    rows = _rows()
    many = dict(batch=1 << 22, kv_heads=16)
    assert _write(_cache(**many), tokens=1) == _lib.W4A16_ERR_TOO_LARGE
    assert _attend(_cache(**many), heads=16) == _lib.W4A16_ERR_TOO_LARGE
    lib = _lib.lib()
    assert lib.w4a16_rotary_kv_write(ctypes.byref(rows), 1 << 23, 1 << 16, ctypes.byref(rows), ctypes.byref(rows),
                                     1 << 24, 1 << 22, 1 << 22, 16, 64, 0, ctypes.byref(_cache(batch=1 << 24)),
                                     1 << 24, None, 0, None) == _lib.W4A16_ERR_TOO_LARGE
    for offset in (0, 2):   # whole vectors, and any alignment
        x = _rows((1 << 22) + offset)
        assert lib.w4a16_rotary(ctypes.byref(x), 1 << 23, 1, 1 << 28, 16, 64, 1 << 22, 1 << 22, 10, 64, 1 << 24, 0, 1,
                                0, 0, None) == _lib.W4A16_ERR_TOO_LARGE
    side = _side()
    assert lib.w4a16_kv_read(ctypes.byref(side), 1 << 23, 1 << 24, 1, 16, 64, 16, 0, 0,
                             None) == _lib.W4A16_ERR_TOO_LARGE


def test_rotary_write_refusals():
    fn = _lib.lib().w4a16_rotary_kv_write
    rows = _rows()

    def call(rot=64, table_rows=16, q=rows, out=1 << 23, heads=4):
        return fn(ctypes.byref(q), out, heads, ctypes.byref(rows), ctypes.byref(rows), 2, 1 << 22, 1 << 22, table_rows,
                  rot, 0, ctypes.byref(_cache()), 1 << 24, None, 0, None)

    assert call(rot=8) == _lib.W4A16_ERR_SHAPE
    assert call(rot=80) == _lib.W4A16_ERR_SHAPE
    assert call(table_rows=15) == _lib.W4A16_ERR_SHAPE
    assert call(q=_rows((1 << 22) + 2)) == _lib.W4A16_ERR_ALIGNMENT
    assert call(out=None) == _lib.W4A16_ERR_NULL
    assert call(heads=-1) == _lib.W4A16_ERR_SHAPE


def test_read_refusals():
    fn = _lib.lib().w4a16_kv_read
    side = _side()

    def call(dim=64, block=16, out=1 << 23, out_type=0, code_type=0, slots=16, c=side):
        return fn(ctypes.byref(c), out, 1, 2, slots, dim, block, code_type, out_type, None)

    assert call(dim=24) == _lib.W4A16_ERR_SHAPE
    assert call(block=8) == _lib.W4A16_ERR_GROUP_SIZE
    assert call(out=None) == _lib.W4A16_ERR_NULL
    assert call(out=(1 << 23) + 4) == _lib.W4A16_ERR_ALIGNMENT
    assert call(out_type=3) == _lib.W4A16_ERR_CONFIG
    assert call(code_type=-1) == _lib.W4A16_ERR_CONFIG
    assert call(slots=-1) == _lib.W4A16_ERR_SHAPE
    assert call(slots=0) == _lib.W4A16_OK


def test_attention_refusals():
    assert _attend(_cache(), heads=3) == _lib.W4A16_ERR_SHAPE
    assert _attend(_cache(), heads=0) == _lib.W4A16_ERR_SHAPE
    assert _attend(_cache(), type_=2) == _lib.W4A16_ERR_CONFIG
    assert _attend(_cache(), out=None) == _lib.W4A16_ERR_NULL
    assert _attend(_cache(), out=(1 << 23) + 8) == _lib.W4A16_ERR_ALIGNMENT
    assert _attend(_cache(), tokens=-1) == _lib.W4A16_ERR_SHAPE
    for scale in (float("nan"), float("inf"), float("-inf")):
        assert _attend(_cache(), scale=scale) == _lib.W4A16_ERR_CONFIG
    assert _attend(_cache(), tokens=0) == _lib.W4A16_OK
    wide = _cache(slots=4096, k=_side(batch_stride=1 << 20, head_stride=1 << 19),
                  v=_side(1 << 21, batch_stride=1 << 20, head_stride=1 << 19))
    need = _lib.lib().w4a16_kv_attention_workspace_bytes(1, 1, 4, 2, 4096, 64)
    assert need > 0
    assert _attend(wide) == _lib.W4A16_ERR_CONFIG
    assert _attend(wide, workspace=1 << 25, nbytes=need - 1) == _lib.W4A16_ERR_CONFIG
    assert _attend(wide, workspace=(1 << 25) + 4, nbytes=need) == _lib.W4A16_ERR_ALIGNMENT
    assert _lib.lib().w4a16_kv_attention_workspace_bytes(0, 1, 4, 2, 4096, 64) == 0
    assert _lib.lib().w4a16_kv_attention_workspace_bytes(1, 1, 3, 2, 4096, 64) == 0


def test_fake_tensors():
    """Shapes for traced calls."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty((2, 3, 4, 64), dtype=torch.bfloat16, device="cuda")
        codes = torch.empty((2, 2, 40, 64), dtype=torch.int8, device="cuda")
        scales = torch.empty((2, 2, 3), device="cuda")
        start = torch.empty((2,), dtype=torch.int64, device="cuda")
        cos = torch.empty((40, 32), device="cuda")
        out = nibble_amd.rotary_kv_write_cuda(q, q[:, :, :2], q[:, :, :2], cos, cos, codes, scales, codes, scales, start)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert nibble_amd.kv_attention_cuda(q, codes, scales, codes, scales, start).shape == q.shape
        assert nibble_amd.kv_read_cuda(codes, scales, torch.float32).dtype == torch.float32
        assert nibble_amd.rotary_cuda(q[0], start, cos, cos).shape == (3, 4, 64)
        assert nibble_amd.kv_write_cuda(q[:, :, :2], q[:, :, :2], codes, scales, codes, scales, start) is None


def test_both_import_names():
    import w4a16
    from w4a16.kv_cache import QuantizedKVCache as same
    from w4a16.rope import rope_tables as tables

    assert same is QuantizedKVCache is w4a16.QuantizedKVCache and tables is rope_tables
    assert w4a16.kv_attention_cuda is nibble_amd.kv_attention_cuda and w4a16.rotary is rotary
