"""The 8-bit key/value cache on the GPU: rotary positions, writing, reading
back and attention against the 64-bit oracle of tests/_kv.py."""

import numpy as np
import pytest
import torch

import nibble_amd
from nibble_amd import QuantizedKVCache, kv_attention_cuda, kv_read_cuda, kv_write_cuda, rotary_cuda, rotary_kv_write_cuda
from nibble_amd import kv_reference as plain
from tests import _kv

pytestmark = pytest.mark.gpu


def _dev(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


# ---------------------------------------------------------------------------- refusals

def test_refusals(gpu):
    """Every refusal raises before anything is launched."""
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device="cuda")
    k = q[:, :, :2]
    codes = lambda *s, dtype=torch.int8: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    kc, vc = codes(2, 2, 40, 64), codes(2, 2, 40, 64)
    sc, vs = torch.ones((2, 2, 3), device="cuda"), torch.ones((2, 2, 3), device="cuda")
    start = torch.zeros((2,), dtype=torch.int64, device="cuda")
    cos = torch.ones((40, 32), device="cuda")

    def refuse(message, call, *args, **kwargs):
        with pytest.raises(RuntimeError, match=message):
            call(*args, **kwargs)

    attend = lambda **c: kv_attention_cuda(*{**dict(q=q, k=kc, ks=sc, v=vc, vs=vs, start=start, counts=None), **c}.values())  # noqa: E731,E501
    refuse("dtype torch.float16 or torch.bfloat16", attend, q=q.float())
    refuse("shape \\[batch, tokens, heads, head_dim\\]", attend, q=q[0])
    refuse("contiguous in its last dimension", attend, q=torch.zeros((2, 3, 4, 128), dtype=torch.float16, device="cuda")[..., ::2])
    refuse("of the cache", attend, q=q[:1])
    refuse("of the cache", attend, q=q[..., :32])
    refuse("positive multiple", attend, q=q[:, :, :3])
    refuse("torch.int8 or torch.float8_e4m3fn", attend, k=kc.view(torch.uint8), v=vc.view(torch.uint8))
    refuse("same dtype", attend, v=vc.view(torch.float8_e4m3fn))
    refuse("same shapes", attend, v=vc[:, :, :39])
    refuse("one scale for every", attend, k=kc[:, :, :32], v=vc[:, :, :32], ks=torch.ones((2, 2, 3), device="cuda"),
           vs=torch.ones((2, 2, 3), device="cuda"))
    refuse("contiguous in slots", attend, k=codes(2, 40, 2, 64).transpose(1, 2), v=vc)
    refuse("scales must have dtype", attend, ks=sc.half())
    refuse("start must have dtype", attend, start=start.int())
    refuse("shape \\[batch\\]", attend, start=start[:1])
    refuse("counts must have dtype", attend, counts=start.int())
    refuse("CUDA", attend, q=q.cpu())
    refuse("must not require grad", attend, q=q.clone().requires_grad_())
    refuse("64, 128 or 256", attend, q=q[..., :32], k=codes(2, 2, 40, 32), v=codes(2, 2, 40, 32))
    refuse("must not share memory", kv_write_cuda, k, k, kc, sc, kc, vs, start)
    refuse("overlap", kv_write_cuda, k, k, kc[:1].expand(2, -1, -1, -1), sc, vc, vs, start)
    refuse("same dtype", kv_write_cuda, k, k.bfloat16(), kc, sc, vc, vs, start)
    refuse("of the cache", kv_write_cuda, q, q, kc, sc, vc, vs, start)
    rotate_write = lambda c, s, qq=q: rotary_kv_write_cuda(qq, k, k, c, s, kc, sc, vc, vs, start)  # noqa: E731
    refuse("a row for every slot", rotate_write, cos[:39], cos[:39])
    refuse("multiple of 16", rotate_write, cos[:, :12].contiguous(), cos[:, :12].contiguous())
    refuse("torch.float32", rotate_write, cos.half(), cos.half())
    refuse("16-byte aligned", rotate_write, cos, cos, torch.zeros((2, 3, 4, 65), dtype=torch.float16, device="cuda")[..., 1:])
    refuse("even number of at most head_dim", rotary_cuda, q[..., :32], start[:1].expand(2, 3), cos, cos)
    refuse("positions must have shape", rotary_cuda, q, start, cos, cos)
    refuse("positions must have dtype", rotary_cuda, q[0], torch.zeros(3, device="cuda"), cos, cos)
    refuse("dtype must be", kv_read_cuda, kc, sc, torch.float64)
    refuse("must not require grad", kv_read_cuda, kc, sc.clone().requires_grad_())
    refuse("must not require grad", attend, vs=vs.clone().requires_grad_())
    refuse("must not require grad", rotate_write, cos, cos.clone().requires_grad_())


# ------------------------------------------------------------------------------ rotary

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("batch,tokens,heads,dim,rot", [(1, 1, 32, 64, 64), (2, 5, 3, 64, 16), (1, 7, 4, 128, 64),
                                                        (2, 3, 5, 80, 80), (1, 9, 2, 33, 10), (3, 2, 1, 6, 2),
                                                        (1, 2, 2, 256, 256)])
def test_rotary(gpu, batch, tokens, heads, dim, rot, dtype, interleaved):
    x = _kv.rows((batch, tokens, heads + 1, dim), dtype, 1)[:, :, 1:]   # a view whose rows lie apart
    cos, sin = _kv.tables(300, rot)
    positions = torch.randint(0, 300, (batch, tokens), generator=_kv.gen(2))
    positions[0, 0], positions[-1, -1] = 299, 0
    got = rotary_cuda(*_dev(x, positions, cos, sin), interleaved)
    assert got.is_contiguous() and got.shape == x.shape
    ref, size = _kv.rotate(x, cos, sin, positions, interleaved)
    _kv.close(got, ref, 3 * 2.0 ** -24 * size)
    assert _kv.same(got, plain.rotary_reference(x, positions, cos, sin, interleaved))


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rotary_layouts(gpu, offset):
    """Misaligned rows, shared positions, transposed tokens and heads."""
    base = _kv.rows((4, 6, 3, 72), "fp16", 3).cuda()
    cos, sin = (t.cuda() for t in _kv.tables(50, 64))
    positions = torch.tensor([3, 49, 0, 7, 7, 12]).cuda()
    x = base[..., offset:offset + 64]
    want = rotary_cuda(x.contiguous(), positions, cos, sin)
    assert _kv.same(rotary_cuda(x, positions, cos, sin), want)
    assert _kv.same(rotary_cuda(x[1], positions, cos, sin), want[1])
    turned = rotary_cuda(x.transpose(1, 2).contiguous().transpose(1, 2), positions.expand(4, 6), cos, sin)
    assert _kv.same(turned, want)


def test_rotary_many_rows(gpu):
    """Enough rows for four heads a thread, a head count that is no multiple of four."""
    x = _kv.rows((1, 5000, 29, 128), "bf16", 4).cuda()
    cos, sin = (t.cuda() for t in _kv.tables(5000, 64))
    positions = torch.arange(5000).cuda()
    got = rotary_cuda(x, positions, cos, sin)
    part = slice(0, 5000, 311)
    assert _kv.same(got[:, part], rotary_cuda(x[:, part].contiguous(), positions[part], cos, sin))
    assert _kv.same(got[..., 64:], x[..., 64:])


@pytest.mark.parametrize("dim", [64, 20])
def test_rotary_outside_the_tables(gpu, dim):
    x = torch.ones((4, 2, dim), dtype=torch.float16, device="cuda")
    cos, sin = (t.cuda() for t in _kv.tables(8, 16))
    got = rotary_cuda(x, torch.tensor([0, -1, 8, 1 << 40]).cuda(), cos, sin)
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1:, :, :16]).all()
    assert torch.equal(got[:, :, 16:], x[:, :, 16:])
    assert rotary_cuda(x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), cos, sin).shape == (0, 2, dim)
    none = rotary_cuda(x, torch.zeros(4, dtype=torch.int64, device="cuda"), cos[:0], sin[:0])
    assert torch.isnan(none[:, :, :16]).all()


# ----------------------------------------------------------------------- write and read

WRITES = [
    # block, slots, tokens, starts, counts
    (64, 64, 1, [40], None), (64, 100, 1, [0, 63, 64, 99], None), (16, 257, 3, [250, 14, 15, 16], None),
    (32, 96, 40, [0, 31, 56], [40, 0, 17]), (128, 300, 200, [100, 7], [200, 150]), (64, 70, 9, [-3, 65, 70, 200], None),
    (16, 33, 33, [0], [33]), (64, 1, 1, [0], None), (128, 130, 129, [1], None), (64, 64, 5, [-9, 1 << 62], [5, 99]),
]


@pytest.mark.parametrize("block,slots,tokens,starts,counts", WRITES)
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,dim,heads", [("fp16", 64, 3), ("bf16", 128, 2), ("fp16", 256, 1)])
def test_write(gpu, block, slots, tokens, starts, counts, codes, dtype, dim, heads):
    batch = len(starts)
    k, v = (_kv.rows((batch, tokens, heads, dim), dtype, i, spread) for i, spread in ((1, 3.0), (2, 0.01)))
    k[0, 0, 0, 3], v[-1, -1, -1, 0], k[-1, 0, 0, 1] = float("nan"), float("-inf"), float("inf")
    kc, ks = _kv.cache(batch, heads, slots, dim, codes, block, 3)
    vc, vs = _kv.cache(batch, heads, slots, dim, codes, block, 4)
    want_k = _kv.write(k, kc, ks, starts, counts, block)
    want_v = _kv.write(v, vc, vs, starts, counts, block)
    kc, ks, vc, vs = _dev(kc, ks, vc, vs)
    kv_write_cuda(*_dev(k, v), kc, ks, vc, vs, torch.tensor(starts).cuda(),
                  None if counts is None else torch.tensor(counts).cuda())
    for got, want in ((kc, want_k[0]), (ks, want_k[1]), (vc, want_v[0]), (vs, want_v[1])):
        assert np.array_equal(_kv.numbers(got), want)


def test_write_extremes(gpu):
    """The ends of the scales' range, zeros, ties and saturation."""
    x = torch.zeros((1, 96, 1, 64), dtype=torch.bfloat16)
    x[0, 0] = 2.0 ** -60
    x[0, 16] = 3e38
    x[0, 17] = 2.0 ** 100
    x[0, 32, 0] = torch.arange(64).float() / 2 + 63.5       # ties of int8 at a scale of 1
    x[0, 48, 0, :4] = torch.tensor([448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10])   # e4m3's end and its subnormals
    for codes in ("int8", "fp8"):
        kc, ks = torch.zeros((1, 1, 96, 64), dtype=_kv.CODES[codes]), torch.ones((1, 1, 6))
        want = _kv.write(x, kc, ks, [0], None, 16)
        kc, ks, vc, vs = _dev(kc, ks, kc.clone(), ks.clone())
        kv_write_cuda(x.cuda(), x.cuda(), kc, ks, vc, vs, torch.tensor([0]).cuda())
        assert np.array_equal(_kv.numbers(kc), want[0]) and np.array_equal(_kv.numbers(ks), want[1])
        assert _kv.same(kc, vc)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_growing_blocks(gpu, codes):
    """Token by token with growing values: the cache and the torch path stay bit for bit the same."""
    x = (_kv.rows((2, 50, 2, 64), "fp16", 5) * torch.linspace(0.01, 60, 50).view(1, 50, 1, 1)).half()
    on_gpu = QuantizedKVCache(2, 2, 60, 64, codes, 32, "cuda")
    on_cpu = QuantizedKVCache(2, 2, 60, 64, codes, 32, "cpu")
    start = torch.tensor([0, 9])
    for t in range(50):
        part = x[:, t:t + 1]
        on_gpu.write(part.cuda(), part.cuda(), (start + t).cuda())
        on_cpu.write(part, part, start + t)
    for a, b in zip(on_gpu.tensors(), on_cpu.tensors()):
        assert _kv.same(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("codes,dtype,dim,rot", [("int8", "fp16", 64, 64), ("fp8", "bf16", 128, 32),
                                                 ("int8", "bf16", 256, 256), ("fp8", "fp16", 64, 16)])
@pytest.mark.parametrize("tokens,starts,counts", [(1, [5, 77, 31], None), (70, [0, 10, 30], [70, 0, 64]),
                                                  (9, [95, -4, 1 << 50], None), (700, [3, 0, 9], None)])
def test_rotary_write_is_rotary_then_write(gpu, interleaved, codes, dtype, dim, rot, tokens, starts, counts):
    slots = 100 if tokens < 100 else 800
    qkv = _kv.rows((3, tokens, 9, dim), dtype, 6).cuda()
    q, k, v = qkv.split([5, 2, 2], dim=2)
    cos, sin = (t.cuda() for t in _kv.tables(slots + 3, rot))
    start, limit = torch.tensor(starts).cuda(), None if counts is None else torch.tensor(counts).cuda()
    first = [t.cuda() for t in (*_kv.cache(3, 2, slots, dim, codes, 64, 7), *_kv.cache(3, 2, slots, dim, codes, 64, 8))]
    second = [t.clone() for t in first]
    got = rotary_kv_write_cuda(q, k, v, cos, sin, *first, start, limit, interleaved)
    positions = start.clamp(max=slots).unsqueeze(1) + torch.arange(tokens, device="cuda")
    positions = torch.where(positions < slots, positions, -1)
    want = rotary_cuda(q, positions, cos, sin, interleaved)
    if limit is not None:
        want[torch.arange(tokens, device="cuda") >= limit.unsqueeze(1)] = 0
    kv_write_cuda(rotary_cuda(k, positions, cos, sin, interleaved), v, *second, start, limit)
    inside = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~inside) and torch.equal(got[inside], want[inside])
    for a, b in zip(first, second):
        assert _kv.same(a, b)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,block", [((1, 4, 2048, 64), 64), ((2, 3, 37, 128), 16), ((3, 1, 1, 256), 128),
                                         ((1, 2, 333, 80), 32)])
def test_read(gpu, codes, dtype, shape, block):
    c, s = _kv.cache(*shape, codes, block, 9)
    s[0, 0, 0] = 2.0 ** 11        # fp16 saturates
    s[-1, -1, -1] = 2.0 ** -24    # fp16's subnormals
    got = kv_read_cuda(c.cuda(), s.cuda(), dtype)
    most = torch.finfo(dtype).max
    want = torch.from_numpy(np.clip(_kv.values(c, s, block), -most, most)).to(dtype)
    assert got.is_contiguous() and _kv.same(got, want)


def test_read_views_and_all_codes(gpu):
    every = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(1, 1, 4, 64).expand(1, 2, 4, 64).contiguous()
    s = torch.ones((1, 2, 1))
    for dtype in (torch.int8, torch.float8_e4m3fn):
        got = kv_read_cuda(every.view(dtype).cuda(), s.cuda(), torch.float32).cpu()
        want = every.view(dtype).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    c, s = (t.cuda() for t in _kv.cache(3, 4, 200, 64, "int8", 32, 10))
    want = kv_read_cuda(c, s)
    assert _kv.same(kv_read_cuda(c[1:, 1:3, :70], s[1:, 1:3, :3]), want[1:, 1:3, :70])
    assert kv_read_cuda(c[:0], s[:0]).shape == (0, 4, 200, 64)


# --------------------------------------------------------------------------- attention

def _check(q, kc, ks, vc, vs, starts, counts, block, scale=None, what=""):
    want, bound = _kv.attend(q, kc, ks, vc, vs, starts, counts, block, scale)
    got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor(starts).cuda(),
                            None if counts is None else torch.tensor(counts).cuda(), scale)
    assert got.is_contiguous()
    _kv.close(got, want, bound, what)
    return got


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(8, 1, 1), (4, 2, 5), (14, 2, 4), (32, 1, 2), (4, 1, 40), (2, 2, 130)])
def test_attention(gpu, dim, codes, dtype, heads, kv_heads, tokens):
    """Every form: 16, 32 and 64 rows of a KV head, prompts; sequences that hold nothing, a few slots, many."""
    starts = [0, 1, 61, 300]
    slots, block = 300 + tokens, {64: 64, 128: 16, 256: 32}[dim]
    q = _kv.rows((4, tokens, heads, dim), dtype, 11)
    kc, ks = _kv.cache(4, kv_heads, slots, dim, codes, block, 12)
    vc, vs = _kv.cache(4, kv_heads, slots, dim, codes, block, 13)
    _check(q, kc, ks, vc, vs, starts, None, block)


@pytest.mark.parametrize("held", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
@pytest.mark.parametrize("tokens", [1, 33])
def test_attention_lengths(gpu, held, tokens):
    dim, block = 64, 128
    q = _kv.rows((1, tokens, 4, dim), "fp16", held)
    kc, ks = _kv.cache(1, 2, 300, dim, "int8", block, 14)
    vc, vs = _kv.cache(1, 2, 300, dim, "int8", block, 15)
    _check(q, kc, ks, vc, vs, [held - 1], None, block)


@pytest.mark.parametrize("tokens,heads", [(1, 8), (6, 8), (20, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_shares_of_a_long_cache(gpu, tokens, heads, dim):
    """One sequence of a long cache: the slots are divided, some shares hold none."""
    q = _kv.rows((2, tokens, heads, dim), "fp16", 16)
    kc, ks = _kv.cache(2, 2, 5000, dim, "fp8", 64, 17)
    vc, vs = _kv.cache(2, 2, 5000, dim, "fp8", 64, 18)
    _check(q, kc, ks, vc, vs, [4970, 40], None, 64)


@pytest.mark.parametrize("tokens", [1, 3, 50])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_attention_ignores_what_lies_behind(gpu, codes, tokens):
    """Slots behind a sequence's tokens, NaN codes and scales of any size among
    them, padding rows and positions outside the cache."""
    q = _kv.rows((5, tokens, 4, 64), "bf16", 19)
    kc, ks = _kv.cache(5, 2, 400, 64, codes, 16, 20)
    vc, vs = _kv.cache(5, 2, 400, 64, codes, 16, 21)
    starts, counts = [37, 0, 395, 10, -2], [tokens, tokens // 2, tokens, 0, tokens]
    want, bound = _kv.attend(q, kc, ks, vc, vs, starts, counts, 16)
    for b, (start, count) in enumerate(zip(starts, counts)):
        end = max(start + count, 0)
        for c, s in ((kc, ks), (vc, vs)):
            c[b, :, end:].view(torch.uint8).fill_(0x7F)
            s[b, :, -(-end // 16):] = 2.0 ** 40
    got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor(starts).cuda(), torch.tensor(counts).cuda())
    _kv.close(got, want, bound)
    assert torch.equal(got[3].cpu(), torch.zeros_like(q[3]))
    assert torch.isnan(got[4, 0]).all()
    padded = got[1, tokens // 2:]
    assert torch.equal(padded, torch.zeros_like(padded))


@pytest.mark.parametrize("tokens", [1, 50])
@pytest.mark.parametrize("slots", [90, 2000])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), -3.0, 0.0, 1e-45, 3e38])
def test_attention_ignores_scales_that_lie_behind(gpu, tokens, slots, junk):
    """Scales of blocks without tokens are never written: memory as it was allocated."""
    q = _kv.rows((3, tokens, 4, 64), "fp16", 57)
    kc, ks = _kv.cache(3, 2, slots, 64, "fp8", 16, 58)
    vc, vs = _kv.cache(3, 2, slots, 64, "fp8", 16, 59)
    starts = [3, 17, slots // 2 - tokens]
    want, bound = _kv.attend(q, kc, ks, vc, vs, starts, None, 16)
    for b, start in enumerate(starts):
        ks[b, :, -(-(start + tokens) // 16):] = junk
        vs[b, :, -(-(start + tokens) // 16):] = junk
    got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor(starts).cuda())
    _kv.close(got, want, bound)


@pytest.mark.parametrize("tokens", [1, 9, 60])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_attention_shares_with_padding(gpu, codes, tokens):
    """Divided slots: padding rows, rows outside the cache, sequences of one share and of many."""
    q = _kv.rows((5, tokens, 8, 64), "fp16", 51)
    kc, ks = _kv.cache(5, 1, 2500, 64, codes, 32, 52)
    vc, vs = _kv.cache(5, 1, 2500, 64, codes, 32, 53)
    starts, counts = [2400, 3, 2495, 1200, -4], [tokens, tokens // 2, tokens, 0, tokens]
    want, bound = _kv.attend(q, kc, ks, vc, vs, starts, counts, 32)
    for b, (start, count) in enumerate(zip(starts, counts)):
        end = max(start + count, 0)
        vc[b, :, end:].view(torch.uint8).fill_(0x7F)
    got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor(starts).cuda(), torch.tensor(counts).cuda())
    _kv.close(got, want, bound)


@pytest.mark.parametrize("dim,codes,dtype", [(64, "int8", "bf16"), (64, "fp8", "fp16"), (128, "int8", "fp16"),
                                             (128, "fp8", "bf16")])
def test_attention_of_many_prompts(gpu, dim, codes, dtype):
    """Enough rows for workgroups of 256 of them; ragged, some of one sequence padding."""
    q = _kv.rows((64, 36, 16, dim), dtype, 54)
    kc, ks = _kv.cache(64, 8, 150, dim, codes, 64, 55)
    vc, vs = _kv.cache(64, 8, 150, dim, codes, 64, 56)
    starts = [(7 * b) % 100 for b in range(64)]
    counts = [36 - b % 5 for b in range(64)]
    got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor(starts).cuda(), torch.tensor(counts).cuda())
    for b in (0, 14, 63):
        one = slice(b, b + 1)
        want, bound = _kv.attend(q[one], kc[one], ks[one], vc[one], vs[one], starts[one], counts[one], 64)
        _kv.close(got[one], want, bound)


@pytest.mark.parametrize("tokens", [1, 70])
def test_attention_of_unequal_values(gpu, tokens):
    """Blocks of values 2^30 apart: the weights keep their precision, whichever
    block a row's weight lies in."""
    q = _kv.rows((2, tokens, 2, 64), "fp16", 22, 4.0)
    kc, ks = _kv.cache(2, 1, 200, 64, "int8", 16, 23)
    vc, vs = _kv.cache(2, 1, 200, 64, "int8", 16, 24)
    vs[0, 0, ::2] = 2.0 ** -24
    vs[1, 0] = 2.0 ** -24
    vs[1, 0, 7] = 2.0 ** 6
    kc[1, 0, 112:128] = 0    # little weight on the large values of the second sequence
    q[1] = q[1].abs()
    kc[1, 0, :112] = kc[1, 0, :112].abs()
    _check(q, kc, ks, vc, vs, [200 - tokens] * 2, None, 16)


@pytest.mark.parametrize("scale", [1.0, 0.01, 0.0, -0.125])
def test_attention_scales(gpu, scale):
    for tokens in (1, 40):
        q = _kv.rows((1, tokens, 4, 64), "fp16", 25)
        kc, ks = _kv.cache(1, 2, 120, 64, "fp8", 32, 26)
        vc, vs = _kv.cache(1, 2, 120, 64, "fp8", 32, 27)
        _check(q, kc, ks, vc, vs, [80], None, 32, scale)


@pytest.mark.parametrize("factor", [2.0 ** -100, 2.0 ** -30, 2.0 ** 40, 0.0])
@pytest.mark.parametrize("tokens", [1, 70])
def test_attention_of_bf16_magnitudes(gpu, factor, tokens):
    """Queries far outside fp16's range: scores from nearly equal to one-hot."""
    q = (_kv.rows((1, tokens, 2, 128), "fp32", 28) * factor).bfloat16()
    kc, ks = _kv.cache(1, 1, 90, 128, "int8", 32, 29)
    vc, vs = _kv.cache(1, 1, 90, 128, "int8", 32, 30)
    ks *= 2.0 ** -20 if factor > 1 else 1.0
    _check(q, kc, ks, vc, vs, [90 - tokens], None, 32, 2.0 ** -20 if factor > 1 else None)


def test_attention_of_values_that_are_not_finite(gpu):
    """A NaN or infinite query makes its own row NaN and no other."""
    for tokens in (4, 70):
        q = _kv.rows((1, tokens, 2, 64), "fp16", 31)
        kc, ks = _kv.cache(1, 1, 100, 64, "int8", 64, 32)
        vc, vs = _kv.cache(1, 1, 100, 64, "int8", 64, 33)
        want = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor([20]).cuda())
        q[0, 1, 0, 5], q[0, 2, 1, 9] = float("nan"), float("inf")
        got = kv_attention_cuda(*_dev(q, kc, ks, vc, vs), torch.tensor([20]).cuda())
        mine = torch.zeros((tokens, 2), dtype=torch.bool)
        mine[1, 0] = mine[2, 1] = True
        assert torch.isnan(got[0][mine.cuda()]).all() and _kv.same(got[0][~mine.cuda()], want[0][~mine.cuda()])


def test_attention_layouts(gpu):
    """Strided and misaligned queries, views of a larger cache, one head for all (the cache's stride 0)."""
    for tokens in (2, 80):
        big = _kv.rows((2, tokens, 7, 72), "fp16", 34).cuda()
        kc, ks, vc, vs = (t.cuda() for t in (*_kv.cache(3, 4, 200, 64, "int8", 32, 35),
                                             *_kv.cache(3, 4, 200, 64, "int8", 32, 36)))
        start = torch.tensor([90, 3]).cuda()
        view = (kc[1:, 1:3, :190], ks[1:, 1:3, :6], vc[1:, 1:3, :190], vs[1:, 1:3, :6])
        whole = tuple(t.contiguous() for t in view)
        for offset in (0, 3, 8):
            q = big[:, :, 1:5, offset:offset + 64]
            want = kv_attention_cuda(q.contiguous(), *whole, start)
            assert _kv.same(kv_attention_cuda(q, *view, start), want)
            swapped = q.transpose(1, 2).contiguous().transpose(1, 2)
            assert _kv.same(kv_attention_cuda(swapped, *view, start), want)
        q = big[:, :, 1:5, :64].contiguous()
        shared = tuple(t[:1, :1].expand(2, 2, *t.shape[2:]) for t in whole)
        assert _kv.same(kv_attention_cuda(q, *shared, start), kv_attention_cuda(q, *(t.contiguous() for t in shared), start))


@pytest.mark.parametrize("tokens", [1, 30])
def test_long_offsets(gpu, tokens):
    """A head of more than 2^31 bytes and batches further apart than that."""
    slots, dim = (1 << 23) + 300, 256
    kc, vc = (torch.zeros((2, 1, slots, dim), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((2, 1, -(-slots // 64)), 2.0 ** -6, device="cuda") for _ in range(2))
    start = slots - tokens
    k, v = (_kv.rows((2, tokens, 1, dim), "fp16", i).cuda() for i in (37, 38))
    starts = torch.tensor([start, start]).cuda()
    kv_write_cuda(k, v, kc, ks, vc, vs, starts)
    block = slots - slots % 64
    assert start >= block
    tail_k, tail_v = (kv_read_cuda(c[:, :, block:], s[:, :, block // 64:], torch.float32)[:, :, start - block:]
                      for c, s in ((kc, ks), (vc, vs)))
    q = _kv.rows((2, tokens, 2, dim), "fp16", 39)
    got = kv_attention_cuda(q.cuda(), kc, ks, vc, vs, starts)
    # all slots before have score 0 and value 0
    kk, vv, qq = tail_k[:, 0].double().cpu(), tail_v[:, 0].double().cpu(), q.double()
    scores = torch.einsum("bthd,bsd->bhts", qq, kk) / 16
    scores = scores.masked_fill(torch.arange(tokens) > torch.arange(tokens).unsqueeze(1), float("-inf"))
    weights = torch.exp(scores)
    total = weights.sum(-1, keepdim=True) + start
    want = torch.einsum("bhts,bsd->bthd", weights / total, vv)
    sizes = torch.einsum("bhts,bsd->bthd", weights / total, vv.abs())
    # weights within fp16's rounding (2^-11; 2^-25 of the largest below its normal
    # range), the sum of 2^23 ones in fp32 by parts of at most 2^20: 2^-12 at most
    bound = (2.0 ** -11 + 2.0 ** -12) * sizes + tokens * 2.0 ** -25 * 2 * vv.abs().max() * (weights / total).max()
    _kv.close(got, want.numpy(), bound.numpy())
    del kc, vc


# ----------------------------------------------------------- together, streams, graphs

def _model_step(cache, qkv, heads, kv, cos, sin, start):
    q, k, v = qkv.split([heads, kv, kv], dim=2)
    return cache.attend(cache.rotary_write(q, k, v, cos, sin, start), start)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_prompt_then_tokens(gpu, codes):
    """A prompt and then tokens, as a decoder runs them: GPU against the torch
    path, and near attention over the unquantized keys and values."""
    heads, kv, dim, prompt, steps = 8, 2, 64, 45, 30
    data = _kv.rows((2, prompt + steps, heads + 2 * kv, dim), "fp16", 40)
    cos, sin = _kv.tables(90, dim)
    on_gpu, on_cpu = (QuantizedKVCache(2, kv, 90, dim, codes, 16, d) for d in ("cuda", "cpu"))
    outs = []
    for start, part in [(0, data[:, :prompt])] + [(t, data[:, t:t + 1]) for t in range(prompt, prompt + steps)]:
        at = torch.tensor([start, start])
        got = _model_step(on_gpu, part.cuda(), heads, kv, cos.cuda(), sin.cuda(), at.cuda())
        turned = on_cpu.rotary_write(*part.split([heads, kv, kv], dim=2), cos, sin, at)
        want, bound = _kv.attend(turned, *on_cpu.tensors(), [start] * 2, None, 16)
        _kv.close(got, want, bound)
        outs.append(got)
    for a, b in zip(on_gpu.tensors(), on_cpu.tensors()):
        assert _kv.same(a, b)
    keys, values = on_gpu.read(75)
    positions = torch.arange(75).expand(2, 75)
    exact_k, _ = _kv.rotate(data[:, :, heads:heads + kv], cos, sin, positions, False)
    # a code is off by half a step of its block's last scale and by half a step of each growth before
    step = _kv.numbers(on_gpu.k_scales).max() * (1 if codes == "int8" else 32)
    assert np.abs(_kv.numbers(keys).transpose(0, 2, 1, 3) - exact_k).max() <= 1.5 * step
    assert values.shape == (2, kv, 75, dim) and torch.isfinite(torch.cat(outs, dim=1)).all()


@pytest.mark.parametrize("slots", [128, 3000])
def test_captured_step(gpu, slots):
    """A decode step in a HIP graph, replayed with eager work between: every
    replay equals the eager step (long caches are attended in shares)."""
    heads, kv, dim = 8, 2, 64
    cos, sin = (t.cuda() for t in _kv.tables(slots, dim))
    captured, eager = (QuantizedKVCache(1, kv, slots, dim, "int8", 64, "cuda") for _ in range(2))
    data = _kv.rows((1, 100, heads + 2 * kv, dim), "fp16", 41).cuda()
    start = torch.zeros((1,), dtype=torch.int64, device="cuda")
    qkv = torch.zeros((1, 1, heads + 2 * kv, dim), dtype=torch.float16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _model_step(captured, qkv, heads, kv, cos, sin, start)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _model_step(captured, qkv, heads, kv, cos, sin, start)
        start.add_(1)
    start.zero_()
    for t in range(6):
        qkv.copy_(data[:, t:t + 1])
        graph.replay()
        want = _model_step(eager, data[:, t:t + 1], heads, kv, cos, sin, torch.tensor([t]).cuda())
        noise = torch.randn((1000, 1000), device="cuda") @ torch.randn((1000, 1000), device="cuda")
        torch.cuda.synchronize()
        assert _kv.same(out, want) and torch.isfinite(noise).all()
    for a, b in zip(captured.tensors(), eager.tensors()):
        assert _kv.same(a, b)


def test_streams(gpu):
    """Calls on another stream, two at once: each has a workspace of its own."""
    q = _kv.rows((1, 1, 8, 64), "fp16", 42).cuda()
    caches = [tuple(t.cuda() for t in (*_kv.cache(1, 2, 4000, 64, "int8", 64, s), *_kv.cache(1, 2, 4000, 64, "int8", 64, s + 1)))
              for s in (43, 45)]
    start = torch.tensor([3999]).cuda()
    want = [kv_attention_cuda(q, *c, start) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, caches)):
            with torch.cuda.stream(s):
                got[i].append(kv_attention_cuda(q, *c, start))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(_kv.same(g, want[i]) for g in got[i])


def test_runs_agree(gpu):
    """The same call gives the same bits."""
    for tokens, batch in ((1, 3), (90, 2)):
        q = _kv.rows((batch, tokens, 8, 128), "bf16", 47).cuda()
        c = [t.cuda() for t in (*_kv.cache(batch, 2, 3000, 128, "fp8", 32, 48), *_kv.cache(batch, 2, 3000, 128, "fp8", 32, 49))]
        start = torch.tensor([2900, 17, 1000][:batch]).cuda()
        want = kv_attention_cuda(q, *c, start)
        assert all(_kv.same(kv_attention_cuda(q, *c, start), want) for _ in range(5))


def test_compiled_step(gpu):
    """torch.compile traces the ops, writes into the cache included."""
    cos, sin = (t.cuda() for t in _kv.tables(64, 64))
    start = torch.tensor([3]).cuda()
    data = _kv.rows((1, 2, 8, 64), "fp16", 50).cuda()
    a, b = (QuantizedKVCache(1, 2, 64, 64, "int8", 64, "cuda") for _ in range(2))

    def step(x, kc, ks, vc, vs):
        q, k, v = x.split([4, 2, 2], dim=2)
        turned = nibble_amd.rotary_kv_write_cuda(q, k, v, cos, sin, kc, ks, vc, vs, start)
        return nibble_amd.kv_attention_cuda(turned, kc, ks, vc, vs, start)

    compiled = torch.compile(step, backend="eager", fullgraph=True)
    assert _kv.same(compiled(data, *a.tensors()), step(data, *b.tensors()))
    assert _kv.same(a.k_codes, b.k_codes)
