"""Forking and reordering caches on the GPU: every byte of the tensors, also of
those that stay."""

import pytest
import torch

from nibble_amd import QuantizedKVCache, kv_fork_cuda, kv_reorder_cuda
from tests import _moves

pytestmark = pytest.mark.gpu


def _ints(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def test_refusals(gpu):
    make = lambda batch=2, heads=2, slots=40, dim=64, codes="int8", block=16: _moves.tensors(batch, heads, slots, dim, codes, block, 1, "cuda")  # noqa: E731,E501
    a, b, two = make(), make(), _ints([0, 1])
    for other in (make(heads=3), make(dim=128), make(codes="fp8"), make(block=32)):
        with pytest.raises(RuntimeError, match="same KV heads"):
            kv_fork_cuda(*a, *other, two, two)
    for message, call in [("must not share memory", lambda: kv_fork_cuda(*a, *a, two, two)),
                          ("source must be contiguous", lambda: kv_fork_cuda(*a, *b, _ints([0]), two)),
                          ("lengths must be contiguous", lambda: kv_fork_cuda(*make(batch=3), *b, two, two)),
                          ("source must have dtype", lambda: kv_reorder_cuda(*a, two.int(), two)),
                          ("lengths must be on", lambda: kv_reorder_cuda(*a, two, two.cpu())),
                          ("overlap", lambda: kv_reorder_cuda(a[0][:1].expand(2, -1, -1, -1), *a[1:], two, two)),
                          ("at most 262144", lambda: kv_reorder_cuda(*make(batch=1025, heads=1, slots=1, dim=256), _ints([0] * 1025),
                                                                     _ints([0] * 1025)))]:
        with pytest.raises(RuntimeError, match=message):
            call()


@pytest.mark.parametrize("held,slots,batch,to_slots,block,source,lengths", _moves.FORKS)
@pytest.mark.parametrize("dim,codes,pad", [(64, "int8", 0), (128, "fp8", 1), (256, "int8", 2)])
def test_fork(gpu, held, slots, batch, to_slots, block, source, lengths, dim, codes, pad):
    a = _moves.tensors(held, 3, slots, dim, codes, block, 1, "cuda", pad)
    b = _moves.tensors(batch, 3, to_slots, dim, codes, block, 5, "cuda")
    before = [x.clone() for x in a]
    want = _moves.expected(a, b, source, lengths, block)
    kv_fork_cuda(*a, *b, _ints(source), _ints(lengths))
    _moves.check(b, want)
    _moves.check(a, before)


@pytest.mark.parametrize("batch,slots,block,source,lengths", _moves.REORDERS)
@pytest.mark.parametrize("dim,codes,pad", [(64, "int8", 0), (128, "fp8", 1), (256, "int8", 2)])
def test_reorder(gpu, batch, slots, block, source, lengths, dim, codes, pad):
    a = _moves.tensors(batch, 3, slots, dim, codes, block, 9, "cuda", pad)
    want = _moves.expected(a, a, source, lengths, block)
    kv_reorder_cuda(*a, _ints(source), _ints(lengths))
    _moves.check(a, want)


@pytest.mark.parametrize("batch,slots,dim", [(31, 700, 128), (64, 65, 64), (70, 140, 256), (257, 33, 256), (300, 40, 64),
                                             (1024, 3, 256), (1025, 17, 128)])
def test_reorder_many(gpu, batch, slots, dim):
    """Beams of all sizes: any sequence from any other, some from outside."""
    g = torch.Generator().manual_seed(batch)
    source = torch.randint(-2, batch + 2, (batch,), generator=g).tolist()
    lengths = torch.randint(0, slots + 1, (batch,), generator=g).tolist()
    a = _moves.tensors(batch, 2, slots, dim, "int8", 16, 3, "cuda")
    want = _moves.expected(a, a, source, lengths, 16)
    kv_reorder_cuda(*a, _ints(source), _ints(lengths))
    _moves.check(a, want)


def test_interleaved_sides(gpu):
    """Keys and values in one buffer, and a cache whose first sequence is the other's last."""
    both = _moves.tensors(4, 4, 50, 64, "int8", 16, 7, "cuda")
    a = (both[0][:, :2], both[1][:, :2], both[0][:, 2:], both[1][:, 2:])
    want = _moves.expected(a, a, [3, 2, 1, 0], [50, 49, 16, 17], 16)
    kv_reorder_cuda(*a, _ints([3, 2, 1, 0]), _ints([50, 49, 16, 17]))
    _moves.check(a, want)
    first, rest = [x[:1] for x in both], [x[1:] for x in both]
    want = _moves.expected(first, rest, [0, -1, 0], [33], 16)
    kv_fork_cuda(*first, *rest, _ints([0, -1, 0]), _ints([33]))
    _moves.check(rest, want)


def test_captured(gpu):
    """A replayed call reads new sources and lengths."""
    a = _moves.tensors(5, 2, 300, 64, "int8", 32, 11, "cuda")
    b = _moves.tensors(8, 2, 400, 64, "int8", 32, 12, "cuda")
    order, source, lengths = _ints([0] * 5), _ints([0] * 8), _ints([0] * 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_reorder_cuda(*a, order, lengths)
        kv_fork_cuda(*a, *b, source, lengths)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        new = [torch.randint(5, (n,), generator=g).tolist() for n in (5, 8)] + [torch.randint(301, (5,), generator=g).tolist()]
        for x, y in zip((order, source, lengths), new):
            x.copy_(_ints(y))
        first = _moves.expected(a, a, new[0], new[2], 32)
        second = _moves.expected(first, b, new[1], new[2], 32)
        graph.replay()
        torch.cuda.synchronize()
        _moves.check(a, first)
        _moves.check(b, second)


def test_methods(gpu):
    a = QuantizedKVCache(2, 2, 100, 64, "fp8", 64, "cuda")
    b = QuantizedKVCache(3, 2, 80, 64, "fp8", 64, "cuda")
    k = torch.randn((2, 100, 2, 64), dtype=torch.float16, device="cuda")
    a.write(k, k.flip(1), _ints([0, 0]))
    b.fork_from(a, _ints([1, 0, 1]), _ints([70, 80]))
    want = _moves.expected(b.tensors(), b.tensors(), [2, 0, 1], [80, 70, 80], 64)
    b.reorder(_ints([2, 0, 1]), _ints([80, 70, 80]))
    _moves.check(b.tensors(), want)
