"""Attention behind shared prefixes on the GPU against the 64-bit oracle."""

import pytest
import torch

from nibble_amd import QuantizedKVCache, kv_attention_cuda, kv_shared_attention_cuda
from tests import _kv, _shared
from tests.test_kv_shared_cpu import CASES

pytestmark = pytest.mark.gpu


def _ints(values):
    return None if values is None else torch.tensor(values, dtype=torch.int64, device="cuda")


def _run(q, prefix, lengths, own, start, counts=None, scale=None):
    return kv_shared_attention_cuda(q.cuda(), *[x.cuda() for x in prefix], _ints(lengths), *[x.cuda() for x in own],
                                    _ints(start), _ints(counts), scale)


def _check(q, prefix, lengths, own, start, counts=None, prefix_block=64, block=32, scale=None):
    got = _run(q, prefix, lengths, own, start, counts, scale)
    ref, bound = _shared.attend(q, prefix, lengths, own, start, counts, prefix_block, block, scale)
    _kv.close(got, ref, bound)
    return got


def test_refusals(gpu):
    q, prefix, own = _shared.case(2, 2, 1, 4, 2, 64, 30, 20)
    lengths, start = [30, 30], [0] * 4
    for message, bad in [("positive multiple", dict(q=q[:, :, :3])), ("of the cache", dict(q=q[:3])),
                         ("same KV heads", dict(prefix=[x[:, :1] for x in prefix])),
                         ("prefix_lengths must be contiguous", dict(lengths=[30])),
                         ("multiple of the prefixes", dict(prefix=[torch.cat((x, x[:1])) for x in prefix], lengths=[1] * 3)),
                         ("finite", dict(scale=float("nan"))), ("start must be contiguous", dict(start=[0, 0])),
                         ("torch.float16 or", dict(q=q.float())), ("must not require grad", dict(q=q.clone().requires_grad_()))]:
        with pytest.raises(RuntimeError, match=message):
            _run(**{**dict(q=q, prefix=prefix, lengths=lengths, own=own, start=start), **bad})
    mixed = [x.view(torch.float8_e4m3fn) if x.dtype == torch.int8 else x for x in prefix]
    with pytest.raises(RuntimeError, match="and codes"):
        _run(q, mixed, lengths, own, start)
    with pytest.raises(RuntimeError, match="prefix_lengths must be on"):
        kv_shared_attention_cuda(q.cuda(), *[x.cuda() for x in prefix], torch.tensor([1, 1]), *[x.cuda() for x in own],
                                 _ints(start))


@pytest.mark.parametrize("groups,per,tokens,lengths,start,counts", CASES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
def test_lengths(gpu, groups, per, tokens, lengths, start, counts, codes, dtype, dim):
    _check(*_mix(_shared.case(groups, per, tokens, 6, 2, dim, 50, 20, codes, dtype), lengths), start, counts)


def _mix(case, lengths):
    q, prefix, own = case
    return q, prefix, lengths, own


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("groups,per,heads,kv_heads,tokens", [(1, 3, 2, 1, 1), (1, 9, 8, 4, 1), (2, 5, 14, 2, 1),
                                                              (1, 20, 8, 2, 2), (2, 3, 4, 1, 9), (1, 3, 4, 2, 70)])
def test_layouts_of_heads(gpu, dim, codes, dtype, groups, per, heads, kv_heads, tokens):
    """Rows of a prefix and of a sequence in every form: few, up to 64, many."""
    batch = groups * per
    q, prefix, own = _shared.case(groups, per, tokens, heads, kv_heads, dim, 300, 130, codes, dtype, 32, 16)
    _check(q, prefix, [299 - 40 * g for g in range(groups)], own, [(17 * b) % (131 - tokens) for b in range(batch)], None, 32, 16)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 400])
@pytest.mark.parametrize("per,tokens", [(2, 1), (5, 1), (30, 1), (3, 12)])
def test_prefix_lengths(gpu, length, per, tokens):
    q, prefix, own = _shared.case(1, per, tokens, 8, 2, 64, 400, 48)
    _check(q, prefix, [length], own, [b % 37 for b in range(per)])


@pytest.mark.parametrize("per,tokens,heads", [(4, 1, 8), (20, 1, 8), (40, 1, 16)])
@pytest.mark.parametrize("dim", [64, 128])
def test_shares_of_long_prefixes(gpu, per, tokens, heads, dim):
    q, prefix, own = _shared.case(1, per, tokens, heads, 2, dim, 5003, 2100)
    _check(q, prefix, [5001], own, [(b * 523) % 2099 for b in range(per)])


@pytest.mark.parametrize("length", [0, 1, 700, 5000])
@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
def test_many_rows_in_a_large_cache(gpu, codes, dtype, length):
    """Tokens of many sequences behind a prefix cache of many slots, however few are held; padding among them."""
    q, prefix, own = _shared.case(1, 20, 1, 16, 2, 64, 42000, 60, codes, dtype)
    _check(q, prefix, [length], own, [(7 * b) % 60 for b in range(20)], [b % 3 for b in range(20)])
    big = [x * 2.0 ** 16 if i == 1 else x for i, x in enumerate(prefix)]
    _check(q, big, [length], own, [(7 * b) % 60 for b in range(20)])


@pytest.mark.parametrize("groups,per,tokens", [(1, 3, 40), (2, 1, 90), (1, 20, 17)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
def test_prompts_behind_long_prefixes(gpu, codes, dtype, dim, groups, per, tokens):
    """Several shares of a prefix, joined by the launch over the sequences' own slots or by one of its own."""
    q, prefix, own = _shared.case(groups, per, tokens, 8, 2, dim, 3001, 1100 if tokens == 40 else 130, codes, dtype)
    batch = groups * per
    lengths, start = [2999 - 1700 * g for g in range(groups)], [(37 * b) % (131 - tokens) for b in range(batch)]
    counts = [max(tokens - 29 * b, 0) for b in range(batch)]
    _check(q, prefix, lengths, own, start, counts)
    big = [x * 2.0 ** 16 if i == 1 else x for i, x in enumerate(prefix)]     # attended to row by row
    got = _check(q, big, lengths, own, start, counts)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_what_lies_behind(gpu, codes, tokens):
    """Slots, scales and workspace that hold anything: NaN codes, any scales."""
    q, prefix, own = _shared.case(2, 3, tokens, 8, 2, 64, 200, 90, codes)
    lengths, start, counts = [100, 33], [0, 9, 31, 32, 40, 47], [tokens, 0, tokens, 1, tokens, tokens]
    clean = _run(q, prefix, lengths, own, start, counts)
    for junk in (float("nan"), float("inf"), 0.0, -3.0):
        p, o = [x.clone() for x in prefix], [x.clone() for x in own]
        for tensors, ends, block in ((p, lengths, 64), (o, [s + c for s, c in zip(start, counts)], 32)):
            for i, end in enumerate(ends):
                for x in (tensors[0], tensors[2]):
                    x.view(torch.int8)[i, :, end:] = 0x7F
                for x in (tensors[1], tensors[3]):
                    x[i, :, -(-end // block):] = junk
        rows = q.clone()
        for b, c in enumerate(counts):
            rows[b, c:] = float("nan")          # padding
        filler = torch.full((1 << 22,), float("nan"), device="cuda")   # what a workspace may find
        del filler
        assert _kv.same(_run(rows, p, lengths, o, start, counts), clean)


@pytest.mark.parametrize("tokens,counts", [(30, [30, 0, 7, 0]), (100, [0, 0, 0, 0]), (100, [1, 100, 0, 64]), (2, [-3, 5, 1, 2])])
def test_padding(gpu, tokens, counts):
    q, prefix, own = _shared.case(2, 2, tokens, 8, 1, 128, 150, 160)
    got = _check(q, prefix, [150, 31], own, [0, 5, 60, 1], counts)
    for b, c in enumerate(counts):
        assert (got[b, max(c, 0):] == 0).all()


@pytest.mark.parametrize("scale", [1.0, 0.01, 0.0, -0.125])
@pytest.mark.parametrize("per", [3, 24])
def test_scales(gpu, scale, per):
    q, prefix, own = _shared.case(1, per, 1, 8, 2, 64, 130, 40)
    _check(q, prefix, [129], own, [b % 40 for b in range(per)], scale=scale)


@pytest.mark.parametrize("per", [3, 40])
def test_sides_of_unequal_scores(gpu, per):
    """A prefix whose scores are far above a sequence's own, and the other way round."""
    q, prefix, own = _shared.case(1, per, 1, 8, 2, 64, 130, 40)
    for factor in (2.0 ** -12, 2.0 ** 6):
        scaled = [x * factor if i == 1 else x for i, x in enumerate(prefix)]
        _check(q, scaled, [130], own, [b % 40 for b in range(per)])


@pytest.mark.parametrize("per", [3, 40])
def test_scores_past_2_to_22(gpu, per):
    """Large scores beside ordinary ones: weights, not NaN."""
    q, prefix, own = _shared.case(1, per, 1, 8, 2, 64, 130, 40)
    big = [x * 2.0 ** 16 if i == 1 else x for i, x in enumerate(prefix)]
    got = _check(q, big, [130], own, [b % 40 for b in range(per)])
    assert torch.isfinite(got).all()


def test_views_and_strides(gpu):
    """Queries of a fused projection, caches of another layout, unaligned rows."""
    q, prefix, own = _shared.case(2, 2, 3, 8, 2, 64, 60, 50)
    lengths, start = [60, 20], [0, 3, 30, 47]
    want = _run(q, prefix, lengths, own, start)
    wide = torch.zeros((4, 3, 12, 64), dtype=q.dtype, device="cuda")
    wide[:, :, 2:10] = q.cuda()
    inner = torch.zeros((4, 3, 8, 65), dtype=q.dtype, device="cuda")
    inner[..., 1:] = q.cuda()
    heads_first = q.cuda().permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    for view in (wide[:, :, 2:10], inner[..., 1:], heads_first):
        got = kv_shared_attention_cuda(view, *[x.cuda() for x in prefix], _ints(lengths), *[x.cuda() for x in own], _ints(start))
        assert _kv.same(got, want)
    # one prefix for both groups by a stride of 0, and a cache's leading slots
    same = [x[:1].cuda().expand(2, *x.shape[1:]) for x in prefix]
    got = kv_shared_attention_cuda(q.cuda(), *same, _ints([60, 60]), *[x.cuda() for x in own], _ints(start))
    ref, bound = _shared.attend(q, [x.cpu() for x in same], [60, 60], own, start, None, 64, 32)
    _kv.close(got, ref, bound)


def test_agrees_with_one_cache(gpu):
    """The same keys and values in one cache a sequence: the same rows up to rounding."""
    q, prefix, own = _shared.case(1, 4, 1, 32, 4, 64, 128, 64, prefix_block=64, block=64)
    whole = [torch.cat((p.expand(4, *p.shape[1:]), o), dim=2).cuda() for p, o in zip(
        [x.view(torch.int8) if i % 2 == 0 else x for i, x in enumerate(prefix)],
        [x.view(torch.int8) if i % 2 == 0 else x for i, x in enumerate(own)])]
    start = [0, 20, 40, 63]
    one = kv_attention_cuda(q.cuda(), *whole, _ints([128 + s for s in start]))
    ref, bound = _shared.attend(q, prefix, [128], own, start, None, 64, 64)
    _kv.close(one, ref, bound)
    _kv.close(_run(q, prefix, [128], own, start), ref, bound)


@pytest.mark.parametrize("per", [2, 24])
def test_long_offsets(gpu, per):
    """A prefix and sequences that end more than 2^32 bytes behind their caches' start."""
    slots = (1 << 32) // 64 // 2 + 200
    q, prefix, own = _shared.case(1, per, 1, 4, 2, 64, 130, 40)
    big = torch.zeros((1, 2, slots, 64), dtype=torch.int8, device="cuda")
    scales = torch.ones((1, 2, -(-slots // 64)), device="cuda")
    at = slots - 130
    lead = at % 64                                     # keep the blocks' borders: the last slots, block by block
    at -= lead
    sides = []
    for codes, s in ((prefix[0], prefix[1]), (prefix[2], prefix[3])):
        c, sc = big.clone(), scales.clone()
        c[:, :, at:at + 130] = codes.cuda()
        sc[:, :, at // 64:at // 64 + 3] = s.cuda()
        sides += [c[:, :, at:], sc[:, :, at // 64:]]
    got = kv_shared_attention_cuda(q.cuda(), *sides, _ints([130]), *[x.cuda() for x in own], _ints([b % 40 for b in range(per)]))
    ref, bound = _shared.attend(q, prefix, [130], own, [b % 40 for b in range(per)], None, 64, 32)
    _kv.close(got, ref, bound)


def test_captured_streams_and_runs(gpu):
    q, prefix, own = _shared.case(1, 12, 1, 32, 4, 64, 700, 100)
    q, prefix, own = q.cuda(), [x.cuda() for x in prefix], [x.cuda() for x in own]
    lengths, start = _ints([700]), _ints([0] * 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_shared_attention_cuda(q, *prefix, lengths, *own, start)
    stream = torch.cuda.Stream()
    for i in range(4):
        q.copy_(_kv.rows(q.shape, "fp16", 90 + i))
        lengths.fill_(700 - 173 * i)
        start.copy_(_ints([(7 * b + 9 * i) % 100 for b in range(12)]))
        graph.replay()
        eager = kv_shared_attention_cuda(q, *prefix, lengths, *own, start)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            aside = kv_shared_attention_cuda(q, *prefix, lengths, *own, start)
        torch.cuda.synchronize()
        assert _kv.same(out, eager) and _kv.same(aside, eager)
        ref, bound = _shared.attend(q.cpu(), [x.cpu() for x in prefix], [700 - 173 * i], [x.cpu() for x in own],
                                    start.tolist(), None, 64, 32)
        _kv.close(eager, ref, bound)


@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
def test_two_graphs_of_prompts_and_tokens(gpu, codes, dtype):
    """Prompts and single tokens behind the same prefixes, captured apart and replayed in turn, one in a stream of its own."""
    q, prefix, own = _shared.case(2, 2, 70, 8, 2, 64, 500, 200, codes, dtype)
    token = _kv.rows((4, 1, 8, 64), dtype, 77)
    q, token, prefix, own = q.cuda(), token.cuda(), [x.cuda() for x in prefix], [x.cuda() for x in own]
    lengths, start, counts = _ints([500, 31]), _ints([0, 9, 100, 130]), _ints([70, 33, 0, 70])
    calls = [lambda: kv_shared_attention_cuda(q, *prefix, lengths, *own, start, counts),
             lambda: kv_shared_attention_cuda(token, *prefix, lengths, *own, start)]
    graphs, outs = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    stream = torch.cuda.Stream()
    for i in range(4):
        q.copy_(_kv.rows(q.shape, dtype, 80 + i))
        token.copy_(_kv.rows(token.shape, dtype, 90 + i))
        lengths.copy_(_ints([500 - 150 * i, 31 + 100 * i]))
        start.copy_(_ints([i, 9 * i, 100 - i, 130]))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for out, call in zip(outs, calls):
            assert _kv.same(out, call())
        ref, bound = _shared.attend(q.cpu(), [x.cpu() for x in prefix], lengths.tolist(), [x.cpu() for x in own],
                                    start.tolist(), counts.tolist(), 64, 32)
        _kv.close(outs[0], ref, bound)


def test_prompt_then_answers(gpu):
    """A prompt, forked into answers or shared by them, then their tokens: the run that a sampled batch makes."""
    heads, kv, dim, n, length = 8, 2, 64, 3, 70
    cos, sin = (x.cuda() for x in _kv.tables(256, dim))
    whole, prompt = QuantizedKVCache(n, kv, 256, dim, "int8", 64, "cuda"), QuantizedKVCache(1, kv, 128, dim, "int8", 64, "cuda")
    own = QuantizedKVCache(n, kv, 64, dim, "int8", 64, "cuda")
    rows = lambda b, t, seed: _kv.rows((b, t, heads + 2 * kv, dim), "fp16", seed).cuda().split([heads, kv, kv], dim=2)  # noqa: E731
    prompt.rotary_write(*rows(1, length, 1), cos, sin, _ints([0]))
    whole.fork_from(prompt, _ints([0] * n), _ints([length]))
    held = torch.zeros((n,), dtype=torch.int64, device="cuda")
    for step in range(6):
        q, k, v = rows(n, 1, 10 + step)
        turned = whole.rotary_write(q, k, v, cos, sin, held + length)
        forked = whole.attend(turned, held + length)
        again = own.rotary_write(q, k, v, cos[length:].contiguous(), sin[length:].contiguous(), held)
        assert _kv.same(turned, again)
        shared = own.attend_shared(again, prompt, _ints([length]), held)
        ref, bound = _kv.attend(turned.cpu(), *[x.cpu() for x in whole.tensors()], (held + length).tolist(), None, 64)
        _kv.close(forked, ref, bound)
        ref, bound = _shared.attend(again.cpu(), [x.cpu() for x in prompt.tensors()], [length],
                                    [x.cpu() for x in own.tensors()], held.tolist(), None, 64, 64)
        _kv.close(shared, ref, bound)
        held += 1
        if step == 3:
            order = _ints([2, 0, 0])
            whole.reorder(order, held + length)
            own.reorder(order, held)
            held = held[order]
