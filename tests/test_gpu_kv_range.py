"""Attention over the 8-bit key/value cache at the ends of its range: caches past
32-bit offsets within a head, weights far below a row's largest, scores and
scale factors of any size, prompts of the widest heads in shares."""

import math

import numpy as np
import pytest
import torch

from nibble_amd import kv_attention_cuda, kv_read_cuda, kv_write_cuda
from tests import _kv

pytestmark = pytest.mark.gpu


def _attend(q, cache, starts, counts=None, scale=None):
    at = torch.tensor(starts).cuda()
    limits = None if counts is None else torch.tensor(counts).cuda()
    return kv_attention_cuda(q.cuda(), *(t.cuda() for t in cache), at, limits, scale)


# --------------------------------------------------------------- offsets within a head

@pytest.mark.parametrize("dim,slots", [(256, (1 << 24) + 5), (128, (1 << 25) + 5), (64, (1 << 26) + 5)])
def test_prompt_in_a_head_past_32_bits(gpu, dim, slots):
    """A prompt at the start and one at the end of a head of more than 2^32
    bytes. Slots 0 .. 69 and the last 70 hold numbers, all between score 0 and
    value 0."""
    tokens = 70
    kc, vc = (torch.zeros((2, 1, slots, dim), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((2, 1, -(-slots // 64)), 2.0 ** -6, device="cuda") for _ in range(2))
    last = slots - tokens
    k, v = (_kv.rows((2, tokens, 1, dim), "fp16", i, spread).cuda() for i, spread in ((61, 1.0), (62, 1000.0)))
    kv_write_cuda(k, v, kc, ks, vc, vs, torch.tensor([0, 0]).cuda())
    kv_write_cuda(k, v, kc, ks, vc, vs, torch.tensor([last, last]).cuda())
    q = _kv.rows((2, tokens, 2, dim), "fp16", 63)
    got = kv_attention_cuda(q.cuda(), kc, ks, vc, vs, torch.tensor([0, last]).cuda())

    def held(codes, scales, at):   # the tokens' values, from the block that `at` lies in
        first = at - at % 64
        end = min(first + 192, slots)
        part = kv_read_cuda(codes[:, :, first:end], scales[:, :, first // 64:-(-end // 64)], torch.float32)
        return part[:, 0, at - first:at - first + tokens].double().cpu()

    kk, vv = ([held(c, s, at) for at in (0, last)] for c, s in ((kc, ks), (vc, vs)))
    del kc, vc
    causal = torch.arange(tokens) <= torch.arange(tokens).unsqueeze(1)
    for b in range(2):
        rows = q[b].double().transpose(0, 1)                                    # [heads, tokens, dim]
        near = torch.exp(torch.matmul(rows, kk[b][b].t().contiguous()) / math.sqrt(dim)) * causal
        total = near.sum(-1, keepdim=True)
        out, size = torch.matmul(near, vv[b][b]), torch.matmul(near, vv[b][b].abs())
        if b == 1:   # the slots at the start, seen whole, and those of weight 1 between
            far = torch.exp(torch.matmul(rows, kk[0][1].t().contiguous()) / math.sqrt(dim))
            total = total + far.sum(-1, keepdim=True) + (last - tokens)
            out, size = out + torch.matmul(far, vv[0][1]), size + torch.matmul(far, vv[0][1].abs())
        want, size = (out / total).transpose(0, 1), (size / total).transpose(0, 1)
        # weights off by 2^-11 of themselves, scores by 2^-12 (fp32 sums of dim products of up to 2^6); a lane adds
        # up the weights of 2^20 slots at most, 16 at a time: 2^16 additions, each off by 2^-24 of the sum so far,
        # which is half of the whole on average: 2^-9
        _kv.close(got[b], want.numpy(), (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -9) * size.numpy(), f"sequence {b}")


# ----------------------------------------------------- weights far below the largest one

@pytest.mark.parametrize("gap", [10.0, 16.0, 17.5, 19.0])
@pytest.mark.parametrize("codes,dim", [("int8", 64), ("fp8", 128), ("int8", 256)])
@pytest.mark.parametrize("batch,kv_heads,tokens", [(1, 1, 1), (32, 8, 1), (1, 1, 70), (64, 8, 70)])
def test_weights_behind_a_sink(gpu, batch, kv_heads, tokens, codes, dim, gap):
    """131072 slots, one of score `gap` whose value is zero and the others of
    score 0: the output is made of weights exp(-gap) of the largest. In shares,
    and (many sequences, which read one cache) by a workgroup alone."""
    slots = 131072
    kc, vc = torch.zeros((1, 1, slots, dim), dtype=_kv.CODES[codes]), torch.zeros((1, 1, slots, dim))
    kc[0, 0, 0] = torch.ones(dim).to(kc.dtype)
    vc[0, 0, 1:] = torch.randint(1, 16, (slots - 1, dim), generator=_kv.gen(64)).float()
    ks = torch.ones((1, 1, slots // 64))
    cache = [t.cuda().expand(batch, kv_heads, *t.shape[2:]) for t in (kc, ks, vc.to(kc.dtype), ks)]
    q = torch.full((batch, tokens, 2 * kv_heads, dim), gap / dim ** 0.5).half()   # q.k scale = gap up to q's rounding
    scores = float(q[0, 0, 0, 0]) * dim * dim ** -0.5
    got = _attend(q, cache, [slots - tokens] * batch)
    seen = torch.arange(slots - tokens + 1, slots + 1)                 # slots of each row
    weight = math.exp(-scores)
    sums = torch.cumsum(vc[0, 0].double(), dim=0)[seen - 1]
    want = weight * sums / (1.0 + weight * (seen.double().unsqueeze(1) - 1.0))
    want = want.unsqueeze(1).expand(batch, tokens, 2 * kv_heads, dim).numpy()
    # each weight off by 2^-11 of itself, or by 2^-25 where the largest is at least 2^7: 2^-32 of the largest times
    # the largest value (16); its exponent, up to 28, by 28 2^-24 and two roundings more; the fp32 sums of each
    # lane, at most slots / 32 additions, by 2^-24 each
    bound = ((2.0 ** -11 + 40 * 2.0 ** -24 + slots / 32 * 2.0 ** -24) * want + slots * 2.0 ** -32 * 16
             / (1.0 + weight * (slots - 1)))
    _kv.close(got, want, bound)


# ------------------------------------------------------------------ scores of any size

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("codes,dim", [("int8", 64), ("fp8", 128), ("int8", 256)])
@pytest.mark.parametrize("power", [6, 14, 18, 22, 28])
@pytest.mark.parametrize("tokens", [2, 80])
def test_large_scores(gpu, tokens, power, codes, dim, dtype):
    """Scores of 2^18 to 2^40: a softmax that is one-hot wherever two scores
    differ by more than their fp32 sums can be off."""
    slots, block = 300, 16
    q = (_kv.rows((1, tokens, 4, dim), "fp32", 65) * 1000).to(_kv.TYPES[dtype])
    kc, ks = _kv.cache(1, 2, slots, dim, codes, block, 66)
    vc, vs = _kv.cache(1, 2, slots, dim, codes, block, 67)
    ks *= 2.0 ** power
    got = _kv.numbers(_attend(q, (kc, ks, vc, vs), [slots - tokens]))[0]
    assert np.isfinite(got).all()
    keys, values = _kv.values(kc, ks, block)[0], _kv.values(vc, vs, block)[0]
    rows = _kv.numbers(q)[0]
    checked = 0
    for t in range(tokens):
        for h in range(4):
            kk, vv = keys[h // 2, :slots - tokens + t + 1], values[h // 2, :slots - tokens + t + 1]
            s = kk @ rows[t, h] * dim ** -0.5
            slip = (dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(rows[t, h])).max() * dim ** -0.5
            best = int(np.argmax(s))
            assert (np.abs(got[t, h]) <= np.abs(vv).max(axis=0) * (1 + 2.0 ** -8)).all()
            if s[best] - np.delete(s, best).max() > 2 * slip + 40:   # the rest weighs less than 300 e^-40
                half = _kv.HALF_STEP[q.dtype]
                # the one weight cancels up to the fp16 rounding of both
                assert (np.abs(got[t, h] - vv[best]) <= (2.0 ** -11 + half * 1.01) * np.abs(vv[best]) + 1e-7).all()
                checked += 1
    assert checked > 2 * tokens


@pytest.mark.parametrize("codes,dim,heads,kv_heads", [("int8", 64, 4, 1), ("fp8", 128, 4, 2), ("int8", 128, 32, 8),
                                                      ("fp8", 256, 2, 1)])
@pytest.mark.parametrize("slots", [700, 2500])
def test_large_scores_of_ragged_prompts(gpu, slots, codes, dim, heads, kv_heads):
    """Large and ordinary scores side by side, in shares of the slots and in
    groups of wavefronts: padding rows, rows outside the cache, sequences of one
    share and of several."""
    tokens, block = 90, 32
    starts, counts = [slots - 80, 3, 0, -4, slots // 2], [tokens, 41, 0, tokens, tokens]
    q = _kv.rows((5, tokens, heads, dim), "bf16", 77)
    q[:, ::3] *= 2.0 ** 30
    kc, ks = _kv.cache(5, kv_heads, slots, dim, codes, block, 78)
    vc, vs = _kv.cache(5, kv_heads, slots, dim, codes, block, 79)
    want, bound = _kv.attend(q, kc, ks, vc, vs, starts, counts, block)
    got = _attend(q, (kc, ks, vc, vs), starts, counts)
    large = torch.zeros(q.shape, dtype=torch.bool)
    large[:, ::3] = True
    keep = ~large.numpy()
    assert np.array_equal(np.isnan(_kv.numbers(got)), np.isnan(want))
    _kv.close(got.cpu().masked_fill(large, 0.0), np.where(keep, want, 0.0), np.where(keep, bound, 0.0))
    # large scores: the first by far takes all
    group, checked = heads // kv_heads, 0
    keys, values, rows, out = _kv.values(kc, ks, block), _kv.values(vc, vs, block), _kv.numbers(q), _kv.numbers(got)
    for b, (start, count) in enumerate(zip(starts, counts)):
        for t in range(0, tokens, 3):
            if t >= count:
                assert (out[b, t] == 0).all()
            elif 0 <= start + t < slots:
                for h in range(heads):
                    kk, vv = keys[b, h // group, :start + t + 1], values[b, h // group, :start + t + 1]
                    s = kk @ rows[b, t, h] * dim ** -0.5
                    slip = (dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(rows[b, t, h])).max() * dim ** -0.5
                    first, *rest = np.sort(s)[::-1][:2]
                    if not rest or first - rest[0] > 2 * slip + 40:
                        best = vv[int(np.argmax(s))]
                        assert (np.abs(out[b, t, h] - best) <= (2.0 ** -11 + 1.01 * 2.0 ** -8) * np.abs(best) + 1e-7).all()
                        checked += 1
    assert checked > 50


@pytest.mark.parametrize("scale", [1e-30, -1e-30, 1e-38])
@pytest.mark.parametrize("tokens", [2, 80])
def test_tiny_scale(gpu, tokens, scale):
    """The largest codes and queries under a factor that makes all scores 0 to
    fp32: every weight is the same."""
    dim, slots = 256, 160
    kc = torch.full((1, 1, slots, dim), 448.0)
    kc[:, :, 1::2] = -448.0
    kc = kc.to(torch.float8_e4m3fn)
    vc = torch.sign(kc.float()).to(torch.float8_e4m3fn)
    ks, vs = torch.full((1, 1, 10), 2.0 ** 40), torch.ones((1, 1, 10))
    q = torch.full((1, tokens, 1, dim), 65504.0).half()
    got = _attend(q, (kc, ks, vc, vs), [slots - tokens], scale=scale)
    seen = np.arange(slots - tokens + 1, slots + 1)
    want = np.broadcast_to((seen % 2 / seen)[:, None, None], (tokens, 1, dim))   # +1 and -1 in turn
    # weights off by 2^-11, and by ln 2 times the exponents' 2^-13.2 where the factor is raised
    _kv.close(got[0], want, 2.0 ** -11 + 2.0 ** -13)


# --------------------------------------------------------- the widest heads, in shares

@pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16")])
@pytest.mark.parametrize("tokens,starts,counts", [(70, [1900, 3, 0], [70, 41, 0]), (150, [1500, 1990, -7], None)])
def test_prompt_of_256_dims_in_shares(gpu, tokens, starts, counts, codes, dtype):
    """Prompts behind held tokens in a cache of 2100 slots: the slots are
    divided, sequences of one share and of several, padding, rows outside."""
    q = _kv.rows((3, tokens, 2, 256), dtype, 68)
    cache = (*_kv.cache(3, 1, 2100, 256, codes, 32, 69), *_kv.cache(3, 1, 2100, 256, codes, 32, 70))
    want, bound = _kv.attend(q, *cache, starts, counts, 32)
    _kv.close(_attend(q, cache, starts, counts), want, bound)
