"""Sampling on the GPU against the 64-bit oracle of tests/_sample.py."""

import math

import pytest
import torch

from nibble_amd import sample_cuda
from nibble_amd.sampling import sample_reference
from tests import _sample

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _run(logits, random, **settings):
    on = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v  # noqa: E731
    return sample_cuda(on(logits), on(random), **{n: on(v) for n, v in settings.items()})


def _check(logits, random, **settings):
    got = _run(logits, random, **settings)
    _sample.check(got, logits, random, **settings)
    return got


def test_refusals(gpu):
    logits, random = torch.zeros((2, 5), device="cuda"), torch.zeros(2, device="cuda")
    for message, call in [
            ("torch.float16, torch.bfloat16 or torch.float32", lambda: sample_cuda(logits.double(), random)),
            ("shape \\[rows, vocabulary\\]", lambda: sample_cuda(logits[0], random)),
            ("contiguous in their last", lambda: sample_cuda(logits.t().contiguous().t(), random)),
            ("must not require grad", lambda: sample_cuda(logits.clone().requires_grad_(), random)),
            ("random must be contiguous", lambda: sample_cuda(logits, random[:1])),
            ("random must have dtype", lambda: sample_cuda(logits, random.double())),
            ("same CUDA device", lambda: sample_cuda(logits, random.cpu())),
            ("top_k must have dtype torch.int64", lambda: sample_cuda(logits, random, top_k=random)),
            ("min_p must have dtype torch.float32", lambda: sample_cuda(logits, random, min_p=random.half())),
            ("top_p must be contiguous with shape", lambda: sample_cuda(logits, random, top_p=torch.zeros(3, device="cuda"))),
            ("temperature must not be negative", lambda: sample_cuda(logits, random, temperature=-0.5)),
            ("top_k must not be negative", lambda: sample_cuda(logits, random, top_k=-1)),
            ("top_p must be between", lambda: sample_cuda(logits, random, top_p=1.01)),
            ("min_p must be between", lambda: sample_cuda(logits, random, min_p=float("nan"))),
            ("at least one logit", lambda: sample_cuda(logits[:, :0], random)),
            ("at most 524288", lambda: sample_cuda(torch.zeros((1, (1 << 19) + 1), device="cuda"), random[:1]))]:
        with pytest.raises(RuntimeError, match=message):
            call()
    assert sample_cuda(logits[:0], random[:0]).shape == (0,)


@pytest.mark.parametrize("row,settings", _sample.EDGES)
@pytest.mark.parametrize("dtype", TYPES)
def test_edges(gpu, row, settings, dtype):
    random = torch.tensor(_sample.EDGE_NUMBERS)
    _check(torch.tensor([row], dtype=dtype).expand(len(random), -1).contiguous(), random, **settings)


SETTINGS = [{}, {"top_k": 1}, {"top_k": 5}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.6, "top_k": 40},
            {"temperature": 0.7, "top_k": 50, "top_p": 0.95}, {"temperature": 3.0, "top_k": 600, "top_p": 0.9},
            {"temperature": 1.4, "top_k": 300, "top_p": 0.8, "min_p": 0.01}, {"temperature": 0.05, "top_p": 0.5},
            {"temperature": 8.0, "top_p": 0.97}]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("n", [2, 63, 1000, 8191, 8193, 32000, 50257])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(gpu, dtype, n, settings):
    _check(_sample.logits(5, n, dtype, n), _sample.numbers(5, n + 1), **settings)


@pytest.mark.parametrize("n", [131072, 262147, 1 << 19])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_vocabularies(gpu, dtype, n):
    for settings in ({}, {"top_k": 1000, "top_p": 0.7}, {"top_p": 0.99}, {"top_k": 100000}):
        _check(_sample.logits(2, n, dtype, 7), _sample.numbers(2, 8), **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_flat_rows(gpu, dtype):
    """Equal logits, and ones of a few values: limits that fall among ties."""
    n = 40000
    for values in (1, 2, 5):
        logits = torch.randint(values, (6, n), generator=torch.Generator().manual_seed(values)).to(dtype)
        for settings in ({}, {"top_k": 777}, {"top_k": 30000, "top_p": 0.33}, {"top_p": 0.61}, {"min_p": 0.2, "top_k": 9000}):
            _check(logits, _sample.numbers(6, values), **settings)
    # sums of equal weights are exact: token floor(u n)
    n = 32768
    random = torch.tensor([0.0, 0.25, 0.5, 0.75, 4095 / 4096, 1 - 2.0 ** -24])
    got = _run(torch.full((6, n), 2.5, dtype=dtype), random)
    assert got.tolist() == [int(u * n) for u in random.tolist()]


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(gpu, dtype):
    logits = _sample.logits(8, 12345, dtype, 11)
    masked = torch.rand(logits.shape, generator=torch.Generator().manual_seed(12)) < 0.95
    masked[3] = True
    masked[3, 12344] = False
    masked[4] = True                      # nothing is left: token 0
    logits = logits.masked_fill(masked, float("-inf"))
    lowest = logits.masked_fill(masked, torch.finfo(dtype).min)
    for settings in ({}, {"top_k": 1000}, {"top_p": 0.9, "top_k": 50}, {"temperature": 2.0, "min_p": 0.02}):
        got = _check(logits, _sample.numbers(8, 13), **settings)
        assert got[3] == 12344 and got[4] == 0
        _check(lowest, _sample.numbers(8, 13), **settings)


def test_settings_of_rows(gpu):
    logits, random = _sample.logits(6, 5000, torch.float32, 3), _sample.numbers(6, 4)
    settings = {"temperature": torch.tensor([1.0, 0.0, 0.5, -1.0, 2.0, float("nan")]),
                "top_k": torch.tensor([0, 3, -7, 5, 1, 9000]), "top_p": torch.tensor([0.5, 1.0, 2.0, float("nan"), -1.0, 0.9]),
                "min_p": torch.tensor([0.0, -1.0, 0.3, 5.0, float("nan"), 0.1])}
    _check(logits, random, **settings)
    for name, value in settings.items():
        _check(logits, random, **{"temperature": 0.9, "top_p": 0.9, name: value})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 0), (5, 3)])
def test_layouts(gpu, dtype, pad, offset):
    """Rows that start at any element, views of wider rows, one row for all."""
    wide = _sample.logits(4, 7001 + pad, dtype, 21)
    flat = torch.cat((torch.full((offset,), 90.0, dtype=dtype), wide.flatten(), torch.full((64,), 90.0, dtype=dtype))).cuda()
    view = flat[offset:offset + wide.numel()].view(wide.shape)[:, :7001]
    random = _sample.numbers(4, 22).cuda()
    got = sample_cuda(view, random, top_k=30, top_p=0.9)
    _sample.check(got, view, random, top_k=30, top_p=0.9)
    one = view[2:3].expand(4, -1)
    _sample.check(sample_cuda(one, random), one, random)


def test_tokens_come_as_often_as_they_are_likely(gpu):
    """Of N numbers spread evenly a token takes its probability times N, by one more or less."""
    logits = _sample.logits(1, 300, torch.float32, 5)
    count = 8192
    random = (torch.arange(count) + 0.5) / count
    got = torch.bincount(sample_cuda(logits.cuda().expand(count, -1), random.cuda(), temperature=0.8).cpu(), minlength=300)
    share = torch.softmax(logits[0].double() / 0.8, dim=0)
    assert ((got - count * share).abs() <= 1 + 1e-6).all()


def test_agrees_with_the_torch_form(gpu):
    logits, random = _sample.logits(40, 3001, torch.float16, 31), _sample.numbers(40, 32)
    for settings in SETTINGS:
        assert torch.equal(_run(logits, random, **settings).cpu(), sample_reference(logits, random, **settings))


def test_captured_and_streams(gpu):
    """A replayed call reads new logits and numbers; a call on a side stream; runs agree."""
    logits, random = _sample.logits(3, 32000, torch.float16, 41).cuda(), _sample.numbers(3, 42).cuda()
    settings = {"temperature": 0.8, "top_k": 64, "top_p": 0.9}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = sample_cuda(logits, random, **settings)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, sample_cuda(logits, random, **settings))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_cuda(logits, random, **settings)
    for seed in range(4):
        logits.copy_(_sample.logits(3, 32000, torch.float16, 50 + seed))
        random.copy_(_sample.numbers(3, 60 + seed))
        graph.replay()
        eager = sample_cuda(logits, random, **settings)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        _sample.check(out, logits, random, **settings)


def test_compiled(gpu):
    def draw(x, u):
        return torch.ops.w4a16.sample(x * 2, u, 0.9, 20)

    logits, random = _sample.logits(2, 999, torch.float16, 71).cuda(), _sample.numbers(2, 72).cuda()
    got = torch.compile(draw, backend="aot_eager", fullgraph=True)(logits, random)
    assert torch.equal(got, draw(logits, random))


@pytest.mark.parametrize("settings", [{}, {"top_k": 400}, {"top_p": 0.9}, {"top_p": 0.5, "top_k": 3000}, {"min_p": 0.3},
                                      {"temperature": 1e-6, "top_p": 0.9}, {"temperature": 30.0, "top_p": 0.99}])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_near_zero(gpu, dtype, settings):
    """Logits around 0 and below 2^-20: few and many, zeros, of both signs, as the largest and among larger ones."""
    g = torch.Generator().manual_seed(3)
    n = 9000
    rows = []
    for share, spread, shift in [(0.001, 1.0, 0.0), (0.001, 1e-3, 0.0), (0.5, 1.0, 0.0), (1.0, 1.0, 0.0), (0.004, 2.0, -5.0),
                                 (0.02, 0.5, -1.5)]:
        row = spread * torch.randn(n, generator=g) + shift
        tiny = torch.rand(n, generator=g) < share
        rows.append(torch.where(tiny, torch.randn(n, generator=g) * 2.0 ** -22, row))
        rows[-1][torch.rand(n, generator=g) < 0.01] = 0.0
        rows[-1][torch.rand(n, generator=g) < 0.01] = -0.0
    _check(torch.stack(rows).to(dtype), _sample.numbers(len(rows), 4), **settings)


@pytest.mark.parametrize("settings", [{}, {"top_p": 0.97}, {"top_k": 2500}])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", TYPES)
def test_min_p_between_zero_and_small_values(gpu, dtype, sign, settings):
    """Logits of 0 beside a bound that is nearer to 0 than 2^-20: kept below it (sign -1), not above."""
    n = 3000
    logits = torch.full((6, n), -1.0)
    logits[:, ::7] = 0.0
    logits[:, 700] = -0.0
    logits[:, 1500] = 2.0 ** -18          # the largest: 0 weighs e^-3.8
    temperature = 1e-6
    min_p = math.exp(-(2.0 ** -18 - sign * 2.0 ** -22) / temperature)
    _check(logits.to(dtype), _sample.numbers(6, 5), temperature=temperature, min_p=min_p, **settings)


@pytest.mark.parametrize("min_p", [0.7, 0.1, 0.02, 0.004, 1e-4])
@pytest.mark.parametrize("top_p", [0.3, 0.8, 0.97, 0.9995])
@pytest.mark.parametrize("top_k", [0, 250, 9000])
@pytest.mark.parametrize("dtype", TYPES)
def test_min_p_beside_top_p(gpu, dtype, top_k, top_p, min_p):
    """Either of them the narrower one, by much and by little."""
    _check(_sample.logits(4, 20011, dtype, 91), _sample.numbers(4, 92), top_k=top_k, top_p=top_p, min_p=min_p,
           temperature=torch.tensor([0.5, 1.0, 1.6, 1e-3]))


@pytest.mark.parametrize("falling", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_sorted_rows(gpu, dtype, falling):
    """Likely tokens side by side, as where vocabularies are in the order of frequency."""
    logits = _sample.logits(6, 50257, dtype, 61).float().sort(dim=1, descending=falling).values.to(dtype)
    for settings in ({}, {"top_k": 600, "top_p": 0.9}, {"top_k": 2500}, {"top_k": 2600}, {"top_k": 30000, "top_p": 0.99},
                     {"top_p": 0.7}, {"top_p": 0.99}, {"top_p": 0.9999}, {"min_p": 0.001}):
        _check(logits, _sample.numbers(6, 62), **settings)
