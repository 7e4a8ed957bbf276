"""64-bit oracle of the 8-bit key/value cache's operators (test infrastructure;
plain loops over blocks and sequences, numpy) and input generators."""

from __future__ import annotations

import math

import numpy as np
import torch

CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def numbers(x: torch.Tensor) -> np.ndarray:
    return x.detach().cpu().to(torch.float32).numpy().astype(np.float64)


def nearest(x: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    """Scaled values to the nearest that a code stands for, ties to even, saturated."""
    if dtype == torch.int8:
        return np.clip(np.rint(x), -127, 127)
    x = np.clip(x, -448, 448)
    exponent = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    step = 2.0 ** (exponent - 3)
    return np.rint(x / step) * step


def scale(amax: float, dtype: torch.dtype) -> float:
    e = -40
    while e < 40 and amax > LARGEST[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, start, counts, block: int):
    """(codes as numbers, scales) after the tokens x [b, t, heads, dim] were written."""
    c, s = numbers(codes), numbers(scales)
    rows = numbers(x)
    rows = np.where(np.isnan(rows), 0.0, rows)
    top = torch.finfo(x.dtype).max
    slots = c.shape[2]
    for b in range(x.shape[0]):
        count = x.shape[1] if counts is None else min(max(int(counts[b]), 0), x.shape[1])
        for h in range(x.shape[2]):
            lo, hi = max(int(start[b]), 0), min(int(start[b]) + count, slots)
            while lo < hi:
                j = lo // block
                end = min((j + 1) * block, hi)
                new = rows[b, lo - int(start[b]):end - int(start[b]), h]
                sc = scale(min(np.abs(new).max(), top), codes.dtype)
                if lo > j * block:
                    was = s[b, h, j]
                    if sc > was:
                        c[b, h, j * block:lo] = nearest(c[b, h, j * block:lo] * (was / sc), codes.dtype)
                    sc = max(sc, was)
                s[b, h, j] = sc
                c[b, h, lo:end] = nearest(new / sc, codes.dtype)
                lo = end
    return c, s


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, interleaved: bool):
    """(rotated rows, |x1 c| + |x2 s| of each value) of x [b, t, heads, dim], positions [b, t]."""
    y, c, s = numbers(x), numbers(cos), numbers(sin)
    half = c.shape[1]
    one = np.arange(half) * 2 if interleaved else np.arange(half)
    two = one + 1 if interleaved else one + half
    size = np.abs(y)
    out = y.copy()
    for b in range(y.shape[0]):
        for t in range(y.shape[1]):
            p = int(positions[b, t])
            cc, ss = (c[p], s[p]) if 0 <= p < c.shape[0] else (np.full(half, np.nan), np.full(half, np.nan))
            x1, x2 = y[b, t][:, one], y[b, t][:, two]
            out[b, t][:, one], out[b, t][:, two] = x1 * cc - x2 * ss, x2 * cc + x1 * ss
            size[b, t][:, one] = np.abs(x1 * cc) + np.abs(x2 * ss)
            size[b, t][:, two] = np.abs(x2 * cc) + np.abs(x1 * ss)
    return out, size


def values(codes: torch.Tensor, scales: torch.Tensor, block: int) -> np.ndarray:
    return numbers(codes) * np.repeat(numbers(scales), block, axis=2)[:, :, :codes.shape[2], None]


def attend(q, k_codes, k_scales, v_codes, v_scales, start, counts, block, scale=None):
    """(outputs, bound of the kernel's error before its last rounding), both
    [b, t, heads, dim].

    The bound: the weights enter the second product as fp16, each off by half a
    step, 2^-11 of itself (of sum w |v|), or 2^-25 of the largest below fp16's
    normal range: n 2^-25 of the largest |v| scale times the largest code,
    which is at most twice max |v| for the values that a scale fits (256 times
    for a block of small codes; the bound takes the scales). A score's fp32 sum
    of dim products is off by at most (dim + 4) 2^-24 sum |q k| scale, and
    exp2 of it by that much and 2^-22 more; twice, as the sum of the weights
    moves as well."""
    x = numbers(q)
    batch, tokens, heads, dim = x.shape
    group = heads // k_codes.shape[1]
    slots = k_codes.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, bound = np.zeros_like(x), np.zeros_like(x)
    for b in range(batch):
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        first = int(start[b])
        end = min(max(first + count, 0), slots)
        pick = lambda c, s: values(c[b:b + 1, :, :end], s[b:b + 1, :, :-(-end // block)], block)[0]  # noqa: E731
        k, v = (pick(k_codes, k_scales), pick(v_codes, v_scales)) if end else (None, None)
        tops = np.repeat(numbers(v_scales)[b], block, axis=1)[:, :end] * LARGEST[v_codes.dtype]
        for t in range(count):
            p = first + t
            if not 0 <= p < slots:
                out[b, t] = np.nan
                continue
            for h in range(heads):
                kk, vv = k[h // group, :p + 1], v[h // group, :p + 1]
                s = kk @ x[b, t, h] * scale
                slip = (dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(x[b, t, h])).max() * abs(scale) + 2.0 ** -22
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, t, h] = w @ vv
                # a weight is lost against the largest weight times its value's scale
                reach = (w * tops[h // group, :p + 1]).max()
                bound[b, t, h] = ((2.0 ** -11 + 2 * slip) * (w @ np.abs(vv))
                                  + min((p + 1) * 2.0 ** -25, 1.0) * reach)
    return out, bound


def close(got: torch.Tensor, ref: np.ndarray, bound, what: str = "") -> None:
    """|got - ref| <= bound + half a step of the output's type (at least that of its smallest normal number)."""
    x = numbers(got)
    assert x.shape == ref.shape, (x.shape, ref.shape)
    assert np.array_equal(np.isnan(x), np.isnan(ref)), f"{what}: NaN in other places"
    half = HALF_STEP[got.dtype]
    allowed = bound * (1 + 2 * half) + half * np.maximum(np.abs(ref), torch.finfo(got.dtype).tiny)
    bad = np.abs(x - ref) > allowed
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; first {i}: {x[i]} against {ref[i]} "
                             f"+- {allowed[i] if np.ndim(allowed) else allowed}")


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def rows(shape, dtype: str, seed: int, spread: float = 1.0) -> torch.Tensor:
    """Normal values, channels of different sizes, on the CPU."""
    g = gen(seed)
    channels = torch.exp(0.5 * torch.randn((shape[-1],), generator=g)) * spread
    return (torch.randn(shape, generator=g) * channels).to(TYPES[dtype])


def cache(batch, heads, slots, dim, codes: str, block: int, seed: int, spread: float = 1.0):
    """(codes, scales) of normal values, quantized block by block, on the CPU."""
    blocks = -(-slots // block)
    x = rows((batch, heads, slots, dim), "fp32", seed, spread)
    c = torch.zeros((batch, heads, slots, dim), dtype=CODES[codes])
    s = torch.full((batch, heads, blocks), 2.0 ** -40)
    for j in range(blocks):
        part = x[:, :, j * block:(j + 1) * block]
        e = torch.ceil(torch.log2(part.abs().amax(dim=(2, 3)) / LARGEST[CODES[codes]]))
        s[:, :, j] = torch.exp2(e)
        scaled = part / s[:, :, j, None, None]
        c[:, :, j * block:(j + 1) * block] = (torch.round(scaled) if codes == "int8" else scaled).to(CODES[codes])
    return c, s


def tables(slots: int, rot: int, theta: float = 10000.0):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angles = torch.outer(torch.arange(slots, dtype=torch.float64), inv)
    return angles.cos().float(), angles.sin().float()


def bits(x: torch.Tensor) -> torch.Tensor:
    return x.detach().cpu().contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and torch.equal(bits(a), bits(b))


assert math.isclose(HALF_STEP[torch.float16], torch.finfo(torch.float16).eps / 2)
