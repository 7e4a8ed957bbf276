"""The 8-bit key/value cache's operators in plain torch: the path of CPU
tensors, and what the HIP kernels compute (``include/w4a16_kv.h``)."""

from __future__ import annotations

import math

import torch

LOWEST, HIGHEST = -40, 40   # exponents of the scales


def _largest(codes: torch.Tensor) -> float:
    return 127.0 if codes.dtype == torch.int8 else 448.0


def block_size(slots: int, blocks: int) -> int:
    """Slots of a scale: the one of 16, 32, 64 and 128 of which ``blocks`` cover ``slots``."""
    for block in (16, 32, 64, 128):
        if -(-slots // block) == blocks:
            return block
    raise ValueError("scales must hold one scale for every 16, 32, 64 or 128 slots")


def scale_of(amax: torch.Tensor, largest: float) -> torch.Tensor:
    """2^e, e the smallest integer in [LOWEST, HIGHEST] with amax <= largest 2^e."""
    amax = amax.float().clamp(max=torch.finfo(torch.float32).max)   # frexp gives infinities no exponent
    mantissa, e = torch.frexp(amax)
    top, shift = math.frexp(largest)
    e = torch.where(amax == 0, LOWEST, e - shift + (mantissa > top).to(e.dtype)).clamp(LOWEST, HIGHEST)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e)


def encode(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Scaled fp32 values -> codes, half to even, saturated."""
    if dtype == torch.int8:
        return torch.round(x).clamp(-127.0, 127.0).to(torch.int8)
    return x.clamp(-448.0, 448.0).to(dtype)


def rotary_reference(x, positions, cos, sin, interleaved=False):
    if positions.dtype != torch.int64:
        raise TypeError("positions must have dtype torch.int64")
    if x.dim() not in (3, 4):
        raise ValueError("x must have shape [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]")
    if positions.shape not in (x.shape[-3:-2], x.shape[:-2]):
        raise ValueError("positions must have shape [tokens] or [batch, tokens]")
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError("cos and sin must have shape [positions, rotated dims / 2]")
    rot = 2 * cos.shape[1]
    if rot < 2 or rot > x.shape[-1]:
        raise ValueError("the rotated part must be an even number of at most head_dim dims")
    known = (positions >= 0) & (positions < cos.shape[0])
    if cos.shape[0] == 0:
        c = s = torch.full((*positions.shape, 1, rot // 2), float("nan"))
    else:
        at, nan = positions.clamp(0, cos.shape[0] - 1), torch.tensor(float("nan"))
        c, s = (torch.where(known.unsqueeze(-1), table[at], nan).unsqueeze(-2) for table in (cos, sin))
    part = x[..., :rot].float()
    if interleaved:
        x1, x2 = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).flatten(-2)
    else:
        x1, x2 = part.chunk(2, dim=-1)
        turned = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)
    return torch.cat((turned.to(x.dtype), x[..., rot:]), dim=-1)


def _check_lengths(x, batch: int, name: str) -> None:
    if x.dtype != torch.int64:
        raise TypeError(f"{name} must have dtype torch.int64")
    if x.shape != (batch,):
        raise ValueError(f"{name} must have shape [batch]")


def _check_rows(x, name: str, codes, tokens: int, heads: int | None = None) -> None:
    """Rows [batch, tokens, heads, head_dim] that go with a cache's codes, as the GPU ops ask for them."""
    if x.dim() != 4 or x.shape[0] != codes.shape[0] or x.shape[1] != tokens or x.shape[3] != codes.shape[3] or (
            heads is not None and x.shape[2] != heads):
        raise ValueError(f"{name} must have shape [batch, tokens, heads, head_dim] of the cache and of the other rows")
    if x.requires_grad:
        raise ValueError(f"{name} must not require grad")


def _spans(start, counts, batch: int, tokens: int):
    """(first position, tokens that are no padding) of each sequence."""
    _check_lengths(start, batch, "start")
    if counts is not None:
        _check_lengths(counts, batch, "counts")
    begins = [int(p) for p in start]
    if counts is None:
        return [(p, tokens) for p in begins]
    return [(p, min(max(int(c), 0), tokens)) for p, c in zip(begins, counts)]


def _write_side(x, codes, scales, b, start, count):
    slots, block = codes.shape[2], block_size(codes.shape[2], scales.shape[2])
    largest = _largest(codes)
    top = torch.finfo(x.dtype).max   # infinities count as the largest finite value
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=float("inf"), neginf=float("-inf"))
    lo, hi = max(start, 0), min(start + count, slots)
    at = lo
    while at < hi:
        j = at // block
        end = min((j + 1) * block, hi)
        new = x[at - start:end - start].transpose(0, 1)                  # [kv_heads, n, dim]
        amax = new.abs().amax(dim=(1, 2)).clamp(max=top)
        scale = scale_of(amax, largest)
        if at > j * block:
            was = scales[b, :, j].clone()
            scale = torch.maximum(scale, was)
            held = codes[b, :, j * block:at]
            rescaled = encode(held.float() * (was / scale)[:, None, None], codes.dtype)
            codes[b, :, j * block:at] = torch.where((scale > was)[:, None, None], rescaled.float(),
                                                    held.float()).to(codes.dtype)
        scales[b, :, j] = scale
        codes[b, :, at:end] = encode(new / scale[:, None, None], codes.dtype)
        at = end


def kv_write_reference(k, v, k_codes, k_scales, v_codes, v_scales, start, counts=None):
    batch, kv_heads = k_codes.shape[:2]
    for x, name in ((k, "k"), (v, "v")):
        _check_rows(x, name, k_codes, k.shape[1], kv_heads)
    for b, (first, count) in enumerate(_spans(start, counts, batch, k.shape[1])):
        _write_side(k[b], k_codes, k_scales, b, first, count)
        _write_side(v[b], v_codes, v_scales, b, first, count)


def rotary_kv_write_reference(q, k, v, cos, sin, k_codes, k_scales, v_codes, v_scales, start, counts=None,
                              interleaved=False):
    tokens, (batch, kv_heads, slots) = q.shape[1], k_codes.shape[:3]
    for x, name, heads in ((q, "q", None), (k, "k", kv_heads), (v, "v", kv_heads)):
        _check_rows(x, name, k_codes, tokens, heads)
    _spans(start, counts, batch, tokens)
    if cos.shape[0] < slots:
        raise ValueError("the rotary tables must have a row for every slot")
    positions = start.unsqueeze(1) + torch.arange(tokens)
    outside = torch.full_like(positions, -1)
    positions = torch.where(positions < slots, positions, outside)
    turned = rotary_reference(q, positions, cos, sin, interleaved)
    if counts is not None:
        turned[torch.arange(tokens) >= counts.unsqueeze(1)] = 0
    kv_write_reference(rotary_reference(k, positions, cos, sin, interleaved), v, k_codes, k_scales, v_codes, v_scales,
                       start, counts)
    return turned


def kv_read_reference(codes, scales, dtype=torch.float16):
    slots = codes.shape[2]
    per_slot = scales.repeat_interleave(block_size(slots, scales.shape[2]), dim=2)[:, :, :slots].unsqueeze(3)
    values = codes.float() * per_slot
    most = torch.finfo(dtype).max
    return values.clamp(-most, most).to(dtype)


def kv_attention_reference(q, k_codes, k_scales, v_codes, v_scales, start, counts=None, scale=None):
    _check_rows(q, "q", k_codes, q.shape[1])
    batch, tokens, heads, dim = q.shape
    kv_heads, slots = k_codes.shape[1], k_codes.shape[2]
    if heads == 0 or heads % kv_heads != 0:
        raise ValueError("heads must be a positive multiple of the cache's KV heads")
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    if not math.isfinite(scale):
        raise ValueError("scale must be a finite number")
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    for b, (first, count) in enumerate(_spans(start, counts, batch, tokens)):
        end = min(max(first + count, 0), slots)
        k, v = (kv_read_reference(c[b:b + 1], s[b:b + 1], torch.float32)[0, :, :end].repeat_interleave(group, dim=0)
                for c, s in ((k_codes, k_scales), (v_codes, v_scales)))
        position = first + torch.arange(count)
        scores = torch.matmul(q[b, :count].float().transpose(0, 1), k.transpose(1, 2)) * scale
        scores = scores.masked_fill(torch.arange(end) > position.unsqueeze(1), float("-inf"))
        row = torch.matmul(torch.softmax(scores, dim=-1), v).transpose(0, 1)
        inside = (position >= 0) & (position < slots)
        row[~inside] = float("nan")
        out[b, :count] = row.to(q.dtype)
    return out
