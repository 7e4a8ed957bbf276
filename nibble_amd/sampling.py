"""Drawing tokens from rows of logits by temperature, top-k, top-p and min-p, from
given uniform numbers: the same numbers give the same tokens."""

from __future__ import annotations

import math

import torch

from nibble_amd.cuda import sample_cuda

ONE = 2.0 ** 44      # the largest logit's weight as a whole number
MOST_LOGITS = 2 ** 19


def _per_row(value, rows: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    """[rows, 1] in 64 bits."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"{name} must have dtype {dtype}")
        if value.shape != (rows,):
            raise ValueError(f"{name} must have shape [rows]")
        if value.requires_grad:
            raise ValueError(f"{name} must not require grad")
        return value.to(torch.int64 if dtype == torch.int64 else torch.float64).unsqueeze(1)
    return torch.full((rows, 1), value, dtype=torch.int64 if dtype == torch.int64 else torch.float64)


def sample_reference(logits, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``sample_cuda`` in torch operations on the CPU, with its whole weights."""
    if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("logits must have dtype torch.float16, torch.bfloat16 or torch.float32")
    if logits.dim() != 2:
        raise ValueError("logits must have shape [rows, vocabulary]")
    if logits.requires_grad:
        raise ValueError("logits must not require grad")
    rows, n = logits.shape
    if not 1 <= n <= MOST_LOGITS:
        raise ValueError("a row must have 1 to 524288 logits")
    for name, value, lowest, highest in (("temperature", temperature, 0.0, math.inf), ("top_k", top_k, 0, math.inf),
                                         ("top_p", top_p, 0.0, 1.0), ("min_p", min_p, 0.0, 1.0)):
        if not isinstance(value, torch.Tensor) and not lowest <= value <= highest:
            raise ValueError(f"{name} must be at least {lowest}" + (f" and at most {highest}" if highest == 1.0 else ""))
    u = _per_row(random, rows, torch.float32, "random")
    heat, mass, least = (_per_row(v, rows, torch.float32, name)
                         for v, name in ((temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")))
    count = _per_row(top_k, rows, torch.int64, "top_k")
    x = logits.double()
    number = torch.where(torch.isnan(x), -math.inf, x)
    top = number.amax(dim=1, keepdim=True)
    greedy = torch.isnan(x).any(dim=1, keepdim=True) | ~(heat > 0) | (top == -math.inf) | (count == 1)
    best = torch.where(torch.isnan(x), math.inf, torch.where(torch.isnan(x).any(dim=1, keepdim=True), -math.inf, x))
    power = (number - top) * (math.log2(math.e) / torch.where(heat > 0, heat, 1.0))
    w = torch.where(power > -46, torch.exp2(power), 0.0)            # NaN (of infinities) as 0
    w = torch.where(number == top, 1.0, w)
    w = torch.where(number == -math.inf, 0.0, w)
    whole = torch.round(w * ONE).to(torch.int64)
    order = torch.argsort(number, dim=1, descending=True, stable=True)
    kept = whole.gather(1, order)
    rank = torch.arange(n).unsqueeze(0)
    kept = kept.masked_fill((count > 0) & (rank >= count), 0)
    total = kept.sum(dim=1, keepdim=True).double()
    before = kept.cumsum(dim=1) - kept
    needed = torch.ceil(mass.clamp(0, 1) * total).clamp(min=1).nan_to_num(math.inf)
    kept = kept.masked_fill((mass < 1) & (before.double() >= needed), 0)
    kept = kept.masked_fill((least > 0) & (w.gather(1, order) < least.clamp(max=1)), 0)
    sums = torch.zeros_like(kept).scatter_(1, order, kept).cumsum(dim=1)
    total = sums[:, -1:]
    target = (u.nan_to_num(0.0).clamp(0, 1) * total.double()).to(torch.int64).clamp(max=total - 1)
    token = torch.where(greedy, best.argmax(dim=1, keepdim=True), (sums > target).to(torch.int8).argmax(dim=1, keepdim=True))
    return token.squeeze(1)


def sample(
    logits: torch.Tensor,
    random: torch.Tensor,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> torch.Tensor:
    """``sample_cuda`` for GPU tensors; the same in torch operations on the CPU."""
    call = sample_cuda if logits.is_cuda else sample_reference
    return call(logits, random, temperature, top_k, top_p, min_p)
