"""Rotary position tables: frequencies of a model's rotary embedding, also
scaled for contexts longer than the model was trained on, and the cos / sin
tables that ``rotary`` and the decoder read.

``scaling`` is the dict that Hugging Face configs call ``rope_scaling``
(``{"rope_type": ..., ...}``, or the older key ``"type"``):

* ``default``: the frequencies as they are, theta^(-2i / dims);
* ``linear``: every frequency divided by ``factor``;
* ``dynamic``: a larger theta for tables longer than
  ``original_max_position_embeddings`` (NTK-aware scaling for the tables'
  whole length);
* ``llama3``: wavelengths above ``original / low_freq_factor`` divided by
  ``factor``, those below ``original / high_freq_factor`` kept, a linear blend
  of both frequencies between;
* ``yarn``: the same two ends by the rotations that a dimension completes
  within the original context (``beta_fast`` 32, ``beta_slow`` 1), and the
  tables multiplied by ``attention_factor`` (0.1 ln(factor) + 1).
"""

from __future__ import annotations

import math

import torch

from nibble_amd.cuda import rotary_cuda
from nibble_amd.kv_reference import rotary_reference


def _number(scaling: dict, key: str) -> float:
    value = scaling.get(key)
    if not isinstance(value, (int, float)) or isinstance(value, bool) or value <= 0:
        raise ValueError(f"rope scaling needs a positive {key}")
    return float(value)


def rope_frequencies(
    dims: int,
    theta: float = 10000.0,
    scaling: dict | None = None,
    length: int | None = None,
) -> tuple[torch.Tensor, float]:
    """Frequencies float64 [dims / 2] (radians per position) and the factor of
    the tables. ``dims``: the rotated dims of a head; ``length``: positions of
    the tables (``dynamic`` scaling depends on it)."""
    if dims <= 0 or dims % 2 != 0:
        raise ValueError("dims must be a positive even number")
    if theta <= 0:
        raise ValueError("theta must be greater than zero")
    exponents = torch.arange(0, dims, 2, dtype=torch.float64) / dims
    inv = theta ** -exponents
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return inv, 1.0
    if kind == "linear":
        return inv / _number(scaling, "factor"), 1.0
    if kind == "dynamic":
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        if dims == 2 or length is None or length <= original:
            return inv, 1.0
        grown = theta * (factor * length / original - (factor - 1.0)) ** (dims / (dims - 2))
        return grown ** -exponents, 1.0
    if kind == "llama3":
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        low, high = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
        if high <= low:
            raise ValueError("rope scaling needs high_freq_factor greater than low_freq_factor")
        turns = original * inv / (2.0 * math.pi)               # rotations within the original context
        share = ((turns - low) / (high - low)).clamp(0.0, 1.0)   # of the unscaled frequency
        return inv * share + inv / factor * (1.0 - share), 1.0
    if kind == "yarn":
        if scaling.get("mscale") or scaling.get("mscale_all_dim") or scaling.get("truncate") is False:
            raise ValueError("yarn scaling with mscale or without truncation is not supported")
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

        def dim_of(rotations: float) -> float:   # the pair that completes so many rotations
            return dims * math.log(original / (rotations * 2.0 * math.pi)) / (2.0 * math.log(theta))

        first = max(math.floor(dim_of(fast)), 0)
        last = min(math.ceil(dim_of(slow)), dims - 1)
        ramp = (torch.arange(dims // 2, dtype=torch.float64) - first) / (last - first if last != first else 0.001)
        share = 1.0 - ramp.clamp(0.0, 1.0)
        given = scaling.get("attention_factor")
        attention = float(given) if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
        return inv * share + inv / factor * (1.0 - share), attention
    raise ValueError(f"unknown rope scaling {kind!r}")


def rope_tables(
    dims: int,
    length: int,
    theta: float = 10000.0,
    scaling: dict | None = None,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin float32 [length, dims / 2] of the positions 0 .. length - 1.
    Angles are formed in 64 bits: at position 100000 a 32-bit angle is off by
    up to 0.004."""
    if length < 0:
        raise ValueError("length must not be negative")
    inv, factor = rope_frequencies(dims, theta, scaling, length)
    angles = torch.outer(torch.arange(length, dtype=torch.float64, device=device), inv.to(device))
    return (angles.cos() * factor).float(), (angles.sin() * factor).float()


def rotary(
    x: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    interleaved: bool = False,
) -> torch.Tensor:
    """``rotary_cuda`` for GPU tensors; the same in torch operations on the CPU."""
    if x.is_cuda:
        return rotary_cuda(x, positions, cos, sin, interleaved)
    return rotary_reference(x, positions, cos, sin, interleaved)
