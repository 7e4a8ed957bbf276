"""Copying and reordering sequences of an 8-bit cache: a plain statement of what
changes (test infrastructure), caches, and the cases of both suites."""

from __future__ import annotations

import torch

from tests import _kv


def tensors(batch, heads, slots, dim, codes, block, seed, device="cpu", pad=0):
    """(k_codes, k_scales, v_codes, v_scales); pad: dims of other values between
    the heads of a head's row, so that strides are not dense."""
    out = []
    for i in range(2):
        c, s = _kv.cache(batch, heads, slots, dim, codes, block, seed + i)
        if pad:
            wide = torch.zeros((batch, heads + pad, slots, dim), dtype=torch.int8)
            wide[:, :heads] = c.view(torch.int8)
            c = wide.to(device).view(c.dtype)[:, :heads]
            s = torch.cat((s, torch.ones((batch, pad, s.shape[2]))), dim=1).to(device)[:, :heads]
        out += [c.to(device), s.to(device)]
    return tuple(out)


def expected(held, to, source, lengths, block):
    """`to` after the call, on the CPU, element by element of batch."""
    held = [x.detach().cpu().clone() for x in held]
    out = [x.detach().cpu().clone() for x in to]
    most = min(held[0].shape[2], out[0].shape[2])
    for b, j in enumerate(source):
        if 0 <= j < held[0].shape[0]:
            n = max(0, min(lengths[j], most))
            for i, end in enumerate((n, -(-n // block)) * 2):
                out[i].view(torch.int8 if i % 2 == 0 else torch.float32)[b, :, :end] = \
                    held[i].view(torch.int8 if i % 2 == 0 else torch.float32)[j, :, :end]
    return out


def check(got, want):
    for x, y in zip(got, want):
        assert _kv.same(x, y)


# (from: batch, slots; to: batch, slots; block; source; lengths)
FORKS = [
    (1, 70, 4, 90, 16, [0, 0, 0, 0], [33]),
    (3, 257, 5, 128, 64, [2, 0, 2, 1, 0], [257, 64, 65]),              # longer than the second's slots
    (2, 40, 3, 500, 32, [1, -1, 7], [0, 40]),                          # sources outside, an empty one
    (2, 1, 2, 1, 128, [1, 0], [1, 1]),
    (4, 130, 2, 130, 128, [3, 3], [-5, 3, 1000, 129]),
    (1, 600, 2, 600, 64, [0, 0], [600]),
]
# (batch, slots, block, source, lengths)
REORDERS = [
    (1, 40, 16, [0], [40]),
    (2, 65, 64, [1, 0], [65, 64]),
    (4, 300, 32, [1, 2, 3, 0], [300, 1, 33, 150]),
    (5, 90, 16, [0, 0, 0, 3, 3], [17, 90, 90, 0, 90]),
    (6, 128, 128, [5, -1, 6, 2, 1, 4], [128, 5, 127, -3, 64, 400]),
    (3, 1, 64, [2, 2, 0], [1, 1, 1]),
]
