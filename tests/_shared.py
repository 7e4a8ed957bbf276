"""Oracle of attention behind shared prefixes (test infrastructure): each sequence
over one cache with its prefix's slots and its own, by the oracle of one cache."""

from __future__ import annotations

import numpy as np
import torch

from tests import _kv


def attend(q, prefix, prefix_lengths, own, start, counts, prefix_block, block, scale=None):
    """(outputs, bound); prefix and own are (k_codes, k_scales, v_codes, v_scales) on the CPU."""
    batch, tokens = q.shape[:2]
    groups, held = prefix[0].shape[0], prefix[0].shape[2]
    slots = own[0].shape[2]
    outs, bounds = [], []
    spread = lambda s, block, n: s.repeat_interleave(block, dim=1)[:, :n]  # noqa: E731
    for b in range(batch):
        g, count = b // (batch // groups), tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        n = int(prefix_lengths[g])
        known = 0 <= n <= held
        n = n if known else 0
        sides = []
        for i in (0, 2):
            codes = torch.cat((prefix[i][g, :, :n].float(), own[i][b].float()), dim=1)
            sides.append(codes.to(own[i].dtype).unsqueeze(0))
            sides.append(torch.cat((spread(prefix[i + 1][g], prefix_block, n), spread(own[i + 1][b], block, slots)),
                                   dim=1).unsqueeze(0))
        first = int(start[b])
        # rows at own positions outside the cache, or behind an unknown prefix, are NaN
        out, bound = _kv.attend(q[b:b + 1], *sides, [n + max(first, -n - tokens)], [count], 1, scale)
        for t in range(count):
            if not (known and 0 <= first + t < slots):
                out[0, t], bound[0, t] = np.nan, 0.0
        outs.append(out)
        bounds.append(bound)
    return np.concatenate(outs), np.concatenate(bounds)


def case(groups, per, tokens, heads, kv_heads, dim, prefix_slots, slots, codes="int8", dtype="fp16", prefix_block=64,
         block=32, seed=1, spread=1.0):
    """(q, prefix, own) on the CPU."""
    q = _kv.rows((groups * per, tokens, heads, dim), dtype, seed)
    make = lambda n, s, bl, x: sum((_kv.cache(n, kv_heads, s, dim, codes, bl, x + i, spread) for i in range(2)), ())  # noqa: E731
    return q, make(groups, prefix_slots, prefix_block, seed + 10), make(groups * per, slots, block, seed + 20)
