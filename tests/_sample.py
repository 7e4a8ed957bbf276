"""64-bit oracle of sampling (test infrastructure; numpy, row by row) and logits."""

from __future__ import annotations

import numpy as np
import torch


def tokens(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> set[int]:
    """The tokens that a row may give. A weight is held to 2^-45 of the largest one
    and to 2^-38 of itself; so sums of n weights are off by less than 2^-38 of
    themselves and n 2^-45, each of two that are compared, and a border that lies
    so near may fall on either side."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any():
        return {int(np.argmax(np.isnan(x)))}
    top = x.max()
    if not temperature > 0 or top == -np.inf or top_k == 1:
        return {int(x.argmax())}
    with np.errstate(invalid="ignore"):
        w = np.exp((x - top) / temperature)
    w[x == top], w[x == -np.inf] = 1.0, 0.0
    slack = len(x) * 2.0 ** -44 + w.sum() * 2.0 ** -37
    order = np.lexsort((np.arange(len(x)), -x))
    if top_k > 0:
        order = order[:top_k]
    found = set()
    for side_p in (-1, 1):
        kept = order
        if top_p < 1.0:
            before = np.cumsum(w[kept]) - w[kept]
            keep = before < max(top_p, 0.0) * w[kept].sum() + side_p * slack
            keep[0] = True
            kept = kept[keep]
        for side_m in (-1, 1):
            least = min(min_p if min_p > 0.0 else 0.0, 1.0) * (1 + side_m * 2.0 ** -37)   # NaN: none
            chosen = kept[(w[kept] >= least) | (w[kept] == 1.0)]
            mask = np.zeros(len(x), dtype=bool)
            mask[chosen] = True
            sums = np.cumsum(np.where(mask, w, 0.0))
            u01 = 0.0 if np.isnan(u) else min(max(float(u), 0.0), 1.0)
            for side_u in (-1, 1):
                at = np.searchsorted(sums, u01 * sums[-1] + side_u * slack, side="right")
                live = np.flatnonzero(mask & (w > 0))
                # the first kept one at or after it (the last, where there is none)
                after = live[live >= at]
                found.add(int(after[0] if len(after) else live[live < at][-1]))
    return found


def check(got: torch.Tensor, logits: torch.Tensor, random: torch.Tensor, **settings) -> None:
    """Each row's token is one that the oracle gives."""
    x, u = logits.detach().cpu().double().numpy(), random.cpu().double().numpy()
    pick = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    settings = {n: v.cpu() if isinstance(v, torch.Tensor) else v for n, v in settings.items()}
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    for r, token in enumerate(got.tolist()):
        allowed = tokens(x[r], u[r], **{n: pick(v, r) for n, v in settings.items()})
        assert token in allowed, f"row {r}: {token}, not {sorted(allowed)}"


def logits(rows: int, n: int, dtype: torch.dtype, seed: int, spread: float = 2.2) -> torch.Tensor:
    """A broad bulk and a head of likely tokens, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, n), generator=g)
    head = torch.randint(n, (rows, min(20, n)), generator=g)
    return x.scatter_add_(1, head, 3.0 + 2.0 * torch.randn((rows, min(20, n)), generator=g).abs()).to(dtype)


def numbers(rows: int, seed: int) -> torch.Tensor:
    return torch.rand((rows,), generator=torch.Generator().manual_seed(seed))


INF, NAN = float("inf"), float("nan")
# rows where sampling can go wrong: (logits, settings)
EDGES = [
    ([0.5], {}),
    ([1.0, 1.0], {"top_p": 0.5}),                               # half of the weight lies before the second: dropped
    ([1.0, 1.0], {"top_p": 0.5000001}),
    ([3.0, 3.0, 3.0, 1.0, 3.0], {"top_k": 2}),                  # ties: the first two
    ([3.0, 3.0, 3.0, 1.0, 3.0], {"top_k": 3, "top_p": 0.4}),
    ([0.0, -0.0, 0.0, -1.0], {"top_k": 2}),                     # -0 equals 0
    ([-0.0, -5.0, 0.0], {"top_p": 0.3}),
    ([-INF, 2.0, -INF, 1.0], {}),
    ([-INF, 2.0, -INF, 1.0], {"top_k": 3}),                     # more than have a weight
    ([-INF, 2.0, -INF, 1.0], {"temperature": INF}),
    ([-INF] * 5, {}),
    ([-INF] * 5, {"top_k": 2, "top_p": 0.5, "min_p": 0.1}),
    ([INF, 1.0, INF, -INF], {}),
    ([INF, 1.0, INF, -INF], {"top_k": 1}),
    ([INF, 1.0, INF, -INF], {"top_p": 0.5, "min_p": 1.0}),
    ([1.0, NAN, INF, NAN], {}),
    ([1.0, -INF, NAN], {"top_k": 2, "temperature": 0.5}),
    ([1.0, 5.0, 5.0, 2.0], {"temperature": 0.0}),
    ([1.0, 5.0, 5.0, 2.0], {"temperature": 1e-30}),
    ([1.0, 5.0, 4.9, 2.0], {"temperature": 1e30}),
    ([60000.0, -60000.0, 59968.0], {}),
    ([1.0, 2.0, 3.0], {"min_p": 1.0}),
    ([1.0, 2.0, 3.0], {"min_p": 0.2}),
    ([1.0, 2.0, 3.0], {"top_p": 0.0}),
    ([1.0, 2.0, 3.0], {"top_k": 3}),
    ([1.0, 2.0, 3.0], {"top_k": 100, "top_p": 0.99, "min_p": 0.05}),
    ([-1.0, -2.0, -3.0, -40.0], {"temperature": 0.7}),          # a weight below 2^-46
]
EDGE_NUMBERS = [0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24, 1.0, -1.0, NAN, INF]
