"""Attention behind shared prefixes in forms that take many rows or slots: each is
named by the kernels that its sizes lead to."""

import pytest
import torch

from tests import _shared
from tests.test_gpu_kv_shared import _check

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("codes,dtype", [("int8", "fp16"), ("fp8", "bf16"), ("int8", "bf16"), ("fp8", "fp16")])


def _both(q, prefix, lengths, own, start, counts=None):
    """Also with scores past 2^22 on the prefix's side, which are weights, not NaN."""
    _check(q, prefix, lengths, own, start, counts)
    big = [x * 2.0 ** 16 if i == 1 else x for i, x in enumerate(prefix)]
    assert torch.isfinite(_check(q, big, lengths, own, start, counts)).all()


@TYPES
@pytest.mark.parametrize("per,tokens", [(2, 5), (10, 1), (12, 1)])
def test_48_rows(gpu, codes, dtype, per, tokens):
    """33 to 48 rows a prefix of head_dim 128, of 4 and of 20 rows a sequence, over several shares."""
    q, prefix, own = _shared.case(3, per, tokens, 8, 2, 128, 3001, 90, codes, dtype)
    batch = 3 * per
    _both(q, prefix, [3001, 1700, 33], own, [(7 * b) % (91 - tokens) for b in range(batch)],
          None if tokens == 1 else [tokens - b % 3 for b in range(batch)])


@TYPES
@pytest.mark.parametrize("dim,slots", [(64, 44000), (128, 700), (256, 500)])
def test_prompt_form_beside_two_row_tiles(gpu, codes, dtype, dim, slots):
    """Many rows behind a prefix beside 36 rows a sequence."""
    q, prefix, own = _shared.case(1, 4, 9, 8, 2, dim, slots, 70, codes, dtype)
    _both(q, prefix, [min(slots, 1900)], own, [0, 17, 40, 61], [9, 4, 0, 9])


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_wavefront_a_row_in_the_join(gpu, codes, dtype, dim):
    """1280 rows of a few shares of the prefix and of their own slots."""
    q, prefix, own = _shared.case(2, 40, 1, 16, 2, dim, 500, 300, codes, dtype)
    _both(q, prefix, [500, 391], own, [(23 * b) % 300 for b in range(80)], [b % 5 for b in range(80)])


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_own_slots_of_prompts_in_shares(gpu, codes, dtype, dim):
    """Tokens behind a prefix and behind up to 1680 own slots, joined by a launch of its own."""
    q, prefix, own = _shared.case(1, 2, 20, 8, 2, dim, 700, 1700, codes, dtype)
    _both(q, prefix, [700], own, [1680, 900], [20, 13])


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_own_prompts_of_many_workgroups(gpu, codes, dtype, dim):
    """64 sequences of 8 KV heads and 66 rows each, most of them padding."""
    q, prefix, own = _shared.case(2, 32, 66, 8, 8, dim, 200, 90, codes, dtype)
    counts = [66 if b in (3, 40) else b % 3 for b in range(64)]
    _both(q, prefix, [200, 77], own, [b % 25 for b in range(64)], counts)
