"""The work that a user of the 8-bit key/value cache has it do, as cases that
can be timed and checked one by one: rotating queries and keys, writing keys
and values into the cache and reading it back, and attention over the cache.

``run`` computes a case in plain torch operations where ``own`` is false, and
calls the library's operators where it is true; both update the state's cache
in place and return whole outputs. ``exact`` states the same operators in 64
bits.

Sizes are those of this repository's decoder (the 1.1B Llama: 32/4 heads of
64, 22 layers; the 8B class: 32/8 heads of 128) and generic serving sizes.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "fp8": 448.0}       # the largest code's value
LOWEST, HIGHEST = -40, 40                  # exponents of the scales


def listed() -> list[dict]:
    return [
        # the smallest call: one decoded token's queries of the 1.1B model
        {"name": "rotary_token_1.1b", "kind": "rotary", "batch": 1, "tokens": 1, "heads": 32, "dim": 64, "rot": 64,
         "interleaved": False, "type": "fp16", "slots": 2048, "far": 1500},
        # a prompt of a model with interleaved pairs in half of its head, deep into a long context
        {"name": "rotary_prompt_2011_part", "kind": "rotary", "batch": 2, "tokens": 2011, "heads": 32, "dim": 128,
         "rot": 64, "interleaved": True, "type": "bf16", "slots": 131072, "far": 120000},
        # one decoded token of the 1.1B model: q and k rotated, k and v written into a short cache, read back
        {"name": "write_token_1.1b", "kind": "write", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 4, "dim": 64,
         "slots": 64, "block": 64, "codes": "int8", "type": "fp16", "start": 40, "ragged": False, "padded": False,
         "rope": True, "interleaved": False},
        # a step of 32 sequences of different lengths, small blocks
        {"name": "write_batch32_fp8", "kind": "write", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "slots": 257, "block": 16, "codes": "fp8", "type": "bf16", "start": 250, "ragged": True,
         "padded": False, "rope": False, "interleaved": False},
        # four padded prompts of up to 2000 tokens, appended to what each sequence holds
        {"name": "write_prompts_4x2000", "kind": "write", "batch": 4, "tokens": 2000, "heads": 32, "kv_heads": 8,
         "dim": 128, "slots": 2100, "block": 64, "codes": "int8", "type": "fp16", "start": 90, "ragged": True,
         "padded": True, "rope": True, "interleaved": False},
        # the 1.1B model's layer cache, read back
        {"name": "read_2048_1.1b", "kind": "read", "batch": 1, "kv_heads": 4, "dim": 64, "slots": 2048, "block": 64,
         "codes": "int8", "type": "fp16"},
        # eight long sequences of the 8B class, read back
        {"name": "read_8x8192_fp8", "kind": "read", "batch": 8, "kv_heads": 8, "dim": 128, "slots": 8192, "block": 32,
         "codes": "fp8", "type": "bf16"},
        # a decoded token of the 1.1B model, 1500 tokens into a 2048-slot cache
        {"name": "attend_token_1.1b", "kind": "attend", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 4,
         "dim": 64, "slots": 2048, "block": 64, "codes": "int8", "type": "fp16", "start": 1500, "ragged": False,
         "padded": False},
        # a step of 32 sequences of the 8B class, up to 8000 tokens each
        {"name": "attend_batch32_8000_fp8", "kind": "attend", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "slots": 8192, "block": 64, "codes": "fp8", "type": "bf16", "start": 8000, "ragged": True,
         "padded": False},
        # five drafted tokens of one sequence at the end of a long context
        {"name": "attend_drafts5_131k", "kind": "attend", "batch": 1, "tokens": 5, "heads": 32, "kv_heads": 8,
         "dim": 128, "slots": 131072, "block": 128, "codes": "int8", "type": "fp16", "start": 130999,
         "ragged": False, "padded": False},
        # a 700-token prompt of the 1.1B model
        {"name": "attend_prompt_700_1.1b", "kind": "attend", "batch": 1, "tokens": 700, "heads": 32, "kv_heads": 4,
         "dim": 64, "slots": 1024, "block": 64, "codes": "int8", "type": "fp16", "start": 0, "ragged": False,
         "padded": False},
        # a long prompt of the 8B class
        {"name": "attend_prompt_4096_fp8", "kind": "attend", "batch": 1, "tokens": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "slots": 4096, "block": 64, "codes": "fp8", "type": "bf16", "start": 0, "ragged": False,
         "padded": False},
    ]


def _log(rng, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "write", "write", "read", "attend", "attend", "attend"])
    heads, kv_heads = rng.choice([(32, 4), (32, 8), (16, 16), (28, 4), (64, 8), (12, 2), (8, 1)])
    dim = rng.choice([64, 64, 128, 128, 128, 256])
    kinds = {"type": rng.choice(["fp16", "bf16"])}
    codes = {"codes": rng.choice(["int8", "fp8"]), "block": rng.choice([16, 32, 64, 64, 128])}
    if kind == "rotary":
        tokens, batch = _log(rng, 1, 4096), rng.choice([1, 1, 2, 4])
        slots = rng.choice([2048, 8192, 131072])
        far = rng.randrange(0, max(1, slots - tokens))
        if far + tokens > slots:
            tokens = slots - far
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5, **kinds,
                "slots": slots, "far": far}
    if kind == "write":
        tokens = rng.choice([1, _log(rng, 1, 16), _log(rng, 1, 2048)])
        batch = _log(rng, 1, 64) if tokens <= 16 else rng.choice([1, 2, 4])
        start = _log(rng, 1, 500) - 1
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "slots": start + tokens + rng.randrange(0, 80), **codes, **kinds, "start": start,
                "ragged": batch > 1, "padded": tokens > 1 and batch > 1 and rng.random() < 0.5,
                "rope": rng.random() < 0.5, "interleaved": rng.random() < 0.5}
    if kind == "read":
        slots = _log(rng, 100, 16384)
        batch = max(1, min(_log(rng, 1, 32), 60_000_000 // (slots * kv_heads * dim)))
        return {"kind": kind, "batch": batch, "kv_heads": kv_heads, "dim": dim, "slots": slots, **codes,
                "type": rng.choice(["fp16", "bf16", "fp32"])}
    if rng.random() < 0.6:   # decoding: a token or a few drafts of each sequence
        tokens = rng.choice([1, 1, 1, rng.randrange(2, 9)])
        start = _log(rng, 1, 130000) - 1
        batch = max(1, min(_log(rng, 1, 64), 250_000_000 // ((start + tokens) * kv_heads * dim)))
    else:                    # prompts, from the start or behind what the cache holds
        tokens = _log(rng, 9, 3000)
        start = rng.choice([0, 0, _log(rng, 1, 1000)])
        batch = max(1, min(rng.choice([1, 1, 2, 4]), 250_000_000_000 // (2 * tokens * (tokens + 2 * start) * heads * dim)))
        if 2 * tokens * (tokens + 2 * start) * heads * dim > 250_000_000_000:
            heads, kv_heads, dim = 32, 8, 64
    return {"kind": "attend", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "slots": start + tokens + rng.randrange(0, 200), **codes, **kinds, "start": start, "ragged": batch > 1,
            "padded": tokens > 1 and batch > 1 and rng.random() < 0.5}


# ------------------------------------------------------------------ the inputs

def _starts(case: dict) -> list[int]:
    """Tokens that each sequence holds before the call: all `start`, or, ragged, from half of it up."""
    start, batch = case["start"], case["batch"]
    if not case["ragged"]:
        return [start] * batch
    return [start - (start // 2) * (7 * b % batch) // batch for b in range(batch)]


def _counts(case: dict) -> list[int]:
    """New tokens of each sequence: all `tokens`, or, padded, fewer (one sequence brings none)."""
    tokens, batch = case["tokens"], case["batch"]
    if not case["padded"]:
        return [tokens] * batch
    return [tokens * ((5 * b + 2) % (batch + 1)) // batch if b else tokens for b in range(batch)]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, gen) -> torch.Tensor:
    return torch.randn(shape, device=DEVICE, generator=gen)


def _keys(shape, gen) -> torch.Tensor:
    """Keys as models have them: some channels several times larger than the rest."""
    channels = torch.exp(0.6 * _normal((shape[-1],), gen))
    return _normal(shape, gen) * channels


def _exponent(amax: torch.Tensor, codes: str) -> torch.Tensor:
    """The smallest e with amax <= MOST 2^e, within the range of the scales."""
    mantissa, e = torch.frexp(amax)                      # amax = mantissa 2^e, mantissa in [1/2, 1)
    top, shift = math.frexp(MOST[codes])
    e = e - shift + (mantissa > top).to(e.dtype)
    return torch.where(amax == 0, torch.full_like(e, LOWEST), e).clamp_(LOWEST, HIGHEST)


def _encode(x: torch.Tensor, codes: str) -> torch.Tensor:
    """Scaled fp32 values -> codes, half to even, saturated."""
    if codes == "int8":
        return torch.round(x).clamp_(-127, 127).to(torch.int8)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _filled(case: dict, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A cache [batch, kv_heads, slots, dim] of the values x: codes and scales."""
    block = case["block"]
    b, h, s, d = x.shape
    blocks = -(-s // block)
    whole = torch.nn.functional.pad(x, (0, 0, 0, blocks * block - s)).reshape(b, h, blocks, block * d)
    e = _exponent(whole.abs().amax(dim=3), case["codes"])
    scales = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    codes = _encode(whole / scales.unsqueeze(3), case["codes"]).reshape(b, h, blocks * block, d)[:, :, :s]
    return codes.contiguous(), scales.contiguous()


def _tables(slots: int, rot: int, theta: float = 10000.0) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin [slots, rot / 2] fp32 of the angles position theta^(-2i / rot)."""
    inv = theta ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
    angles = torch.outer(torch.arange(slots, device=DEVICE, dtype=torch.float64), inv)
    return angles.cos().float(), angles.sin().float()


def prepare(case: dict, seed: int) -> dict:
    gen = _gen(seed)
    kind, d = case["kind"], case["dim"]
    state: dict = {"case": case}
    dtype = TYPES[case["type"]]
    if kind == "rotary":
        b, t, h = case["batch"], case["tokens"], case["heads"]
        # the queries of a fused q|k|v projection: rows with other values behind them
        state["x"] = _normal((b, t, h + 4, d), gen).to(dtype)[:, :, :h]
        state["positions"] = (case["far"] + torch.arange(t, device=DEVICE)).expand(b, t).contiguous()
        state["cos"], state["sin"] = _tables(case["slots"], case["rot"])
        return state
    b, kv, s = case["batch"], case["kv_heads"], case["slots"]
    # what the cache holds; slots behind a sequence's tokens hold leftovers of earlier ones
    state["k_codes"], state["k_scales"] = _filled(case, _keys((b, kv, s, d), gen))
    state["v_codes"], state["v_scales"] = _filled(case, _normal((b, kv, s, d), gen))
    if kind == "read":
        return state
    t, h = case["tokens"], case["heads"]
    state["start"] = torch.tensor(_starts(case), device=DEVICE)
    state["counts"] = torch.tensor(_counts(case), device=DEVICE) if case["padded"] else None
    if kind == "attend":
        state["q"] = _normal((b, t, h, d), gen).to(dtype)
        return state
    # q, k and v are views of one projection's rows; keys a little larger than the cache's, so that scales grow
    qkv = torch.cat([_normal((b, t, h, d), gen), 1.5 * _keys((b, t, kv, d), gen), _normal((b, t, kv, d), gen)], dim=2)
    state["q"], state["k"], state["v"] = qkv.to(dtype).split([h, kv, kv], dim=2)
    if case["rope"]:
        state["cos"], state["sin"] = _tables(s, d)
    return state


# -------------------------------------------------------------- the plain form

def _rotate(x, cos, sin, positions, interleaved):
    """x [b, t, heads, dim] rotated by the tables' rows at positions [b, t]."""
    rot = 2 * cos.shape[1]
    c, s = cos[positions].unsqueeze(2), sin[positions].unsqueeze(2)
    part, rest = x[..., :rot].float(), x[..., rot:]
    if interleaved:
        x1, x2 = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).flatten(-2)
    else:
        x1, x2 = part.chunk(2, dim=-1)
        turned = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _write(x, codes, scales, start, counts, block, name):
    """New tokens x [b, t, kv_heads, dim] into codes / scales at slots start ..:
    the blocks that they touch are rebuilt, one region of whole blocks for each sequence."""
    b, t, h, d = x.shape
    s, blocks = codes.shape[2], scales.shape[2]
    n = min(blocks, (t + block - 2) // block + 1)                  # blocks of a region
    first = (start // block).clamp(max=blocks - n)
    at_block = first.unsqueeze(1) + torch.arange(n, device=DEVICE)                       # [b, n]
    slot = (first * block).unsqueeze(1) + torch.arange(n * block, device=DEVICE)         # [b, n block]
    slot = slot.clamp(max=s - 1)                                   # past the end: the last slot once more
    token = slot - start.unsqueeze(1)
    count = torch.full_like(start, t) if counts is None else counts
    new = (token >= 0) & (token < count.unsqueeze(1))
    rows = torch.arange(b, device=DEVICE).unsqueeze(1)
    values = x[rows, token.clamp(0, t - 1)].float().permute(0, 2, 1, 3)                  # [b, h, n block, d]
    old = codes[rows, :, slot].float().permute(0, 2, 1, 3)
    was = scales[rows, :, at_block].permute(0, 2, 1)                                     # [b, h, n]
    fresh = torch.where(new[:, None, :, None], values, torch.zeros_like(values))
    e = _exponent(fresh.reshape(b, h, n, block * d).abs().amax(dim=3), name)
    scale = torch.ldexp(torch.ones_like(was), e)
    lives = (at_block * block < start.unsqueeze(1)).unsqueeze(1)                         # earlier tokens in the block
    scale = torch.where(lives, torch.maximum(scale, was), scale)
    touched = new.reshape(b, 1, n, block).any(dim=3)
    scale = torch.where(touched, scale, was)
    per_slot = scale.repeat_interleave(block, dim=2).unsqueeze(3)
    old_slot = was.repeat_interleave(block, dim=2).unsqueeze(3)
    earlier = (token < 0).unsqueeze(1).unsqueeze(3)                # slots behind the new tokens keep their codes
    kept = _encode(torch.where(earlier, old * (old_slot / per_slot), old), name)
    result = torch.where(new[:, None, :, None], _encode(fresh / per_slot, name).float(), kept.float())
    codes[rows, :, slot] = result.permute(0, 2, 1, 3).to(codes.dtype)
    scales[rows, :, at_block] = scale.permute(0, 2, 1)


def _read(codes, scales, block, dtype):
    s = codes.shape[2]
    per_slot = scales.repeat_interleave(block, dim=2)[:, :, :s].unsqueeze(3)
    return (codes.float() * per_slot).to(dtype)


def _attend(q, k, v, start, counts):
    """q [b, t, heads, dim]; k, v fp32 [b, kv_heads, slots, dim]."""
    b, t, h, d = q.shape
    kv, s = k.shape[1], k.shape[2]
    rows = q.float().permute(0, 2, 1, 3).reshape(b, kv, (h // kv) * t, d)
    scores = torch.matmul(rows, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    scores = scores.reshape(b, h, t, s)
    position = start.unsqueeze(1) + torch.arange(t, device=DEVICE)                       # [b, t]
    hidden = torch.arange(s, device=DEVICE) > position.unsqueeze(2)                      # [b, t, s]
    scores = scores.masked_fill(hidden.unsqueeze(1), float("-inf"))
    weights = torch.exp(scores - scores.amax(dim=3, keepdim=True))
    weights = weights / weights.sum(dim=3, keepdim=True)
    out = torch.matmul(weights.reshape(b, kv, (h // kv) * t, s), v)
    out = out.reshape(b, h, t, d).permute(0, 2, 1, 3)
    if counts is not None:
        padding = torch.arange(t, device=DEVICE) >= counts.unsqueeze(1)
        out = out.masked_fill(padding[:, :, None, None], 0.0)
    return out.to(q.dtype).contiguous()


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if own:
        from nibble_amd import kv_attention_cuda, kv_read_cuda, kv_write_cuda, rotary_cuda, rotary_kv_write_cuda

        if kind == "rotary":
            return rotary_cuda(state["x"], state["positions"], state["cos"], state["sin"], case["interleaved"])
        cache = (state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
        if kind == "attend":
            return kv_attention_cuda(state["q"], *cache, state["start"], state["counts"])
        out = {}
        if kind == "write":
            if case["rope"]:
                out["q"] = rotary_kv_write_cuda(state["q"], state["k"], state["v"], state["cos"], state["sin"],
                                                *cache, state["start"], state["counts"], case["interleaved"])
            else:
                kv_write_cuda(state["k"], state["v"], *cache, state["start"], state["counts"])
            out["k_scales"], out["v_scales"] = state["k_scales"], state["v_scales"]
        dtype = TYPES[case["type"]]
        out["k"] = kv_read_cuda(state["k_codes"], state["k_scales"], dtype)
        out["v"] = kv_read_cuda(state["v_codes"], state["v_scales"], dtype)
        return out
    if kind == "rotary":
        return _rotate(state["x"], state["cos"], state["sin"], state["positions"], case["interleaved"])
    block, name = case["block"], case["codes"]
    if kind == "attend":
        k = _read(state["k_codes"], state["k_scales"], block, torch.float32)
        v = _read(state["v_codes"], state["v_scales"], block, torch.float32)
        return _attend(state["q"], k, v, state["start"], state["counts"])
    out = {}
    if kind == "write":
        k = state["k"]
        if case["rope"]:
            # tokens past a sequence's count are padding: their queries come out as zeros, their keys nowhere
            at = torch.arange(case["tokens"], device=DEVICE)
            positions = (state["start"].unsqueeze(1) + at).clamp(max=case["slots"] - 1)
            out["q"] = _rotate(state["q"], state["cos"], state["sin"], positions, case["interleaved"])
            if state["counts"] is not None:
                out["q"] = out["q"].masked_fill((at >= state["counts"].unsqueeze(1))[:, :, None, None], 0.0)
            k = _rotate(k, state["cos"], state["sin"], positions, case["interleaved"])
        _write(k, state["k_codes"], state["k_scales"], state["start"], state["counts"], block, name)
        _write(state["v"], state["v_codes"], state["v_scales"], state["start"], state["counts"], block, name)
        out["k_scales"], out["v_scales"] = state["k_scales"], state["v_scales"]
    dtype = TYPES[case["type"]]
    out["k"] = _read(state["k_codes"], state["k_scales"], block, dtype)
    out["v"] = _read(state["v_codes"], state["v_scales"], block, dtype)
    return out


# ------------------------------------------------------------------- the work

def work(case: dict) -> dict:
    kind, d = case["kind"], case["dim"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
    if kind == "rotary":
        values = case["batch"] * case["tokens"] * case["heads"] * d
        pairs = case["batch"] * case["tokens"] * case["heads"] * case["rot"] // 2
        return {"bytes": 2 * size * values + 4 * case["tokens"] * case["rot"] + 8 * case["batch"] * case["tokens"],
                "flops": 6 * pairs}
    kv, s = case["kv_heads"], case["slots"]
    cached = case["batch"] * kv * s * d
    scales = 4 * case["batch"] * kv * -(-s // case["block"])
    if kind == "read":
        return {"bytes": 2 * (cached * (1 + size) + scales), "flops": 2 * cached}
    starts, counts = _starts(case), _counts(case)
    if kind == "write":
        new = sum(counts)
        moved = 2 * new * kv * d * (size + 1)                        # k and v in, codes out
        turned = 0
        if case["rope"]:
            moved += size * (new + case["batch"] * case["tokens"]) * case["heads"] * d + 4 * case["tokens"] * d
            turned = 3 * d * new * (case["heads"] + kv)
        return {"bytes": moved + 2 * (cached * (1 + size) + scales), "flops": turned + 4 * new * kv * d + 2 * cached}
    h, t = case["heads"], case["tokens"]
    held = sum(a + c for a, c in zip(starts, counts) if c)
    seen = sum(c * a + c * (c + 1) // 2 for a, c in zip(starts, counts))     # (query, slot) pairs
    return {"bytes": 2 * held * kv * (d + 4 / case["block"]) + 2 * size * case["batch"] * t * h * d,
            "flops": 4 * d * h * seen}


# ------------------------------------------------------------------ in 64 bits

def _exact_turn(x, cos, sin, interleaved):
    """x [t, heads, dim] in 64 bits, rotated by cos / sin [t, rot / 2]."""
    y = x.clone()
    half = cos.shape[1]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(x[..., one], x[..., two]) * torch.complex(cos, sin).unsqueeze(1)
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_round(x, codes):
    """Scaled values in 64 bits to the nearest values that a code stands for, ties to even."""
    if codes == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)   # spacing of e4m3
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_write(case, x, codes, scales, b, start, count):
    """Sequence b's new tokens x [count, kv_heads, dim] block by block."""
    block, most = case["block"], MOST[case["codes"]]
    at = start
    while at < start + count:
        j = at // block
        end = min((j + 1) * block, start + count)
        new = x[at - start:end - start].permute(1, 0, 2)                              # [kv_heads, n, dim]
        amax = new.abs().amax(dim=(1, 2))
        e = torch.ceil(torch.log2((amax / most).clamp(min=2.0 ** LOWEST)))
        scale = torch.exp2(e.clamp(LOWEST, HIGHEST))
        if j * block < start:
            was = scales[b, :, j].clone()
            scale = torch.maximum(scale, was)
            held = slice(j * block, start)
            codes[b, :, held] = _exact_round(codes[b, :, held] * (was / scale)[:, None, None], case["codes"])
        scales[b, :, j] = scale
        codes[b, :, at:end] = _exact_round(new / scale[:, None, None], case["codes"])
        at = end


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind, d = case["kind"], case["dim"]
    if kind == "rotary":
        at = state["positions"][0]
        cos, sin = state["cos"].double()[at], state["sin"].double()[at]
        return torch.stack([_exact_turn(x.double(), cos, sin, case["interleaved"]) for x in state["x"]])
    block, s = case["block"], case["slots"]
    codes = {n: state[n + "_codes"].double() for n in "kv"}
    scales = {n: state[n + "_scales"].double() for n in "kv"}
    out = {}
    if kind == "write":
        turned = []
        for b, (start, count) in enumerate(zip(_starts(case), _counts(case))):
            k, v = state["k"][b].double(), state["v"][b].double()
            if case["rope"]:
                at = (start + torch.arange(case["tokens"], device=DEVICE)).clamp(max=s - 1)
                cos, sin = state["cos"].double()[at], state["sin"].double()[at]
                turned.append(_exact_turn(state["q"][b].double(), cos, sin, case["interleaved"]))
                turned[-1][count:] = 0
                k = _exact_turn(k, cos, sin, case["interleaved"]).to(TYPES[case["type"]]).double()
            _exact_write(case, k[:count], codes["k"], scales["k"], b, start, count)
            _exact_write(case, v[:count], codes["v"], scales["v"], b, start, count)
        if turned:
            out["q"] = torch.stack(turned)
        out["k_scales"], out["v_scales"] = scales["k"], scales["v"]
    if kind != "attend":
        for n in "kv":
            out[n] = codes[n] * scales[n].repeat_interleave(block, dim=2)[:, :, :s].unsqueeze(3)
        return out
    t, h, kv = case["tokens"], case["heads"], case["kv_heads"]
    if work(case)["flops"] > 1e12:
        return None
    result = torch.zeros((case["batch"], t, h, d), dtype=torch.float64, device=DEVICE)
    for b, (start, count) in enumerate(zip(_starts(case), _counts(case))):
        end = start + count
        hidden = torch.arange(end, device=DEVICE) > (start + torch.arange(count, device=DEVICE)).unsqueeze(1)
        for g in range(kv if count else 0):
            per_slot = {n: scales[n][b, g].repeat_interleave(block)[:end].unsqueeze(1) for n in "kv"}
            keys, values = (codes[n][b, g, :end] * per_slot[n] for n in "kv")
            for i in range(g * (h // kv), (g + 1) * (h // kv)):
                scores = state["q"][b, :count, i].double() @ keys.t().contiguous() / math.sqrt(d)
                result[b, :count, i] = scores.masked_fill(hidden, float("-inf")).softmax(dim=1) @ values
    return result
