"""The work of answering one prompt several times, as cases that can be timed
and checked one by one: drawing tokens from rows of logits, attention of a batch
whose sequences share a prefix, copying a prompt's cache into several sequences
and moving sequences within a cache.

``run`` computes a case in plain torch operations where ``own`` is false, and
calls the library's operators where it is true; caches are updated in place and
returned whole. ``exact`` states the same operators in 64 bits.

Sizes are those of this repository's decoder (the 1.1B Llama: 32/4 heads of
64, 32000 tokens; the 8B class: 32/8 heads of 128) and generic serving sizes.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "fp8": 448.0}       # the largest code's value
LOWEST, HIGHEST = -40, 40                  # exponents of the scales


def listed() -> list[dict]:
    return [
        # the smallest call: the next token of one sequence of the 1.1B model
        {"name": "sample_token_1.1b", "kind": "sample", "rows": 1, "vocab": 32000, "type": "fp16",
         "temperature": 0.75, "top_k": 50, "top_p": 0.9375, "min_p": 0.0, "mixed": False, "masked": 0.0},
        # seven requests of one serving step, each with its own settings (greedy ones among them), an odd vocabulary
        {"name": "sample_requests7_50257", "kind": "sample", "rows": 7, "vocab": 50257, "type": "fp32",
         "temperature": 1.0, "top_k": 200, "top_p": 0.9, "min_p": 0.05, "mixed": True, "masked": 0.0},
        # sixteen answers under a grammar that allows a tenth of the tokens, drawn from all of them
        {"name": "sample_grammar16_32000", "kind": "sample", "rows": 16, "vocab": 32000, "type": "bf16",
         "temperature": 1.25, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False, "masked": 0.9},
        # a full batch of a large vocabulary by top-p
        {"name": "sample_batch256_128000", "kind": "sample", "rows": 256, "vocab": 128000, "type": "bf16",
         "temperature": 0.875, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "mixed": False, "masked": 0.0},
        # a step of sixteen answers of the 1.1B model, 1500 tokens of prompt and about 100 of each answer
        {"name": "attend_answers16_1.1b", "kind": "attend", "groups": 1, "batch": 16, "tokens": 1, "heads": 32,
         "kv_heads": 4, "dim": 64, "prefix": 1500, "slots": 256, "block": 64, "codes": "int8", "type": "fp16",
         "start": 100, "padded": False},
        # a step of 64 sequences of the 8B class behind one long system prompt
        {"name": "attend_batch64_8192_fp8", "kind": "attend", "groups": 1, "batch": 64, "tokens": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "prefix": 8192, "slots": 1024, "block": 64, "codes": "fp8", "type": "bf16",
         "start": 800, "padded": False},
        # four documents of 30001 tokens, two drafted answers of three tokens to each
        {"name": "attend_drafts4x2_30001", "kind": "attend", "groups": 4, "batch": 8, "tokens": 3, "heads": 28,
         "kv_heads": 4, "dim": 128, "prefix": 30001, "slots": 77, "block": 32, "codes": "int8", "type": "fp16",
         "start": 60, "padded": False},
        # four padded questions of up to 500 tokens behind a shared prompt, taken in at once
        {"name": "attend_questions4x500_6000", "kind": "attend", "groups": 1, "batch": 4, "tokens": 500, "heads": 32,
         "kv_heads": 8, "dim": 128, "prefix": 6000, "slots": 512, "block": 64, "codes": "fp8", "type": "bf16",
         "start": 0, "padded": True},
        # the 1.1B model's layer cache of a short prompt into four answers
        {"name": "fork_4_1.1b", "kind": "fork", "held": 1, "batch": 4, "kv_heads": 4, "dim": 64, "from_slots": 300,
         "slots": 512, "block": 64, "codes": "int8", "length": 299},
        # three prompts of the 8B class into eight beams each
        {"name": "fork_3x8_4000_fp8", "kind": "fork", "held": 3, "batch": 24, "kv_heads": 8, "dim": 128,
         "from_slots": 4100, "slots": 4500, "block": 32, "codes": "fp8", "length": 4001},
        # finished ones out of five short answers: the others move up
        {"name": "reorder_5_compact", "kind": "reorder", "order": "compact", "batch": 5, "kv_heads": 4, "dim": 64,
         "slots": 256, "block": 64, "codes": "int8", "length": 131},
        # a beam search's step over 32 sequences of the 8B class
        {"name": "reorder_beams32_2000", "kind": "reorder", "order": "beams", "batch": 32, "kv_heads": 8, "dim": 128,
         "slots": 2300, "block": 64, "codes": "fp8", "length": 2000},
    ]


def _log(rng, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["sample", "sample", "attend", "attend", "attend", "fork", "reorder"])
    if kind == "sample":
        vocab = _log(rng, 1000, 160000)
        return {"kind": kind, "rows": max(1, min(_log(rng, 1, 256), 30_000_000 // vocab)), "vocab": vocab,
                "type": rng.choice(["fp16", "bf16", "fp32"]), "temperature": rng.choice([0.5, 0.8, 1.0, 1.3]),
                "top_k": rng.choice([0, 0, _log(rng, 1, 1000)]), "top_p": rng.choice([1.0, rng.uniform(0.3, 0.99)]),
                "min_p": rng.choice([0.0, 0.0, rng.uniform(0.01, 0.3)]), "mixed": rng.random() < 0.5,
                "masked": rng.choice([0.0, 0.0, rng.uniform(0.1, 0.99)])}
    heads, kv_heads = rng.choice([(32, 4), (32, 8), (16, 16), (28, 4), (64, 8), (12, 2), (8, 1)])
    dim = rng.choice([64, 64, 128, 128, 128, 256])
    codes = {"codes": rng.choice(["int8", "fp8"]), "block": rng.choice([16, 32, 64, 64, 128])}
    if kind == "attend":
        groups = rng.choice([1, 1, 1, 2, 4])
        tokens = rng.choice([1, 1, 1, rng.randrange(2, 9), _log(rng, 9, 600)])
        batch = groups * (_log(rng, 1, 64) if tokens < 9 else rng.choice([1, 2, 4]))
        if batch * tokens * heads * dim * tokens > 4_000_000_000:
            batch, heads, kv_heads, dim = groups, 32, 8, 64
        most = 1_200_000_000 // (batch * tokens * heads)          # scores of the plain form
        prefix = max(1, min(_log(rng, 30, 60000), 30_000_000 // (groups * kv_heads * dim), most))
        if 4 * dim * heads * batch * tokens * prefix > 100_000_000_000:
            prefix = 100_000_000_000 // (4 * dim * heads * batch * tokens)
        start = _log(rng, 1, 500) - 1
        return {"kind": kind, "groups": groups, "batch": batch, "tokens": tokens, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "slots": start + tokens + rng.randrange(0, 100),
                **codes, "type": rng.choice(["fp16", "bf16"]), "start": start,
                "padded": tokens > 1 and batch > 1 and rng.random() < 0.5}
    length = _log(rng, 10, 8000)
    batch = max(2, min(_log(rng, 2, 64), 60_000_000 // (length * kv_heads * dim)))
    common = {"kind": kind, "batch": batch, "kv_heads": kv_heads, "dim": dim, "slots": length + rng.randrange(0, 300),
              **codes, "length": length}
    if kind == "fork":
        return {**common, "held": rng.choice([1, 1, 2, min(batch, 5)]), "from_slots": length + rng.randrange(0, 100)}
    return {**common, "order": rng.choice(["beams", "compact", "rotate"])}


# ------------------------------------------------------------------ the inputs

def _ragged(most: int, n: int) -> list[int]:
    """Lengths of n sequences, from about half of the largest up to it."""
    return [most - (most // 2) * (7 * b % n) // n for b in range(n)]


def _counts(case: dict) -> list[int]:
    """New tokens of each sequence: all `tokens`, or, padded, fewer (one sequence brings none)."""
    tokens, batch = case["tokens"], case["batch"]
    if not case["padded"]:
        return [tokens] * batch
    return [tokens * ((5 * b + 2) % (batch + 1)) // batch if b else tokens for b in range(batch)]


def _source(case: dict) -> list[int]:
    """Which sequence each one comes from."""
    n = case["batch"]
    if case["kind"] == "fork":
        return [b * case["held"] // n for b in range(n)]
    if case["order"] == "compact":         # every third one is finished: the last live ones take their places
        last, source = n - 1, list(range(n))
        for b in range(0, n, 3):
            while last > b and last % 3 == 0:
                last -= 1
            if last <= b:
                break
            source[b], last = last, last - 1
        return source
    if case["order"] == "rotate":
        return [(b + 1) % n for b in range(n)]
    return [(b * b + 3 * b) % n for b in range(n)]   # beams: some live on several times, some end


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, gen) -> torch.Tensor:
    return torch.randn(shape, device=DEVICE, generator=gen)


def _keys(shape, gen) -> torch.Tensor:
    """Keys as models have them: some channels several times larger than the rest."""
    channels = torch.exp(0.6 * _normal((shape[-1],), gen))
    return _normal(shape, gen) * channels


def _cache(case: dict, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A cache [batch, kv_heads, slots, dim] of the values x: codes, and a power-of-two scale for each block."""
    block, name = case["block"], case["codes"]
    b, h, s, d = x.shape
    blocks = -(-s // block)
    whole = torch.nn.functional.pad(x, (0, 0, 0, blocks * block - s)).reshape(b, h, blocks, block * d)
    e = torch.ceil(torch.log2((whole.abs().amax(dim=3) / MOST[name]).clamp(min=2.0 ** LOWEST))).clamp(LOWEST, HIGHEST)
    scales = torch.exp2(e)
    scaled = whole / scales.unsqueeze(3)
    codes = scaled.round().clamp(-127, 127) if name == "int8" else scaled.clamp(-448.0, 448.0)
    codes = codes.to(CODES[name]).reshape(b, h, blocks * block, d)[:, :, :s]
    return codes.contiguous(), scales.contiguous()


def prepare(case: dict, seed: int) -> dict:
    gen = _gen(seed)
    kind = case["kind"]
    state: dict = {"case": case}
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits as models give them: a broad bulk and a head of a few dozen likely tokens
        logits = 2.2 * _normal((rows, vocab), gen)
        likely = torch.randint(vocab, (rows, 40), device=DEVICE, generator=gen)
        logits.scatter_add_(1, likely, 4.0 + 2.0 * _normal((rows, 40), gen).abs())
        if case["masked"] > 0.0:
            masked = torch.rand((rows, vocab), device=DEVICE, generator=gen) < case["masked"]
            masked[:, vocab // 2] = False
            logits = logits.masked_fill(masked, float("-inf"))
        state["logits"] = logits.to(TYPES[case["type"]])
        state["random"] = torch.rand((rows,), device=DEVICE, generator=gen)
        settings = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if case["mixed"]:
            # a setting for each row: some greedy, some without a limit
            at = torch.arange(rows, device=DEVICE)
            settings["temperature"] = (case["temperature"] * (1.0 + 0.1 * (at % 5))).masked_fill(at % 4 == 3, 0.0)
            settings["top_k"] = (case["top_k"] * (1 + at % 3)).masked_fill(at % 5 == 1, 0)
            settings["top_p"] = (case["top_p"] - 0.02 * (at % 6)).masked_fill(at % 7 == 2, 1.0).float()
            settings["min_p"] = (case["min_p"] * (at % 3)).float()
        state.update(settings)
        return state
    kv, d, s, b = case["kv_heads"], case["dim"], case["slots"], case["batch"]
    state["k_codes"], state["k_scales"] = _cache(case, _keys((b, kv, s, d), gen))
    state["v_codes"], state["v_scales"] = _cache(case, _normal((b, kv, s, d), gen))
    if kind == "attend":
        g, p = case["groups"], case["prefix"]
        # the prefixes' caches have slots behind their tokens, which hold leftovers
        state["pk_codes"], state["pk_scales"] = _cache(case, _keys((g, kv, p + 40, d), gen))
        state["pv_codes"], state["pv_scales"] = _cache(case, _normal((g, kv, p + 40, d), gen))
        state["prefix"] = torch.tensor([p - 5 * i if p > 50 else p for i in range(g)], device=DEVICE)
        state["start"] = torch.tensor(_ragged(case["start"], b), device=DEVICE)
        state["counts"] = torch.tensor(_counts(case), device=DEVICE) if case["padded"] else None
        # the queries of a fused q|k|v projection: rows with other values behind them
        h = case["heads"]
        state["q"] = _normal((b, case["tokens"], h + 2 * kv, d), gen).to(TYPES[case["type"]])[:, :, :h]
        return state
    if kind == "fork":
        shape = (case["held"], kv, case["from_slots"], d)
        state["fk_codes"], state["fk_scales"] = _cache(case, _keys(shape, gen))
        state["fv_codes"], state["fv_scales"] = _cache(case, _normal(shape, gen))
    state["source"] = torch.tensor(_source(case), device=DEVICE)
    state["lengths"] = torch.tensor(_ragged(case["length"], case["held"] if kind == "fork" else b), device=DEVICE)
    return state


# -------------------------------------------------------------- the plain form

def _sample(logits, random, temperature, top_k, top_p, min_p):
    rows, n = logits.shape
    column = lambda v, t: torch.as_tensor(v, device=DEVICE).to(t).expand(rows).unsqueeze(1)  # noqa: E731
    heat, most = column(temperature, torch.float64), column(top_k, torch.int64)
    mass, least = column(top_p, torch.float64), column(min_p, torch.float64)
    x = logits.double()
    top = x.amax(dim=1, keepdim=True)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(heat > 0, heat, 1.0)))
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(n, device=DEVICE)
    keep = (rank < most) | (most <= 0)
    ws = ws * keep
    before = ws.cumsum(dim=1) - ws
    keep &= (before < mass * ws.sum(dim=1, keepdim=True)) | (mass >= 1.0)
    keep &= ws >= least
    keep &= (heat > 0) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    sums = (w * kept).cumsum(dim=1)
    return (sums > random.double().unsqueeze(1) * sums[:, -1:]).to(torch.int8).argmax(dim=1)


def _read(codes, scales, block):
    per_slot = scales.repeat_interleave(block, dim=2)[:, :, :codes.shape[2]].unsqueeze(3)
    return codes.float() * per_slot


def _attend(q, pk, pv, prefix, k, v, start, counts):
    """q [b, t, heads, dim]; pk, pv [groups, kv_heads, prefix slots, dim]; k, v [b, kv_heads, slots, dim], fp32."""
    b, t, h, d = q.shape
    g, kv, ps = pk.shape[:3]
    s, r = k.shape[2], h // kv
    rows = q.float().permute(0, 2, 1, 3) * (1.0 / math.sqrt(d))                            # [b, h, t, d]
    together = rows.reshape(g, b // g, kv, r * t, d).transpose(1, 2).reshape(g, kv, b // g * r * t, d)
    first = torch.matmul(together, pk.transpose(2, 3).contiguous())
    first = first.masked_fill(torch.arange(ps, device=DEVICE) >= prefix[:, None, None, None], float("-inf"))
    second = torch.matmul(rows.reshape(b, kv, r * t, d), k.transpose(2, 3).contiguous()).reshape(b, h, t, s)
    position = start.unsqueeze(1) + torch.arange(t, device=DEVICE)
    hidden = torch.arange(s, device=DEVICE) > position.unsqueeze(2)
    second = second.masked_fill(hidden.unsqueeze(1), float("-inf"))
    second = second.reshape(g, b // g, kv, r * t, s).transpose(1, 2).reshape(g, kv, b // g * r * t, s)
    top = torch.maximum(first.amax(dim=3, keepdim=True), second.amax(dim=3, keepdim=True))
    first, second = torch.exp(first - top), torch.exp(second - top)
    total = first.sum(dim=3, keepdim=True) + second.sum(dim=3, keepdim=True)
    second = second.reshape(g, kv, b // g, r * t, s).transpose(1, 2).reshape(b, kv, r * t, s)
    out = torch.matmul(second, v).reshape(g, b // g, kv, r * t, d).transpose(1, 2).reshape(g, kv, b // g * r * t, d)
    out = (out + torch.matmul(first, pv)) / total
    out = out.reshape(g, kv, b // g, r, t, d).permute(0, 2, 4, 1, 3, 5).reshape(b, t, h, d)
    if counts is not None:
        padding = torch.arange(t, device=DEVICE) >= counts.unsqueeze(1)
        out = out.masked_fill(padding[:, :, None, None], 0.0)
    return out.to(q.dtype).contiguous()


def _move(held, to, source, lengths, block):
    """Rows source of the tensors `held` (codes, or scales of `block` slots) into `to`, as far as they are held."""
    n = min(held.shape[2], to.shape[2])
    at = torch.arange(n, device=DEVICE) * block
    moved = at < lengths[source].unsqueeze(1)                                              # [b, n]
    moved = moved[:, None, :, None] if to.dim() == 4 else moved[:, None, :]
    raw = (lambda x: x.view(torch.int8)) if to.dim() == 4 else (lambda x: x)
    rows = raw(held)[source, :, :n]
    raw(to)[:, :, :n] = torch.where(moved, rows, raw(to)[:, :, :n])


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if kind == "sample":
        call = _sample
        if own:
            from nibble_amd import sample_cuda as call
        return call(state["logits"], state["random"], state["temperature"], state["top_k"], state["top_p"],
                    state["min_p"])
    cache = (state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
    if kind == "attend":
        prefix = (state["pk_codes"], state["pk_scales"], state["pv_codes"], state["pv_scales"])
        if own:
            from nibble_amd import kv_shared_attention_cuda

            return kv_shared_attention_cuda(state["q"], *prefix, state["prefix"], *cache, state["start"],
                                            state["counts"])
        block = case["block"]
        return _attend(state["q"], _read(*prefix[:2], block), _read(*prefix[2:], block), state["prefix"],
                       _read(*cache[:2], block), _read(*cache[2:], block), state["start"], state["counts"])
    held = tuple(state[n] for n in ("fk_codes", "fk_scales", "fv_codes", "fv_scales")) if kind == "fork" else cache
    if own:
        from nibble_amd import kv_fork_cuda, kv_reorder_cuda

        if kind == "fork":
            kv_fork_cuda(*held, *cache, state["source"], state["lengths"])
        else:
            kv_reorder_cuda(*cache, state["source"], state["lengths"])
    else:
        for x, to, block in zip(held, cache, (1, case["block"], 1, case["block"])):
            _move(x, to, state["source"], state["lengths"], block)
    return dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), cache))


# ------------------------------------------------------------------- the work

def work(case: dict) -> dict:
    kind = case["kind"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case.get("type", "fp16")]
    if kind == "sample":
        values = case["rows"] * case["vocab"]
        settings = 20 if case["mixed"] else 0                            # temperature, k, p, min p of a row
        return {"bytes": size * values + (4 + 8 + settings) * case["rows"], "flops": 3 * values}
    kv, d, b = case["kv_heads"], case["dim"], case["batch"]
    slot = 2 * kv * (d + 4 / case["block"])                              # bytes of a slot's key and value
    if kind != "attend":
        lengths = _ragged(case["length"], case["held"] if kind == "fork" else b)
        moved = [(j, lengths[j]) for i, j in enumerate(_source(case)) if kind == "fork" or i != j]
        return {"bytes": slot * (sum(n for _, n in moved) + sum(n for _, n in set(moved))), "flops": 0}
    h, t = case["heads"], case["tokens"]
    starts, counts = _ragged(case["start"], b), _counts(case)
    held = case["groups"] * case["prefix"] + sum(a + c for a, c in zip(starts, counts) if c)
    seen = sum(c * (case["prefix"] + a) + c * (c + 1) // 2 for a, c in zip(starts, counts))
    return {"bytes": slot * held + 2 * size * b * t * h * d, "flops": 4 * d * h * seen}


# ------------------------------------------------------------------ in 64 bits

def _exact_token(x: np.ndarray, u: float, heat: float, most: int, mass: float, least: float) -> int:
    """One row: x in 64 bits."""
    best = int(x.argmax())
    if heat <= 0.0:
        return best
    live = np.flatnonzero(x > -np.inf)
    order = live[np.lexsort((live, -x[live]))]
    if most > 0:
        order = order[:most]
    w = np.exp((x[order] - x[best]) / heat)
    if mass < 1.0:
        ends = np.concatenate(([0.0], np.cumsum(w)))
        n = max(1, int(np.searchsorted(ends[:-1], mass * w.sum(), side="left")))
        order, w = order[:n], w[:n]
    order, w = order[w >= least], w[w >= least]
    back = np.argsort(order)
    sums = np.cumsum(w[back])
    return int(order[back][np.searchsorted(sums, u * sums[-1], side="right")])


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        rows = case["rows"]
        of = lambda v: v.double().cpu().numpy() if torch.is_tensor(v) else np.full(rows, float(v))  # noqa: E731
        settings = [of(state[n]) for n in ("random", "temperature", "top_k", "top_p", "min_p")]
        x = state["logits"].double().cpu().numpy()
        return torch.tensor([_exact_token(x[i], settings[0][i], settings[1][i], int(settings[2][i]), settings[3][i],
                                          settings[4][i]) for i in range(rows)], device=DEVICE)
    block = case["block"]
    if kind != "attend":
        out = {}
        lengths = state["lengths"].tolist()
        for n in ("k_codes", "k_scales", "v_codes", "v_scales"):
            to = state[n].to(torch.float64)
            held = state["f" + n].to(torch.float64) if kind == "fork" else to.clone()
            for b, j in enumerate(_source(case)):
                end = lengths[j] if n.endswith("codes") else -(-lengths[j] // block)
                to[b, :, :end] = held[j, :, :end]
            out[n] = to if n.endswith("scales") or case["codes"] == "fp8" else to.to(torch.int8)
        return out
    if work(case)["flops"] > 3e11:
        return None
    values = {}
    for n in ("pk", "pv", "k", "v"):
        codes, scales = state[n + "_codes"].double(), state[n + "_scales"].double()
        slots = torch.arange(codes.shape[2], device=DEVICE) // block
        values[n] = codes * scales[:, :, slots].unsqueeze(3)
    b, t, h, d = state["q"].shape
    r, per = h // case["kv_heads"], b // case["groups"]
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device=DEVICE)
    ends = state["prefix"].tolist()
    for i, (start, count) in enumerate(zip(_ragged(case["start"], b), _counts(case))):
        if count == 0:
            continue
        p = ends[i // per]
        ahead = torch.arange(start + count, device=DEVICE) - (start + torch.arange(count, device=DEVICE)).unsqueeze(1)
        ahead = torch.cat((torch.zeros((count, p), dtype=torch.int64, device=DEVICE), ahead), dim=1)
        for j in range(case["kv_heads"]):
            k, v = (torch.cat((values["p" + n][i // per, j, :p], values[n][i, j, :start + count])) for n in "kv")
            for m in range(j * r, (j + 1) * r):
                scores = state["q"][i, :count, m].double() @ k.t().contiguous() / math.sqrt(d)
                out[i, :count, m] = scores.masked_fill(ahead > 0, float("-inf")).softmax(dim=1) @ v
    return out
