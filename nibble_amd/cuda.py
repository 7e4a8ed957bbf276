"""Python wrappers of the torch ops ``w4a16::linear``, ``w4a16::dequantize``,
``w4a16::quantize``, of the ops of the 8-bit key/value cache (``rotary``,
``kv_write``, ``rotary_kv_write``, ``kv_read``, ``kv_attention``,
``kv_shared_attention``, ``kv_fork``, ``kv_reorder``) and of ``sample``.

Mirrors reference ``w4a16/cuda.py``: importing the compiled extension
(``nibble_amd._C``, here a thin libtorch shim over the HIP C ABI) registers
the ops; a missing extension is recorded, ``cuda_extension_available()``
reports it and the wrappers raise ``RuntimeError``. There is no fallback:
GPU tensors only ever run the HIP kernels. On PyTorch-ROCm "cuda" tensors
are HIP tensors, so the reference's names are kept.
"""

from __future__ import annotations

import importlib

import torch

try:
    importlib.import_module("nibble_amd._C")
except (ImportError, OSError) as error:
    _EXTENSION_LOAD_ERROR: Exception | None = error
else:
    _EXTENSION_LOAD_ERROR = None


if _EXTENSION_LOAD_ERROR is None:
    # Shape/dtype-only implementations so torch.compile can trace through the
    # ops with fake tensors (reference w4a16/cuda.py:14-36).
    @torch.library.register_fake("w4a16::linear")
    def _linear_fake(activations, packed_weights, scales, group_size):
        return activations.new_empty((activations.shape[0], packed_weights.shape[0]))

    @torch.library.register_fake("w4a16::dequantize")
    def _dequantize_fake(packed_weights, scales, group_size):
        return packed_weights.new_empty(
            (packed_weights.shape[0], packed_weights.shape[1] * 2), dtype=torch.float16
        )

    @torch.library.register_fake("w4a16::quantize")
    def _quantize_fake(weights, group_size):
        rows, cols = weights.shape
        return (
            weights.new_empty((rows, cols // 2), dtype=torch.uint8),
            weights.new_empty((rows, cols // group_size), dtype=torch.float16),
        )

    @torch.library.register_fake("w4a16::rotary")
    def _rotary_fake(x, positions, cos, sin, interleaved=False):
        return x.new_empty(x.shape)

    @torch.library.register_fake("w4a16::kv_write")
    def _kv_write_fake(k, v, k_codes, k_scales, v_codes, v_scales, start, counts=None):
        return None

    @torch.library.register_fake("w4a16::rotary_kv_write")
    def _rotary_kv_write_fake(q, k, v, cos, sin, k_codes, k_scales, v_codes, v_scales, start, counts=None,
                              interleaved=False):
        return q.new_empty(q.shape)

    @torch.library.register_fake("w4a16::kv_read")
    def _kv_read_fake(codes, scales, dtype):
        return codes.new_empty(codes.shape, dtype=dtype)

    @torch.library.register_fake("w4a16::kv_attention")
    def _kv_attention_fake(q, k_codes, k_scales, v_codes, v_scales, start, counts=None, scale=None):
        return q.new_empty(q.shape)


    @torch.library.register_fake("w4a16::kv_shared_attention")
    def _kv_shared_attention_fake(q, prefix_k_codes, prefix_k_scales, prefix_v_codes, prefix_v_scales, prefix_lengths,
                                  k_codes, k_scales, v_codes, v_scales, start, counts=None, scale=None):
        return q.new_empty(q.shape)

    @torch.library.register_fake("w4a16::kv_fork")
    def _kv_fork_fake(k_codes, k_scales, v_codes, v_scales, to_k_codes, to_k_scales, to_v_codes, to_v_scales, source,
                      lengths):
        return None

    @torch.library.register_fake("w4a16::kv_reorder")
    def _kv_reorder_fake(k_codes, k_scales, v_codes, v_scales, source, lengths):
        return None

    @torch.library.register_fake("w4a16::sample")
    def _sample_fake(logits, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, temperatures=None, top_ks=None,
                     top_ps=None, min_ps=None):
        return logits.new_empty((logits.shape[0],), dtype=torch.int64)


def cuda_extension_available() -> bool:
    """Whether the compiled W4A16 HIP extension is loaded."""
    return _EXTENSION_LOAD_ERROR is None


def extension_load_error() -> Exception | None:
    return _EXTENSION_LOAD_ERROR


def _require_extension() -> None:
    if _EXTENSION_LOAD_ERROR is not None:
        raise RuntimeError(
            "The W4A16 HIP extension is not built. Build it with "
            "`python -c 'import __graft_entry__ as g; g.build()'`."
        ) from _EXTENSION_LOAD_ERROR


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_transformed = torch._C._functorch.is_functorch_wrapped_tensor
_dispatch_modes = torch._C._len_torch_dispatch_stack


def addressable(*tensors: torch.Tensor) -> bool:
    """Whether a choice may look at where these tensors' memory starts: ordinary
    tensors of a call that runs now. False for a traced call (its graph also
    serves other tensors), under a dispatch mode, for a wrapper of
    ``torch.func`` and for a subclass, which may have no memory of their own."""
    if torch.compiler.is_compiling() or torch.jit.is_tracing() or _dispatch_modes():
        return False
    for tensor in tensors:
        if type(tensor) not in _PLAIN or _transformed(tensor):
            return False
    return True


def linear_cuda(
    activations: torch.Tensor,
    packed_weights: torch.Tensor,
    scales: torch.Tensor,
    group_size: int = 128,
) -> torch.Tensor:
    """Fused W4A16 linear on the GPU (reference ``w4a16/cuda.py:52-69``).

    group_size 128 with 16-byte aligned operands runs the tuned gfx950 kernels
    (up to 16 rows) and the W4A16 GEMM (above); group sizes 32 and 64 at M <= 8
    with K a multiple of 128 run their matrix-core kernel; anything else runs
    the scalar HIP kernel.
    """
    _require_extension()
    # the overload itself: naming the packet looks it up on every call (about 1 us)
    return torch.ops.w4a16.linear.default(activations, packed_weights, scales, group_size)


def dequantize_cuda(
    packed_weights: torch.Tensor,
    scales: torch.Tensor,
    group_size: int = 128,
) -> torch.Tensor:
    """Packed INT4 -> fp16 [N, K] in one pass (reference ``w4a16/cuda.py:72-83``).

    Bit-identical to ``dequantize_weights(...).to(torch.float16)``; needs
    group_size a multiple of 32 and 16-byte aligned packed weights.
    """
    _require_extension()
    return torch.ops.w4a16.dequantize(packed_weights, scales, group_size)


def quantize_cuda(weights: torch.Tensor, group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """fp16 / fp32 weights [N, K] -> (packed uint8 [N, K / 2], fp16 scales) in
    one pass, the bytes of ``quantize_and_pack_weights``; group_size a power of
    two from 16 to 512, weights contiguous and 16-byte aligned."""
    _require_extension()
    return torch.ops.w4a16.quantize(weights, group_size)


def rotary_cuda(
    x: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    interleaved: bool = False,
) -> torch.Tensor:
    """Rotary positions on the GPU: x fp16 / bf16 [tokens, heads, head_dim] or
    [batch, tokens, heads, head_dim] (any strides, the last dimension
    contiguous) with its first 2 * cos.shape[1] dims rotated by the rows
    ``positions`` (int64 [tokens] or [batch, tokens]) of the fp32 tables; the
    other dims are copied. Pairs are dims (i, i + half), or (2i, 2i + 1) when
    ``interleaved``. A position outside the tables gives NaN."""
    _require_extension()
    return torch.ops.w4a16.rotary.default(x, positions, cos, sin, interleaved)


def kv_write_cuda(
    k: torch.Tensor,
    v: torch.Tensor,
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    start: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> None:
    """Quantizes k and v fp16 / bf16 [batch, tokens, kv_heads, head_dim] into
    the slots start[b] .. of an 8-bit cache (codes int8 or float8_e4m3fn
    [batch, kv_heads, slots, head_dim], power-of-two scales fp32 [batch,
    kv_heads, blocks]; one scale for every 16, 32, 64 or 128 slots). The first
    counts[b] tokens of a sequence are written (None: all). A block's scale
    grows with its tokens, and its earlier codes are rescaled then."""
    _require_extension()
    torch.ops.w4a16.kv_write.default(k, v, k_codes, k_scales, v_codes, v_scales, start, counts)


def rotary_kv_write_cuda(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    start: torch.Tensor,
    counts: torch.Tensor | None = None,
    interleaved: bool = False,
) -> torch.Tensor:
    """``rotary_cuda`` of q and k at positions start[b] + t and
    ``kv_write_cuda`` of the rotated k and of v, in one launch; returns the
    rotated q (zeros in padding rows). The tables need a row for every slot and
    a rotated part that is a multiple of 16."""
    _require_extension()
    return torch.ops.w4a16.rotary_kv_write.default(q, k, v, cos, sin, k_codes, k_scales, v_codes, v_scales, start,
                                                   counts, interleaved)


def kv_read_cuda(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values code * scale of an 8-bit cache's keys or values (or of a view
    of its leading slots), rounded once to fp16, bf16 or fp32."""
    _require_extension()
    return torch.ops.w4a16.kv_read.default(codes, scales, dtype)


def kv_attention_cuda(
    q: torch.Tensor,
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    start: torch.Tensor,
    counts: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Causal attention of q fp16 / bf16 [batch, tokens, heads, head_dim] over
    an 8-bit cache that holds the tokens' own keys and values: token t of
    sequence b sees the slots 0 .. start[b] + t. Rows at or past counts[b] are
    padding and come out zero. ``scale`` defaults to head_dim ** -0.5."""
    _require_extension()
    return torch.ops.w4a16.kv_attention.default(q, k_codes, k_scales, v_codes, v_scales, start, counts, scale)


def kv_shared_attention_cuda(
    q: torch.Tensor,
    prefix_k_codes: torch.Tensor,
    prefix_k_scales: torch.Tensor,
    prefix_v_codes: torch.Tensor,
    prefix_v_scales: torch.Tensor,
    prefix_lengths: torch.Tensor,
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    start: torch.Tensor,
    counts: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """``kv_attention_cuda`` of a batch whose sequences share prefixes: a cache
    of G prefixes and one of the B sequences' own slots, B a multiple of G;
    token t of sequence b sees the slots 0 .. prefix_lengths[g] - 1 of prefix g
    = b // (B // G) and its own slots 0 .. start[b] + t. A prefix is read once
    for all of its sequences."""
    _require_extension()
    return torch.ops.w4a16.kv_shared_attention.default(
        q, prefix_k_codes, prefix_k_scales, prefix_v_codes, prefix_v_scales, prefix_lengths, k_codes, k_scales,
        v_codes, v_scales, start, counts, scale)


def kv_fork_cuda(
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    to_k_codes: torch.Tensor,
    to_k_scales: torch.Tensor,
    to_v_codes: torch.Tensor,
    to_v_scales: torch.Tensor,
    source: torch.Tensor,
    lengths: torch.Tensor,
) -> None:
    """Copies sequences of one 8-bit cache into another: sequence b of the
    second becomes what sequence source[b] of the first holds, lengths[source[b]]
    slots of it (int64 tensors); it stays as it is where source[b] is outside
    the first. The caches have the same KV heads, head_dim, block and codes and
    share no memory."""
    _require_extension()
    torch.ops.w4a16.kv_fork.default(k_codes, k_scales, v_codes, v_scales, to_k_codes, to_k_scales, to_v_codes,
                                    to_v_scales, source, lengths)


def kv_reorder_cuda(
    k_codes: torch.Tensor,
    k_scales: torch.Tensor,
    v_codes: torch.Tensor,
    v_scales: torch.Tensor,
    source: torch.Tensor,
    lengths: torch.Tensor,
) -> None:
    """The sequences of an 8-bit cache in another order, in place: every
    sequence b becomes what sequence source[b] held before, its first
    lengths[source[b]] slots (int64 [batch], the newest tokens' slots among
    them); one whose source is outside the batch stays as it is."""
    _require_extension()
    torch.ops.w4a16.kv_reorder.default(k_codes, k_scales, v_codes, v_scales, source, lengths)


def sample_cuda(
    logits: torch.Tensor,
    random: torch.Tensor,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> torch.Tensor:
    """A token (int64 [rows]) from each row of logits fp16, bf16 or fp32 [rows,
    vocabulary], drawn by the uniform numbers ``random`` (float32 [rows], in
    [0, 1)): temperature first (0: the largest logit), then the ``top_k`` most
    likely tokens (0: all), of those the most likely ones that hold ``top_p`` of
    the probability together (1: all), and of those the ones at least ``min_p``
    times as likely as the first. The token is the first by index at which the
    running sum of the kept probabilities exceeds ``random`` times their sum.
    Each setting is a number for all rows or a tensor with one a row (float32,
    ``top_k`` int64). At most 524288 logits a row."""
    _require_extension()
    single, rows = [], []
    for value, unset in ((temperature, 1.0), (top_k, 0), (top_p, 1.0), (min_p, 0.0)):
        tensor = isinstance(value, torch.Tensor)
        single.append(unset if tensor else value)
        rows.append(value if tensor else None)
    return torch.ops.w4a16.sample.default(logits, random, *single, *rows)
