"""``QuantizedKVCache``: a static key/value cache in 8 bits.

Codes are int8 or e4m3 (``dtype`` "int8" / "fp8"), one byte a value, with a
power-of-two fp32 scale for each ``block_size`` slots of a sequence's KV head.
int8 keeps an absolute step per block (at least 1/127 of its largest value and
less than 2/127), e4m3 a relative one (2^-3). Half of the bytes of an fp16
cache, so half of what a decode step reads of it.

GPU tensors run the HIP kernels (``torch.ops.w4a16.kv_write`` and so on; head
dims 64, 128 and 256) and raise without the extension; CPU tensors run the same
operators in torch operations.

    cache = QuantizedKVCache(batch, kv_heads, max_seq_len, head_dim, dtype="int8")
    q = cache.rotary_write(q, k, v, cos, sin, start)   # or cache.write(k, v, start)
    out = cache.attend(q, start)
"""

from __future__ import annotations

import torch

from nibble_amd import kv_reference
from nibble_amd.cuda import kv_attention_cuda, kv_read_cuda, kv_write_cuda, rotary_kv_write_cuda

CODE_TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


class QuantizedKVCache:
    """Keys and values [batch, kv_heads, max_seq_len, head_dim] of one layer."""

    def __init__(
        self,
        batch: int,
        kv_heads: int,
        max_seq_len: int,
        head_dim: int,
        dtype: str = "int8",
        block_size: int = 64,
        device: torch.device | str | None = None,
    ) -> None:
        if dtype not in CODE_TYPES:
            raise ValueError("dtype must be 'int8' or 'fp8'")
        if min(batch, kv_heads, max_seq_len, head_dim) <= 0:
            raise ValueError("batch, kv_heads, max_seq_len and head_dim must be greater than zero")
        if block_size not in (16, 32, 64, 128):
            raise ValueError("block_size must be 16, 32, 64 or 128")
        shape = (batch, kv_heads, max_seq_len, head_dim)
        blocks = (batch, kv_heads, -(-max_seq_len // block_size))
        self.k_codes = torch.zeros(shape, dtype=CODE_TYPES[dtype], device=device)
        self.v_codes = torch.zeros(shape, dtype=CODE_TYPES[dtype], device=device)
        smallest = 2.0 ** kv_reference.LOWEST   # an empty block imposes nothing on its first tokens
        self.k_scales = torch.full(blocks, smallest, dtype=torch.float32, device=device)
        self.v_scales = torch.full(blocks, smallest, dtype=torch.float32, device=device)
        self.block_size = block_size

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """(k_codes, k_scales, v_codes, v_scales)."""
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors())

    def write(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """k, v fp16 / bf16 [batch, tokens, kv_heads, head_dim] into the slots
        start[b] .. (int64 [batch]); the first counts[b] tokens, or all. Slots
        behind them are taken to be free."""
        call = kv_write_cuda if self.k_codes.is_cuda else kv_reference.kv_write_reference
        call(k, v, *self.tensors(), start, counts)

    def rotary_write(
        self,
        q: torch.Tensor,
        k: torch.Tensor,
        v: torch.Tensor,
        cos: torch.Tensor,
        sin: torch.Tensor,
        start: torch.Tensor,
        counts: torch.Tensor | None = None,
        interleaved: bool = False,
    ) -> torch.Tensor:
        """Rotates q and k at positions start[b] + t, writes k and v; returns the rotated q."""
        call = rotary_kv_write_cuda if self.k_codes.is_cuda else kv_reference.rotary_kv_write_reference
        return call(q, k, v, cos, sin, *self.tensors(), start, counts, interleaved)

    def attend(
        self,
        q: torch.Tensor,
        start: torch.Tensor,
        counts: torch.Tensor | None = None,
        scale: float | None = None,
    ) -> torch.Tensor:
        """Causal attention of q [batch, tokens, heads, head_dim] at positions
        start[b] + t over the cache, which holds the tokens already."""
        call = kv_attention_cuda if self.k_codes.is_cuda else kv_reference.kv_attention_reference
        return call(q, *self.tensors(), start, counts, scale)

    def read(self, slots: int | None = None, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [batch, kv_heads, slots, head_dim] of the first
        ``slots`` slots (None: all) as fp16, bf16 or fp32."""
        held = self.k_codes.shape[2]
        slots = held if slots is None else slots
        if not 0 <= slots <= held:
            raise ValueError("slots must be between 0 and max_seq_len")
        if slots == 0:
            shape = (*self.k_codes.shape[:2], 0, self.k_codes.shape[3])
            return (torch.empty(shape, dtype=dtype, device=self.k_codes.device),
                    torch.empty(shape, dtype=dtype, device=self.k_codes.device))
        blocks = -(-slots // self.block_size)
        call = kv_read_cuda if self.k_codes.is_cuda else kv_reference.kv_read_reference
        return (call(self.k_codes[:, :, :slots], self.k_scales[:, :, :blocks], dtype),
                call(self.v_codes[:, :, :slots], self.v_scales[:, :, :blocks], dtype))
