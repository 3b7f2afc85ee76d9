"""The paged cache in 4 bits, beside the 16-bit one of :mod:`pageserve_amd.paged`.

A key or value costs 4.5 bits a dim instead of 16, so as much memory holds 3.5
times the tokens and a decoding step reads as much less.  The reference keeps its
cache in the model's type (engine/paged_attention.py:62-79); the rules are those
of the 4-bit weights (:mod:`pageserve_amd.quantization4`), per 32 neighbouring
dims of a token and key head:

    scale = max(absmax, 1e-8) / 6, cut to its first 6 significant bits, bf16
    code  = the one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 nearest to |x| / scale (a tie
            goes to the even code), with the sign of x

so that every value * scale is a bf16 number.  A group that holds an infinity or a
NaN gets it as its scale.  Block tables, slots, lengths and their calls are those
of the 16-bit cache.

Everything runs on the current stream of the tensors' device, asynchronously; CPU
tensors are refused.
"""

from __future__ import annotations

import torch

from . import _native
from .quantization import _DTYPE_CODE

__all__ = ["KVCache4", "write_kv4", "read_kv4"]


class KVCache4:
    """Keys and values of one layer in 4 bits: ``blocks`` blocks of ``block_size`` (a
    multiple of 16) tokens, head_dim 64 or 128.  A new one holds zeros.

    ``k`` and ``v`` (uint8 (blocks, kv_heads, block_size, head_dim / 2)) are the
    codes in the order that the kernels read them (include/pageserve_amd.h),
    ``k_scale`` and ``v_scale`` (bf16 (blocks, kv_heads, block_size, head_dim / 32))
    the scales in the dims' order.  :func:`write_kv4` and :func:`read_kv4` take and
    give rows in the usual one."""

    __slots__ = ("k", "k_scale", "v", "v_scale")

    def __init__(self, blocks: int, block_size: int, kv_heads: int, head_dim: int,
                 device: torch.device | str = "cuda"):
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if block_size < 16 or block_size % 16:
            raise ValueError(f"block_size must be a multiple of 16, got {block_size}")
        self.k, self.v = (torch.zeros((blocks, kv_heads, block_size, head_dim // 2), dtype=torch.uint8, device=device)
                          for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros((blocks, kv_heads, block_size, head_dim // 32), dtype=torch.bfloat16,
                                                  device=device) for _ in range(2))

    @classmethod
    def of(cls, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor, v_scale: torch.Tensor) -> "KVCache4":
        """A cache of these tensors (stored ones, parts of a larger buffer), as they are."""
        obj = cls.__new__(cls)
        obj.k, obj.k_scale, obj.v, obj.v_scale = k, k_scale, v, v_scale
        return obj

    @property
    def parts(self) -> list[torch.Tensor]:
        return [self.k, self.k_scale, self.v, self.v_scale]

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def storage_bytes(self) -> int:
        return sum(p.numel() * p.element_size() for p in self.parts)


def write_kv4(k: torch.Tensor, v: torch.Tensor, cache: KVCache4, slots: torch.Tensor) -> None:
    """Stores the rows of ``k`` and ``v`` (rows, kv_heads, head_dim), bf16 or fp16, in
    4 bits at their slots of the cache: :func:`write_kv`'s arguments and rules.  A row
    whose slot (int64) is outside the cache, as -1 is, is left out; no two rows may
    have the same slot."""
    _native.load_host().write_kv4(k, v, *cache.parts, slots)


def read_kv4(cache: KVCache4, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
             ) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows at ``slots`` (int64) back, ``(k, v)`` of shape (rows, kv_heads,
    head_dim): value * scale, exact in bf16 and fp32 (and in fp16 as far as its
    range reaches); zeros for a slot outside the cache."""
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    k, v = _native.load_host().read_kv4(*cache.parts, slots, _DTYPE_CODE[dtype])
    return k, v
