"""4-bit weights with group scales, beside the 8-bit ones of
:mod:`pageserve_amd.quantization`.

Half the bytes of the 8-bit weight, for work that can bear the rounding: the
drafting pass of speculative decoding above all, whose tokens the full weights
verify.  The reference has no such form; the rules are its 8-bit ones
(engine/quantization.py:16-23: symmetric, absmax) per group of 32, 64 or 128
columns of a row:

    scale = bf16(max(absmax, 1e-8) / 6)
    code  = the one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 nearest to |w| / scale (a tie
            goes to the even code), with the sign of w

The sixteen values are those gfx950 widens to bf16 in hardware, exactly.

``QuantizedWeight4(weight, group)`` quantizes where the weight lives: on a GPU by
the HIP kernel, on the CPU by the same formula in torch, bit for bit the same.
:func:`linear4` takes GPU weights only.
"""

from __future__ import annotations

import torch

from . import _native
from .quantization import _DTYPE_CODE

__all__ = ["QuantizedWeight4", "linear4"]

GROUPS = (32, 64, 128)
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _check_shape(shape, group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group must be 32, 64 or 128, got {group}")
    if len(shape) != 2:
        raise ValueError("weight must be a 2-D tensor (out_features, in_features)")
    if shape[1] % 16:
        raise ValueError(f"in_features must be a multiple of 16, got {shape[1]}")


def _blocks(n: int, k: int) -> tuple[int, int]:
    return -(-n // 16), -(-k // 128)


def _pack(codes: torch.Tensor, scale: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Row-major codes (uint8 [n, k]) and scales (bf16 [n, groups]) -> the packed
    layout of the kernels (include/pageserve_amd.h), on their device."""
    n, k = codes.shape
    tn, tk = _blocks(n, k)
    s = 128 // group
    c = torch.zeros((tn * 16, tk * 128), dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes
    # [tile, row, block, dword, column eighth of the dword's 32, byte, nibble]
    c = c.view(tn, 16, tk, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
    qp = (c[..., 0] | (c[..., 1] << 4)).contiguous().view(-1)
    p = torch.zeros((tn * 16, tk * s), dtype=torch.bfloat16, device=scale.device)
    p[:n, :scale.shape[1]] = scale
    sp = p.view(tn, 16, tk, s).transpose(1, 2).contiguous().view(-1)
    return qp, sp


def _cpu_quantize4(weight: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = weight.shape
    w = torch.nn.functional.pad(weight.float(), (0, -k % group)).view(n, -(-k // group), group)
    a = w.abs()
    scale = (a.amax(2, keepdim=True).clamp(min=1e-8) / 6.0).to(torch.bfloat16) if k else a.new_zeros(n, 0, 1).bfloat16()
    s = scale.float()
    code = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s)
            + (a >= 3.5 * s) + (a > 5.0 * s))
    code = code + 8 * ((w < 0) & (code > 0)).to(torch.uint8)
    return code.flatten(1)[:, :k], scale.squeeze(2)


class QuantizedWeight4:
    """A weight stored as 4-bit codes with one bf16 scale per ``group`` columns.

    ``qp`` (uint8, half a byte per weight) and ``sp`` (bf16) are the packed codes
    and scales that :func:`linear4` streams, padded with zeros to 16 rows x 128
    columns; :attr:`codes` and :attr:`scale` are their row-major forms, rebuilt on
    access; :meth:`dense` is the dequantized weight in the weight's dtype."""

    def __init__(self, weight: torch.Tensor, group: int = 128):
        if not isinstance(weight, torch.Tensor):
            raise TypeError("weight must be a torch.Tensor")
        _check_shape(weight.shape, group)
        self.dtype, self.shape, self.group = weight.dtype, torch.Size(weight.shape), group
        weight = weight.detach()
        if not weight.is_cuda:
            self.qp, self.sp = _pack(*_cpu_quantize4(weight, group), group)
            return
        w = weight if weight.dtype in (torch.float32, torch.bfloat16) else weight.float()
        self.qp, self.sp = _native.load_host().quantize4(w, group)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, group: int,
                   dtype: torch.dtype = torch.bfloat16) -> "QuantizedWeight4":
        """A weight from row-major codes (any integer type, [out_features, in_features],
        0..15: the value's index, plus 8 for a negative one; of others the low four bits
        count) and scales (bf16 [out_features, ceil(in_features / group)])."""
        if codes.is_floating_point() or codes.is_complex() or codes.dtype is torch.bool:
            raise TypeError(f"codes must be of an integer type, got {codes.dtype}")
        if scale.dtype != torch.bfloat16:
            raise TypeError(f"scale must be bf16, got {scale.dtype}")
        _check_shape(codes.shape, group)
        n, k = codes.shape
        if tuple(scale.shape) != (n, -(-k // group)) or scale.device != codes.device:
            raise ValueError(f"scale must be [{n}, {-(-k // group)}] on {codes.device}")
        obj = cls.__new__(cls)
        obj.dtype, obj.shape, obj.group = dtype, torch.Size(codes.shape), group
        obj.qp, obj.sp = _pack(codes.to(torch.uint8) & 15, scale.detach(), group)
        return obj

    @property
    def device(self) -> torch.device:
        return self.qp.device

    @property
    def codes(self) -> torch.Tensor:
        n, k = self.shape
        tn, tk = _blocks(n, k)
        b = self.qp.view(tn, tk, 4, 16, 4, 4)
        c = torch.stack((b & 15, b >> 4), -1).permute(0, 3, 1, 4, 2, 5, 6)
        return c.reshape(tn * 16, tk * 128)[:n, :k].contiguous()

    @property
    def scale(self) -> torch.Tensor:
        n, k = self.shape
        tn, tk = _blocks(n, k)
        s = 128 // self.group
        p = self.sp.view(tn, tk, 16, s).transpose(1, 2).reshape(tn * 16, tk * s)
        return p[:n, :-(-k // self.group)].contiguous()

    def to(self, device) -> "QuantizedWeight4":
        self.qp, self.sp = self.qp.to(device), self.sp.to(device)
        return self

    @property
    def storage_bytes(self) -> int:
        return self.qp.numel() + 2 * self.sp.numel()

    def dense(self) -> torch.Tensor:
        """value * scale (exact in fp32), rounded once to the weight's dtype."""
        n, k = self.shape
        if not self.qp.is_cuda:
            value = torch.tensor(VALUES + tuple(-v for v in VALUES))
            per = self.scale.float().repeat_interleave(self.group, 1)[:, :k]
            return (value[self.codes.long()] * per).to(self.dtype)
        kdt = self.dtype if self.dtype in _DTYPE_CODE else torch.float32
        out = _native.load_host().dequantize4(self.qp, self.sp, n, k, self.group, _DTYPE_CODE[kdt])
        return out if kdt == self.dtype else out.to(self.dtype)

    def linear(self, x: torch.Tensor, bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
               residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        return linear4(x, self, bias, out_dtype=out_dtype, residual=residual, out=out)


def linear4(x: torch.Tensor, weight: QuantizedWeight4, bias: torch.Tensor | None = None,
            out_dtype: torch.dtype = torch.bfloat16, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` with a 4-bit weight: the arguments and results
    of :func:`pageserve_amd.linear`.  x: bf16 [..., in_features] on the weight's
    GPU; the codes are widened exactly and a group's fp32 sum is multiplied by
    its scale, so the only rounding is the output's.  Made for a few tokens: above
    64 the weight is read once per 64."""
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
    if not weight.qp.is_cuda:
        raise RuntimeError("linear4: the weight must be on a ROCm GPU (call .to('cuda') first)")
    n, k = weight.shape
    return _native.load_host().linear4(x, weight.qp, weight.sp, bias, n, k, weight.group,
                                       out_dtype is torch.float32, residual, out)
