"""Weight packing, the swap-time step of the low-bit projections: per-output-channel
symmetric int8, and 4 bits with a scale for each group of inputs.

The reference has no int8 path (reference DESIGN.md:120 lists quantisation as future
work); the format is this build's: for each output row r of an ``[N, K]``
weight, ``s[r] = max_k |W[r, k]| / 127`` in fp32 and
``q[r, k] = clamp(rint(W[r, k] / s[r]), -127, 127)`` as int8 (ties to even;
rows that are all zero get ``s = 0, q = 0``). The kernels compute with the
dequantised weight ``bf16(fp32(q * s))``.

4 bits: for each group of 32, 64 or 128 inputs of a row, ``s`` is ``max |W| / 7``
rounded to five significant bits (ties to even) and ``code = rint(W / s)`` in -7 ..
7. bf16 holds ``code * s`` exactly, so the weight the kernels compute with is that
product itself. ``q`` packs two codes a byte, ``code + 8`` of inputs 2j (low half)
and 2j + 1; a group with an infinity or a NaN has the scale NaN.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._checks import inner_contiguous, require_bf16_hip


def quantize_w8_per_row(W: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantise a bf16 ``[N, K]`` weight on its HIP device.

    Returns ``(q, s)``: int8 ``[N, K]`` (contiguous) and fp32 ``[N]``.
    """
    if W.dim() != 2:
        raise ValueError(f"W must be 2D (N, K), got shape {tuple(W.shape)}")
    require_bf16_hip("quantize_w8_per_row", W=W)
    q, s = _lib.ops().quantize_w8(inner_contiguous(W))
    return q, s


def dequantize_w8(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """``bf16(q.float() * s[:, None])``: the weight the int8 kernels compute
    with (a torch expression, for inspection; not used by the kernels)."""
    return (q.float() * s[:, None]).to(torch.bfloat16)


def quantize_w4(W: torch.Tensor, group: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack a bf16 ``[N, K]`` weight in 4 bits on its HIP device.

    Returns ``(q, s)``: uint8 ``[N, ceil(K/2)]`` and bfloat16 ``[N, ceil(K/group)]``.
    """
    return _lib.ops().quantize_w4(W.detach(), group)  # which checks them


def dequantize_w4(q: torch.Tensor, s: torch.Tensor, K: int, *, group: int = 128) -> torch.Tensor:
    """The bf16 ``[N, K]`` weight that ``(q, s)`` stand for (exact; a torch
    expression, for inspection)."""
    code = torch.stack([q & 15, q >> 4], dim=2).reshape(q.shape[0], -1)[:, :K].float() - 8
    return (code * s.float().repeat_interleave(group, dim=1)[:, :K]).to(torch.bfloat16)


def pack_weight(W: torch.Tensor, w4_group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, s)`` of a module's weight: 4 bits in groups of ``w4_group``, or int8
    per row with 0."""
    return quantize_w4(W, w4_group) if w4_group else quantize_w8_per_row(W)
