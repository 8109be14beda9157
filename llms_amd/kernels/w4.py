"""Projections on 4-bit weights with a scale for each group of inputs: the QKV,
gate-up-SiLU and plain ``down``/``o`` projections with their weights in a quarter
of the bf16 bytes, with or without the RMSNorm before them.

The reference has no such path (reference DESIGN.md:120 lists quantisation as future
work). The format is :func:`~llms_amd.kernels.quant.quantize_w4`'s: the weight is
exactly ``code * scale``, read in 4 bits at every row count and multiplied in the
matrix cores with fp32 sums (``llms_amd/csrc/fp_w4.hip``). Outputs are rounded once: the
gate-up product is of the fp32 sums, where the bf16 form rounds each of its steps.

Path: wrapper -> ``torch.ops.llms_amd.linear_w4`` / ``gate_up_silu_w4`` -> C ABI
``fp_linear_w4`` / ``fp_gate_up_silu_w4`` -> HIP kernels on torch's current stream.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._checks import inner_contiguous, refuse_grad, require_bf16_hip, require_device
from .fused_norm import _check_norm

GROUPS = (32, 64, 128)


def _check_w4(fn: str, x: torch.Tensor, q: torch.Tensor, s: torch.Tensor, group: int) -> None:
    K = x.shape[-1] if x.dim() else 0
    if group not in GROUPS:
        raise ValueError(f"{fn}: group must be one of {GROUPS}, got {group}")
    if q.dim() != 2 or q.shape[1] != (K + 1) // 2:
        raise ValueError(f"{fn}: q shape {tuple(q.shape)} does not hold (N, {(K + 1) // 2}) bytes of rows of {K}")
    if s.shape != (q.shape[0], -(-K // group)):
        raise ValueError(f"{fn}: s shape {tuple(s.shape)} != {(q.shape[0], -(-K // group))}")
    if q.dtype != torch.uint8 or s.dtype != torch.bfloat16:
        raise TypeError(f"{fn}: q must be uint8 and s bfloat16")
    if not (x.device == q.device == s.device):
        raise ValueError(f"x ({x.device}), q ({q.device}), s ({s.device}) must be on the same device")
    require_bf16_hip(fn, x=x)
    require_device(fn, q, "q")
    refuse_grad(fn, x, s)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [M, K] with unit inner stride and rows that do not share memory."""
    t = inner_contiguous(t)
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) < t.shape[1] else t


def _norm(fn: str, x: torch.Tensor, norm_weight: torch.Tensor, eps: float) -> torch.Tensor:
    _check_norm(x, norm_weight, eps, fn)
    refuse_grad(fn, norm_weight)
    return norm_weight.contiguous()


def _linear(fn, x, gamma, eps, q, s, group):
    _check_w4(fn, x, q, s, group)
    K = x.shape[-1]
    y = _lib.ops().linear_w4(_rows(x.reshape(-1, K)), gamma, float(eps), _rows(q), _rows(s), group)
    return y.reshape(*x.shape[:-1], q.shape[0])


def _gate_up(fn, x, gamma, eps, qg, sg, qu, su, group):
    if qg.shape != qu.shape:
        raise ValueError(f"{fn}: qg shape {tuple(qg.shape)} != qu shape {tuple(qu.shape)}")
    _check_w4(fn, x, qg, sg, group)
    _check_w4(fn, x, qu, su, group)
    K = x.shape[-1]
    y = _lib.ops().gate_up_silu_w4(_rows(x.reshape(-1, K)), gamma, float(eps), _rows(qg), _rows(sg),
                                   _rows(qu), _rows(su), group)
    return y.reshape(*x.shape[:-1], qg.shape[0])


def _check_split(fn, q, n_q, n_k):
    if q.dim() != 2 or n_q < 1 or n_k < 0 or n_q + 2 * n_k != q.shape[0]:
        raise ValueError(f"{fn}: n_q + 2*n_k ({n_q} + 2*{n_k} = {n_q + 2 * n_k}) != q.shape[0] ({q.shape[0]})")


def fused_linear_w4(x: torch.Tensor, q: torch.Tensor, s: torch.Tensor, *, group: int = 128) -> torch.Tensor:
    """``x @ W.T`` with ``W = code * s`` in 4 bits.

    Args:
        x: ``(..., K)`` bfloat16 on a HIP device.
        q, s: ``(N, ceil(K/2))`` uint8 and ``(N, ceil(K/group))`` bfloat16, of
            :func:`~llms_amd.kernels.quant.quantize_w4` with the same ``group``
            (32, 64 or 128).
    """
    return _linear("fused_linear_w4", x, None, 0.0, q, s, group)


def fused_qkv_w4(x: torch.Tensor, q_qkv: torch.Tensor, s_qkv: torch.Tensor, *, n_q: int, n_k: int,
                 group: int = 128):
    """``(q, k, v) = split(x @ W_qkv.T, [n_q, n_k, n_k])`` with W_qkv in 4 bits:
    views of one buffer."""
    _check_split("fused_qkv_w4", q_qkv, n_q, n_k)
    return _linear("fused_qkv_w4", x, None, 0.0, q_qkv, s_qkv, group).split([n_q, n_k, n_k], dim=-1)


def fused_gate_up_silu_w4(x: torch.Tensor, qg: torch.Tensor, sg: torch.Tensor, qu: torch.Tensor,
                          su: torch.Tensor, *, group: int = 128) -> torch.Tensor:
    """``silu(x @ Wg.T) * (x @ Wu.T)`` with both weights in 4 bits, rounded once."""
    return _gate_up("fused_gate_up_silu_w4", x, None, 0.0, qg, sg, qu, su, group)


def fused_rmsnorm_qkv_w4(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, q_qkv: torch.Tensor,
                         s_qkv: torch.Tensor, *, n_q: int, n_k: int, group: int = 128):
    """:func:`fused_qkv_w4` of ``RMSNorm(x)``."""
    fn = "fused_rmsnorm_qkv_w4"
    _check_split(fn, q_qkv, n_q, n_k)
    gamma = _norm(fn, x, norm_weight, eps)
    return _linear(fn, x, gamma, eps, q_qkv, s_qkv, group).split([n_q, n_k, n_k], dim=-1)


def fused_rmsnorm_gate_up_silu_w4(x: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                                  qg: torch.Tensor, sg: torch.Tensor, qu: torch.Tensor,
                                  su: torch.Tensor, *, group: int = 128) -> torch.Tensor:
    """:func:`fused_gate_up_silu_w4` of ``RMSNorm(x)``."""
    fn = "fused_rmsnorm_gate_up_silu_w4"
    return _gate_up(fn, x, _norm(fn, x, norm_weight, eps), eps, qg, sg, qu, su, group)
