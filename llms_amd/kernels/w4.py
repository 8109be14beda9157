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
from ._checks import refuse_grad


def _linear(x, gamma, eps, q, s, group, fn):
    refuse_grad(fn, x, s) if gamma is None else refuse_grad(fn, x, s, gamma)
    return _lib.ops().linear_w4(x, gamma, eps, q, s, group)  # which checks the rest


def _gate_up(x, gamma, eps, qg, sg, qu, su, group, fn):
    refuse_grad(fn, x, sg, su) if gamma is None else refuse_grad(fn, x, sg, su, gamma)
    return _lib.ops().gate_up_silu_w4(x, gamma, eps, qg, sg, qu, su, group)


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
    return _linear(x, None, 0.0, q, s, group, "fused_linear_w4")


def fused_qkv_w4(x: torch.Tensor, q_qkv: torch.Tensor, s_qkv: torch.Tensor, *, n_q: int, n_k: int,
                 group: int = 128):
    """``(q, k, v) = split(x @ W_qkv.T, [n_q, n_k, n_k])`` with W_qkv in 4 bits:
    views of one buffer."""
    _check_split("fused_qkv_w4", q_qkv, n_q, n_k)
    return _linear(x, None, 0.0, q_qkv, s_qkv, group, "fused_qkv_w4").split_with_sizes((n_q, n_k, n_k), -1)


def fused_gate_up_silu_w4(x: torch.Tensor, qg: torch.Tensor, sg: torch.Tensor, qu: torch.Tensor,
                          su: torch.Tensor, *, group: int = 128) -> torch.Tensor:
    """``silu(x @ Wg.T) * (x @ Wu.T)`` with both weights in 4 bits, rounded once."""
    return _gate_up(x, None, 0.0, qg, sg, qu, su, group, "fused_gate_up_silu_w4")


def fused_rmsnorm_qkv_w4(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, q_qkv: torch.Tensor,
                         s_qkv: torch.Tensor, *, n_q: int, n_k: int, group: int = 128):
    """:func:`fused_qkv_w4` of ``RMSNorm(x)``."""
    fn = "fused_rmsnorm_qkv_w4"
    _check_split(fn, q_qkv, n_q, n_k)
    return _linear(x, norm_weight, eps, q_qkv, s_qkv, group, fn).split_with_sizes((n_q, n_k, n_k), -1)


def fused_rmsnorm_gate_up_silu_w4(x: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                                  qg: torch.Tensor, sg: torch.Tensor, qu: torch.Tensor,
                                  su: torch.Tensor, *, group: int = 128) -> torch.Tensor:
    """:func:`fused_gate_up_silu_w4` of ``RMSNorm(x)``."""
    return _gate_up(x, norm_weight, eps, qg, sg, qu, su, group, "fused_rmsnorm_gate_up_silu_w4")
