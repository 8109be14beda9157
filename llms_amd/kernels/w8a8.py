"""Projections in 8-bit integers: the QKV, gate-up-SiLU and plain ``down``/``o``
projections on int8 weights with a scale for each output, with their tokens quantised to
8 bits on the way in (a scale for each token), with or without the RMSNorm before them.

The reference has no such path (reference DESIGN.md:120 lists quantisation as future
work). The weights are :func:`~llms_amd.kernels.quant.quantize_w8_per_row`'s, as the
weight-only int8 projections take them; those turn them into bf16 in every call, here
they meet the tokens' codes in the integer matrix cores (``llms_amd/csrc/fp_w8a8.hip``). Of a token with
``top = max|x|`` the codes are ``round(127 x / top)`` (ties to even) and the scale is
``top / 127``; sums of codes are exact, so an output is rounded once, whatever the other
tokens of the call are. A token with an infinity or a NaN has NaN outputs.

Path: wrapper -> ``torch.ops.llms_amd.linear_w8a8`` / ``gate_up_silu_w8a8`` -> C ABI
``fp_linear_w8a8`` / ``fp_gate_up_silu_w8a8`` -> HIP kernels on torch's current stream.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._checks import refuse_grad
from .w4 import _check_split


def _linear(x, gamma, eps, q, s, fn):
    refuse_grad(fn, x, s) if gamma is None else refuse_grad(fn, x, s, gamma)
    return _lib.ops().linear_w8a8(x, gamma, eps, q, s)  # which checks the rest


def _gate_up(x, gamma, eps, qg, sg, qu, su, fn):
    refuse_grad(fn, x, sg, su) if gamma is None else refuse_grad(fn, x, sg, su, gamma)
    return _lib.ops().gate_up_silu_w8a8(x, gamma, eps, qg, sg, qu, su)


def fused_linear_w8a8(x: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """``x8 @ (q * s[:, None]).T`` with ``x8`` the tokens of ``x`` in 8 bits.

    Args:
        x: ``(..., K)`` bfloat16 on a HIP device, K up to 2^17.
        q, s: ``(N, K)`` int8 and ``(N,)`` float32, of
            :func:`~llms_amd.kernels.quant.quantize_w8_per_row`.
    """
    return _linear(x, None, 0.0, q, s, "fused_linear_w8a8")


def fused_qkv_w8a8(x: torch.Tensor, q_qkv: torch.Tensor, s_qkv: torch.Tensor, *, n_q: int, n_k: int):
    """``(q, k, v) = split(x8 @ W_qkv.T, [n_q, n_k, n_k])`` with W_qkv in 8 bits: views of one
    buffer."""
    _check_split("fused_qkv_w8a8", q_qkv, n_q, n_k)
    return _linear(x, None, 0.0, q_qkv, s_qkv, "fused_qkv_w8a8").split_with_sizes((n_q, n_k, n_k), -1)


def fused_gate_up_silu_w8a8(x: torch.Tensor, qg: torch.Tensor, sg: torch.Tensor, qu: torch.Tensor,
                            su: torch.Tensor) -> torch.Tensor:
    """``silu(x8 @ Wg.T) * (x8 @ Wu.T)`` with both weights in 8 bits, rounded once."""
    return _gate_up(x, None, 0.0, qg, sg, qu, su, "fused_gate_up_silu_w8a8")


def fused_rmsnorm_qkv_w8a8(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, q_qkv: torch.Tensor,
                           s_qkv: torch.Tensor, *, n_q: int, n_k: int):
    """:func:`fused_qkv_w8a8` of ``RMSNorm(x)``."""
    fn = "fused_rmsnorm_qkv_w8a8"
    _check_split(fn, q_qkv, n_q, n_k)
    return _linear(x, norm_weight, eps, q_qkv, s_qkv, fn).split_with_sizes((n_q, n_k, n_k), -1)


def fused_rmsnorm_gate_up_silu_w8a8(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, qg: torch.Tensor,
                                    sg: torch.Tensor, qu: torch.Tensor, su: torch.Tensor) -> torch.Tensor:
    """:func:`fused_gate_up_silu_w8a8` of ``RMSNorm(x)``."""
    return _gate_up(x, norm_weight, eps, qg, sg, qu, su, "fused_rmsnorm_gate_up_silu_w8a8")
