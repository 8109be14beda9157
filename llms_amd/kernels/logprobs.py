"""Log-probabilities of given tokens, the entropy and the most likely tokens of
every row of logits: what scoring a text, accepting a draft or showing
alternatives reads from a model's answer.

The reference reads its logits with torch (``log_softmax`` and ``topk``, several
passes over fp32 copies). Here one pass over the logits as they are keeps the
running sums and the top tokens (``llms_amd/csrc/fp_logprob.hip``).

Path: wrapper -> ``torch.ops.llms_amd.token_logprobs`` -> C ABI
``fp_token_logprobs`` -> HIP kernels on torch's current stream.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ._checks import inner_contiguous, refuse_grad

MAX_TOP_K = 64
MAX_VOCAB = 1 << 20


class TokenLogprobs(NamedTuple):
    """``logprob``, ``entropy`` float32 of the rows' shape; ``top_ids`` (int64)
    and ``top_logprobs`` (float32) with one more dimension of ``top_k``."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """``log_softmax(logits)`` at ``tokens``, its entropy and its ``top_k`` largest.

    Args:
        logits: ``(..., V)`` bfloat16, float16 or float32 on a HIP device, V up to 2^20.
        tokens: ``(...)`` int64. A negative token asks for none and has
            ``logprob`` 0; one of V or more has NaN.
        top_k: how many of the most likely tokens to return, up to 64 (ties go
            to the lowest token).

    Everything is summed in float32. Logits of -inf (masked tokens) have
    probability 0 and add nothing to the entropy; a row with a NaN or +inf, or of
    nothing but -inf, has NaN for both.
    """
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(
            f"tokens shape {tuple(tokens.shape)} != logits shape {tuple(logits.shape)} without its last dim"
        )
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"token_logprobs: logits must be bfloat16, float16 or float32, got {logits.dtype}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"token_logprobs: tokens must be int64, got {tokens.dtype}")
    V = logits.shape[-1]
    if not 0 <= top_k <= min(V, MAX_TOP_K):
        raise ValueError(f"token_logprobs: top_k must be 0 to {min(V, MAX_TOP_K)}, got {top_k}")
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"token_logprobs: rows of 1 to {MAX_VOCAB} logits are taken, got {V}")
    if logits.device.type != "cuda":
        raise ValueError(f"token_logprobs: logits is on {logits.device}; it runs only on a HIP (ROCm) device")
    if tokens.device != logits.device:
        raise ValueError(f"logits ({logits.device}) and tokens ({tokens.device}) must be on the same device")
    refuse_grad("token_logprobs", logits)
    lead = logits.shape[:-1]
    x = inner_contiguous(logits.reshape(-1, V))
    if x.shape[0] > 1 and x.stride(0) < V:  # rows that share memory (an expanded view)
        x = x.contiguous()
    lp, h, ids, top = _lib.ops().token_logprobs(x, tokens.reshape(-1).contiguous(), top_k)
    if len(lead) == 1:
        return TokenLogprobs(lp, h, ids, top)
    return TokenLogprobs(lp.reshape(lead), h.reshape(lead), ids.reshape(*lead, top_k),
                         top.reshape(*lead, top_k))
