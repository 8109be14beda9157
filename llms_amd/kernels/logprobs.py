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
from ._checks import refuse_grad


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
    refuse_grad("token_logprobs", logits)
    return TokenLogprobs(*_lib.ops().token_logprobs(logits, tokens, top_k))  # which checks the rest
