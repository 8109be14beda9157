"""A key/value cache in 8 bits with one scale for each block of 64 tokens and head,
and causal attention over it: half the cache bytes of a bf16 decode step.

The reference's cache is bf16 (``src/engine/kv_cache.py:19-47``). Here a block is packed
once, from its bf16 tokens, when its last token arrives; the tokens of the
unfinished block (and of the one before it) are kept in bf16. What the cache holds
therefore does not depend on how its tokens were cut into calls, and a
verify step that takes back a few tokens finds them unpacked. Going further back,
to any position, works too: the block it lands in goes on from its packed values.

What a call answers does depend on the cut. Attention reads the cache as it is after
the call's write, so a block that the call completes is read in 8 bits by all of the
call's rows, those before its end included, and its scale is the largest entry of all 64
tokens: such a row depends, within the rounding of 8 bits, on up to 63 tokens behind it.
Where a row must not (scoring a text, drafts that may be rejected), no token but a call's
last may end a block: calls of one token, or calls cut before and behind each block's last
token (``teacher_forced_logprobs(kv8=True, causal=True)`` does that).

Path: wrapper -> ``torch.ops.llms_amd.attention_kv8`` / ``write_kv8`` /
``read_kv8`` -> C ABI ``fp_kv8_attention`` / ``fp_kv8_write`` / ``fp_kv8_read`` -> HIP
kernels (``llms_amd/csrc/fp_kv8.hip``) on torch's current stream.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ._checks import autocast, plain_norm, refuse_grad, transformed

BLOCK = 64
MAX_SEQ = 1 << 23


class KVCache8:
    """The 8-bit caches of a model's layers, for up to ``max_batch`` sequences of
    up to ``max_seq`` tokens (the counterpart of the harness's ``KVCache``).

    ``cur_len`` is the model's count of tokens, as in ``KVCache``. Tokens are
    written in order: a call may start anywhere up to the tokens written so far (what
    is behind it is dropped), not later (the unfinished block would be lost).
    A key or value that is not finite is held as NaN: it spoils the rows that see the key,
    and the value's column in the rows that its block is read for (0 * NaN, as torch's
    product would, before its position too). Calls on one cache must be ordered
    (one stream, or streams that wait for each other).
    """

    def __init__(self, layers: list, max_batch: int, n_kv_heads: int, head_dim: int, max_seq: int) -> None:
        self.layers = layers  # a buffer of bytes each (see parts)
        self.max_batch, self.n_kv_heads, self.head_dim, self.max_seq = max_batch, n_kv_heads, head_dim, max_seq
        self.size = (max_batch, n_kv_heads, head_dim, max_seq)
        self.cur_len = 0

    @classmethod
    def alloc(cls, num_layers: int, max_seq: int, *, max_batch: int = 1, n_kv_heads: int, head_dim: int,
              device) -> "KVCache8":
        if num_layers < 1 or max_batch < 1 or n_kv_heads < 1:
            raise ValueError(f"KVCache8: num_layers, max_batch and n_kv_heads must be at least 1, got "
                             f"{num_layers}, {max_batch}, {n_kv_heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"KVCache8: heads of 64 or 128 are taken, got {head_dim}")
        if not 1 <= max_seq <= MAX_SEQ:
            raise ValueError(f"KVCache8: max_seq must be 1 to {MAX_SEQ}, got {max_seq}")
        size = max_batch, n_kv_heads, head_dim, max_seq
        n = _lib.ops().kv8_layout(*size)[-1]
        c = cls([torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(num_layers)], *size)
        for i in range(num_layers):
            c.parts(i)[-1].fill_(-1)
        return c

    def parts(self, layer: int) -> list:
        """A layer's codes of keys ``[max_batch, heads, blocks, 64, D]`` and values (``.., D, 64``),
        their scales, the bf16 tails of keys ``[.., 2, 64, D]`` and values (``.., D, 64``) and the
        blocks in the tails ``[.., 2]``: views of its buffer."""
        lead, D, nb = (self.max_batch, self.n_kv_heads), self.head_dim, -(-self.max_seq // BLOCK)
        shapes = [(nb, BLOCK, D), (nb, D, BLOCK), (nb,), (nb,), (2, BLOCK, D), (2, D, BLOCK), (2,)]
        types = [torch.int8] * 2 + [torch.float32] * 2 + [torch.bfloat16] * 2 + [torch.int32]
        out = []
        for at, shape, t in zip(_lib.ops().kv8_layout(*self.size), shapes, types):
            n = math.prod(lead + shape) * t.itemsize
            out.append(self.layers[layer][at : at + n].view(t).view(*lead, *shape))
        return out

    @property
    def device(self) -> torch.device:
        return self.layers[0].device

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, start_pos, *, lengths=None) -> None:
        """Put ``k``, ``v`` ``[B, T, n_kv_heads, D]`` (bfloat16, normalised and rotated)
        at positions ``start_pos ..``; arguments as in :func:`attention_kv8`."""
        start, pos = _place("KVCache8.write", start_pos, lengths)
        refuse_grad("KVCache8.write", k, v)
        _lib.ops().write_kv8(k, v, self.layers[layer], self.size, start, pos, lengths)  # which checks the rest

    def read(self, layer: int, start_pos, T: int, *, batch: int | None = None):
        """The keys and values ``[B, T, n_kv_heads, D]`` in float32 that attention sees at
        positions ``start_pos .. start_pos + T - 1`` of sequences that end there (with
        ``start_pos`` 0 and ``T`` the length: all). B is ``batch``, the number of
        positions in ``start_pos [B]``, or ``max_batch``."""
        if batch is None:
            batch = start_pos.shape[0] if torch.is_tensor(start_pos) and start_pos.dim() == 1 else self.max_batch
        if not 1 <= batch <= self.max_batch or T < 1:
            raise ValueError(f"KVCache8.read: batch {batch} and T {T} must be 1 to {self.max_batch} and at least 1")
        start, pos = _place("KVCache8.read", start_pos, None)
        return _lib.ops().read_kv8(self.layers[layer], self.size, batch, T, start, pos)

    def tails(self) -> list:
        """The buffers of every layer that a write outside the sequence would lose."""
        at = _lib.ops().kv8_layout(*self.size)[4]
        return [c[at:] for c in self.layers]


def _place(fn: str, start_pos, lengths):
    """(start_pos as an int, as a tensor or None)."""
    if lengths is not None and not torch.is_tensor(lengths):
        raise ValueError(f"{fn}: lengths must be an int64 tensor, got {type(lengths).__name__}")
    if torch.is_tensor(start_pos):
        return 0, start_pos
    if type(start_pos) is not int:
        raise TypeError(f"{fn}: start_pos must be an int or an int64 tensor, got {type(start_pos).__name__}")
    return start_pos, None


def attention_kv8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KVCache8, layer: int, start_pos,
                  *, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Write the new keys and values into ``cache`` and attend over it.

    Args:
        q: ``[B, T, heads, D]`` bfloat16 on the cache's device; k, v:
            ``[B, T, n_kv_heads, D]``; normalised and rotated. D is 64 or 128, heads a
            multiple of ``n_kv_heads``.
        start_pos: the position of token 0: an int, or an int64 tensor on the device, 0-dim
            or ``[B]`` for sequences of different lengths (a call captured in a
            HIP graph replays at any positions).
        lengths: how many of the T tokens each sequence has (int64 ``[B]`` on the
            device, default T): the others are not written.

    Returns:
        ``[B, T, heads, D]`` bfloat16: softmax attention with scale ``D ** -0.5`` of the token
        at position p over positions 0 .. p, as the cache holds them after the write: in
        8 bits where this call's tokens end their block, whose scale later tokens of the
        block take part in (see the module's head for calls where that must not be). Rows
        past a sequence's length, and at device positions outside the cache (whose tokens
        are not written), are zero.
    """
    fn = "attention_kv8"
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{fn}: q {tuple(q.shape)} and k {tuple(k.shape)} must be (B, T, heads, {cache.head_dim})")
    start, pos = _place(fn, start_pos, lengths)
    refuse_grad(fn, q, k, v)
    return _lib.ops().attention_kv8(q, k, v, None, None, 0.0, 0.0, None, None, cache.layers[layer], cache.size,
                                    start, pos, lengths)  # which checks the rest


def attention_core_kv8(q, k, v, *, q_norm, k_norm, num_heads: int, cache: KVCache8, layer: int, cos, sin,
                       start_pos) -> torch.Tensor:
    """What ``TritonAttention.forward`` does between its projections with an 8-bit
    cache: QK-norm and RoPE of the flat projections ``[B, T, heads * D]`` in the
    kernel that writes the keys (in torch where a norm is not the plain one, a type is not
    bf16's or rows of cos and sin share memory), the cache write and attention. Returns
    ``[B, T, num_heads * D]``."""
    fn, D = "attention_kv8", cache.head_dim
    B, T, _ = q.shape
    fused = (plain_norm(q_norm) and plain_norm(k_norm) and not autocast()
             and all(t.dtype == torch.bfloat16 and t.shape == (D,) and t.is_contiguous() and t.data_ptr() % 8 == 0
                     for t in (q_norm.weight, k_norm.weight))
             and all(t.dtype == torch.bfloat16 and t.shape == (T, D) and t.stride(1) == 1 and t.device == q.device
                     and (T == 1 or t.stride(0) >= D) for t in (cos, sin))
             and not transformed(q_norm.weight, k_norm.weight, cos, sin))
    if not fused:
        from ._eager import apply_rope

        q4, k4, v4 = (t.view(B, T, -1, D) for t in (q, k, v))
        q4, k4 = apply_rope(q_norm(q4).transpose(1, 2), k_norm(k4).transpose(1, 2), cos, sin)
        return attention_kv8(q4.transpose(1, 2), k4.transpose(1, 2), v4, cache, layer, start_pos).view(B, T, -1)
    start, pos = _place(fn, start_pos, None)
    refuse_grad(fn, q, k, v)
    return _lib.ops().attention_kv8(q, k, v, q_norm.weight, k_norm.weight, q_norm.eps, k_norm.eps, cos, sin,
                                    cache.layers[layer], cache.size, start, pos, None)
