"""A key/value cache in 8 bits with one scale for each block of 64 tokens and head,
and causal attention over it: half the cache bytes of a bf16 decode step.

The reference's cache is bf16 (``src/engine/kv_cache.py:19-47``). Here a block is packed
once, from its bf16 tokens, when its last token arrives; the tokens of the
unfinished block (and of the one before it) are kept in bf16. What the cache holds
therefore does not depend on how its tokens were cut into calls, and a
verify step that takes back a few tokens finds them unpacked. Going further back,
to any position, works too: the block it lands in goes on from its packed values.

Path: wrapper -> ``torch.ops.llms_amd.attention_kv8`` / ``write_kv8`` /
``read_kv8`` -> C ABI ``fp_kv8_attention`` / ``fp_kv8_write`` / ``fp_kv8_read`` -> HIP
kernels (``llms_amd/csrc/fp_kv8.hip``) on torch's current stream.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._checks import autocast, plain_norm, refuse_grad, require_bf16_hip, transformed

BLOCK = 64
MAX_SEQ = 1 << 23


class KVCache8:
    """The 8-bit caches of a model's layers, for up to ``max_batch`` sequences of
    up to ``max_seq`` tokens (the counterpart of the harness's ``KVCache``).

    ``cur_len`` is the model's count of tokens, as in ``KVCache``. Tokens are
    written in order: a call may start anywhere up to the tokens written so far (what
    is behind it is dropped), not later (the unfinished block would be lost).
    A key or value that is not finite is held as NaN. Calls on one cache must be ordered
    (one stream, or streams that wait for each other).
    """

    def __init__(self, layers: list, max_seq: int) -> None:
        # per layer: codes, scales and bf16 tails of keys and of values, the blocks in the tails
        self.layers = layers
        self.max_seq = max_seq
        self.cur_len = 0
        c = layers[0][0]
        self.max_batch, self.n_kv_heads, _, _, self.head_dim = c.shape

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
        lead, nb, D = (max_batch, n_kv_heads), -(-max_seq // BLOCK), head_dim
        layers = []
        for _ in range(num_layers):
            z = lambda *s, t: torch.zeros(*lead, *s, dtype=t, device=device)  # noqa: E731
            layers.append([z(nb, BLOCK, D, t=torch.int8), z(nb, D, BLOCK, t=torch.int8),
                           z(nb, t=torch.float32), z(nb, t=torch.float32),
                           z(2, BLOCK, D, t=torch.bfloat16), z(2, D, BLOCK, t=torch.bfloat16),
                           torch.full((*lead, 2), -1, dtype=torch.int32, device=device)])
        return cls(layers, max_seq)

    @property
    def device(self) -> torch.device:
        return self.layers[0][0].device

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, start_pos, *, lengths=None) -> None:
        """Put ``k``, ``v`` ``[B, T, n_kv_heads, D]`` (bfloat16, normalised and rotated)
        at positions ``start_pos ..``; arguments as in :func:`attention_kv8`."""
        B, T = _tokens("KVCache8.write", self, k, v)
        start, pos = _place("KVCache8.write", self, B, T, start_pos, lengths)
        if B and T:
            _lib.ops().write_kv8(_flat(k), _flat(v), self.layers[layer], self.max_seq, start, pos, lengths)

    def read(self, layer: int, start_pos, T: int, *, batch: int | None = None):
        """The keys and values ``[B, T, n_kv_heads, D]`` in float32 that attention sees at
        positions ``start_pos .. start_pos + T - 1`` of sequences that end there (with
        ``start_pos`` 0 and ``T`` the length: all). B is ``batch``, the number of
        positions in ``start_pos [B]``, or ``max_batch``."""
        if batch is None:
            batch = start_pos.shape[0] if torch.is_tensor(start_pos) and start_pos.dim() == 1 else self.max_batch
        if not 1 <= batch <= self.max_batch or T < 1:
            raise ValueError(f"KVCache8.read: batch {batch} and T {T} must be 1 to {self.max_batch} and at least 1")
        start, pos = _place("KVCache8.read", self, batch, T, start_pos, None)
        if self.device.type != "cuda":
            raise ValueError(f"KVCache8.read: the cache is on {self.device}; it runs only on a HIP (ROCm) device")
        return _lib.ops().read_kv8(self.layers[layer], self.max_seq, batch, T, start, pos)

    def tails(self) -> list:
        """The buffers of every layer that a write outside the sequence would lose."""
        return [t for c in self.layers for t in c[4:]]


def _flat(t: torch.Tensor) -> torch.Tensor:
    """t [B, T, H, D] as rows [B, T, H * D] that the kernels take (a copy where a
    head, a row or the batch is not laid out for them)."""
    B, T, H, D = t.shape
    s = t.stride()
    ok = s[3] == 1 and (H == 1 or s[2] == D) and t.data_ptr() % 8 == 0
    ld = s[1] if T > 1 else s[0] if B > 1 else H * D
    if not ok or ld % 4 or ld < H * D or (B > 1 and s[0] != T * ld):
        t = t.contiguous()
    return t.reshape(B, T, H * D) if t.is_contiguous() else t.as_strided((B, T, H * D), (T * ld, ld, 1))


def _tokens(fn: str, cache: KVCache8, k: torch.Tensor, v: torch.Tensor) -> tuple[int, int]:
    if k.dim() != 4 or k.shape != v.shape or k.shape[2:] != (cache.n_kv_heads, cache.head_dim):
        raise ValueError(f"{fn}: k {tuple(k.shape)} and v {tuple(v.shape)} must be "
                         f"(B, T, {cache.n_kv_heads}, {cache.head_dim})")
    if k.shape[0] > cache.max_batch:
        raise ValueError(f"{fn}: {k.shape[0]} sequences, the cache holds {cache.max_batch}")
    require_bf16_hip(fn, k=k, v=v)
    if not (k.device == v.device == cache.device):
        raise ValueError(f"{fn}: k ({k.device}), v ({v.device}) and the cache ({cache.device}) "
                         "must be on the same device")
    refuse_grad(fn, k, v)
    return k.shape[0], k.shape[1]


def _place(fn: str, cache: KVCache8, B: int, T: int, start_pos, lengths):
    """(start_pos as an int, as a device tensor or None)."""
    if lengths is not None:
        if not torch.is_tensor(lengths) or lengths.dtype != torch.int64 or lengths.shape != (B,):
            raise ValueError(f"{fn}: lengths must be an int64 tensor of {B} elements")
        if lengths.device != cache.device or not lengths.is_contiguous():
            raise ValueError(f"{fn}: lengths must be contiguous on {cache.device}")
    if torch.is_tensor(start_pos):
        if start_pos.dtype != torch.int64 or start_pos.shape not in ((), (B,)):
            raise ValueError(f"{fn}: start_pos must be an int or an int64 tensor of shape () or ({B},), got "
                             f"{start_pos.dtype} {tuple(start_pos.shape)}")
        if start_pos.device != cache.device or not start_pos.is_contiguous():
            raise ValueError(f"{fn}: start_pos must be contiguous on {cache.device}")
        return 0, start_pos
    if type(start_pos) is not int:
        raise TypeError(f"{fn}: start_pos must be an int or an int64 tensor, got {type(start_pos).__name__}")
    if start_pos < 0 or start_pos + T > cache.max_seq:
        raise ValueError(f"{fn}: positions {start_pos} .. {start_pos + T - 1} are outside the cache of "
                         f"{cache.max_seq}")
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
        at position p over positions 0 .. p. Rows past a sequence's length, and at device
        positions outside the cache (whose tokens are not written), are zero.
    """
    fn = "attention_kv8"
    B, T = _tokens(fn, cache, k, v)
    if q.dim() != 4 or q.shape[:2] != (B, T) or q.shape[3] != cache.head_dim:
        raise ValueError(f"{fn}: q {tuple(q.shape)} must be ({B}, {T}, heads, {cache.head_dim})")
    H = q.shape[2]
    if H < 1 or H % cache.n_kv_heads:
        raise ValueError(f"{fn}: {H} query heads are no multiple of {cache.n_kv_heads} kv heads")
    require_bf16_hip(fn, q=q)
    if q.device != cache.device:
        raise ValueError(f"{fn}: q ({q.device}) and the cache ({cache.device}) must be on the same device")
    refuse_grad(fn, q)
    start, pos = _place(fn, cache, B, T, start_pos, lengths)
    if B == 0 or T == 0:
        return torch.empty_like(q)
    y = _lib.ops().attention_kv8(_flat(q), _flat(k), _flat(v), None, None, 0.0, 0.0, None, None,
                                 cache.layers[layer], cache.max_seq, start, pos, lengths)
    return y.view(B, T, H, cache.head_dim)


def attention_core_kv8(q, k, v, *, q_norm, k_norm, num_heads: int, cache: KVCache8, layer: int, cos, sin,
                       start_pos) -> torch.Tensor:
    """What ``TritonAttention.forward`` does between its projections with an 8-bit
    cache: QK-norm and RoPE of the flat projections ``[B, T, heads * D]`` in the
    kernel that writes the keys (in torch where a norm is not the plain one or a
    type is not bf16's), the cache write and attention. Returns ``[B, T, num_heads * D]``."""
    fn, D = "attention_kv8", cache.head_dim
    B, T, _ = q.shape
    q4, k4, v4 = (t.view(B, T, -1, D) for t in (q, k, v))
    fused = (plain_norm(q_norm) and plain_norm(k_norm) and not autocast()
             and all(t.dtype == torch.bfloat16 and t.shape == (D,) and t.is_contiguous()
                     for t in (q_norm.weight, k_norm.weight))
             and all(t.dtype == torch.bfloat16 and t.shape == (T, D) and t.stride(1) == 1 and t.device == q.device
                     for t in (cos, sin))
             and not transformed(q_norm.weight, k_norm.weight, cos, sin))
    if not fused:
        from ._eager import apply_rope

        q4, k4 = apply_rope(q_norm(q4).transpose(1, 2), k_norm(k4).transpose(1, 2), cos, sin)
        return attention_kv8(q4.transpose(1, 2), k4.transpose(1, 2), v4, cache, layer, start_pos).view(B, T, -1)
    _tokens(fn, cache, k4, v4)
    require_bf16_hip(fn, q=q)
    refuse_grad(fn, q)
    start, pos = _place(fn, cache, B, T, start_pos, None)
    return _lib.ops().attention_kv8(_flat(q4), _flat(k4), _flat(v4), q_norm.weight, k_norm.weight, q_norm.eps,
                                    k_norm.eps, cos, sin, cache.layers[layer], cache.max_seq, start, pos, None)
