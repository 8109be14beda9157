"""Key/value caches of two parts and attention over them: sequences that continue one
text, whose keys and values are held and read once for all (``KVCacheShared``), and
texts without an end, of which a window of the last tokens and the first few stay
(``KVCacheWindow``).

The reference has neither (its cache is one tensor per layer, ``src/engine/kv_cache.py:19-47``).
Both caches are bf16 and have a fixed part, positions ``0 .. n - 1`` (the shared text, or
the first tokens), and an own part of each sequence. One kernel family attends over both
(``llms_amd/csrc/fp_seg.hip``): softmax in fp32 with scale ``D ** -0.5`` over the entries that
a token sees. What it does not see has no part in it, whatever it holds. A row that sees a score that is NaN or
the positive infinity is NaN (a score of the negative one has no weight, as in torch), and so is the column of a value
that is not finite in the rows that see it.

Path: wrapper -> ``torch.ops.llms_amd.attention_seg`` / ``write_seg`` -> C ABI
``fp_seg_attention`` / ``fp_seg_write`` -> HIP kernels on torch's current stream.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._checks import autocast, plain_norm, refuse_grad, transformed
from .kv8 import _place

MAX_LEN = 1 << 28
MAX_POS = 1 << 30  # of a window's cache


class _TwoParts:
    """What the two caches share. ``k``, ``v``: a tensor per layer; ``parts`` the views of it that
    the operator takes. Calls on one cache must be ordered (one stream, or streams that
    wait for each other). ``cur_len`` is the model's count of tokens, as in ``KVCache``."""

    window = 0

    def parts(self, layer: int) -> list:
        raise NotImplementedError

    def _pieces(self, T: int):
        """Cuts of a call's tokens: (first, end)."""
        return [(0, T)]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, start_pos, *, lengths=None) -> None:
        """Put ``k``, ``v`` ``[B, T, n_kv_heads, D]`` (bfloat16, normalised and rotated) at positions
        ``start_pos ..``; arguments as in the attention call."""
        fn = f"{type(self).__name__}.write"
        start, pos = _place(fn, start_pos, lengths)
        refuse_grad(fn, k, v)
        _check_tokens(fn, k, self, start, pos)
        for lo, hi in self._pieces(k.shape[1]):
            s, p, n = _at(lo, hi, k.shape[1], start, pos, lengths)
            _lib.ops().write_seg(k[:, lo:hi], v[:, lo:hi], *self.parts(layer), self.window, s, p, n)

    def step_slots(self, T: int):
        """A position for a step of T tokens, and views of what the step would write there."""
        raise NotImplementedError


def _at(lo: int, hi: int, T: int, start: int, pos, lengths):
    """start_pos and lengths of a call's tokens lo .. hi - 1."""
    if lo == 0 and hi == T:
        return start, pos, lengths
    return (start + lo, None if pos is None else pos + lo,
            None if lengths is None else (lengths - lo).clamp(0, hi - lo))


def _check_tokens(fn: str, k: torch.Tensor, cache: _TwoParts, start: int, pos) -> None:
    """What the operator would find only after some of a call's steps were done (it checks the rest)."""
    if k.dim() not in (3, 4):
        raise ValueError(f"{fn}: k {tuple(k.shape)} must be (B, T, {cache.n_kv_heads}, {cache.head_dim})")
    if cache.window and pos is None and start + k.shape[1] > MAX_POS:
        raise ValueError(f"{fn}: positions {start} .. {start + k.shape[1] - 1} are outside 0 .. {MAX_POS - 1}")


class KVCacheShared(_TwoParts):
    """A text that up to ``max_batch`` sequences continue, by up to ``max_new`` tokens each.

    Args:
        prefix_k, prefix_v: per layer the text's keys and values ``[n_kv_heads, P, D]`` (bfloat16,
            normalised and rotated), which are used as they are, not copied, and not written to.
            Token p of a sequence is at position p from the text's start: its own start at P.

    ``k``, ``v``: per layer the sequences' own ``[max_batch, n_kv_heads, max_new, D]``. A call may
    start anywhere from P on, and over what was written before.
    """

    def __init__(self, prefix_k: list, prefix_v: list, *, max_batch: int, max_new: int) -> None:
        name = "KVCacheShared"
        if len(prefix_k) < 1 or len(prefix_k) != len(prefix_v):
            raise ValueError(f"{name}: keys of {len(prefix_k)} layers and values of {len(prefix_v)}")
        if max_batch < 1 or not 1 <= max_new <= MAX_LEN:
            raise ValueError(f"{name}: max_batch and max_new must be at least 1, got {max_batch}, {max_new}")
        first = prefix_k[0]
        if first.dim() != 3 or first.shape[2] not in (64, 128) or not 1 <= first.shape[1] <= MAX_LEN:
            raise ValueError(f"{name}: a text's keys must be (n_kv_heads, P, 64 or 128) with P at least 1, "
                             f"got {tuple(first.shape)}")
        for t in (*prefix_k, *prefix_v):
            if t.shape != first.shape or t.dtype != torch.bfloat16 or t.device != first.device:
                raise ValueError(f"{name}: keys and values of all layers must be alike and bfloat16, got "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        self.n_kv_heads, self.prefix_len, self.head_dim = first.shape
        self.max_batch, self.max_new = max_batch, max_new
        self.max_seq = self.prefix_len + max_new
        self.cur_len = self.prefix_len
        self.prefix_k, self.prefix_v = [], []
        for k, v in zip(prefix_k, prefix_v):
            k, v = k.detach(), v.detach()
            if k.stride() != v.stride() or any(_off(t) for t in (k, v)):
                k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
            self.prefix_k.append(k)
            self.prefix_v.append(v)
        new = lambda: torch.zeros(max_batch, self.n_kv_heads, max_new, self.head_dim,  # noqa: E731
                                  dtype=torch.bfloat16, device=first.device)
        self.k = [new() for _ in prefix_k]
        self.v = [new() for _ in prefix_k]

    @classmethod
    def of(cls, cache, length: int, *, max_batch: int, max_new: int) -> "KVCacheShared":
        """The first ``length`` tokens of sequence 0 in a plain cache (``harness.KVCache``: lists ``k``, ``v`` of
        ``[batch, n_kv_heads, max_seq, D]``) as the shared text: views of its tensors."""
        if isinstance(cache, _TwoParts):  # (its tensors do not hold position p at p)
            raise TypeError(f"KVCacheShared.of: a text is taken from a plain cache, not a {type(cache).__name__}")
        if not 1 <= length <= cache.k[0].shape[2]:
            raise ValueError(f"KVCacheShared.of: length {length} of a cache of {cache.k[0].shape[2]}")
        return cls([t[0, :, :length] for t in cache.k], [t[0, :, :length] for t in cache.v], max_batch=max_batch,
                   max_new=max_new)

    def parts(self, layer: int) -> list:
        return [self.prefix_k[layer], self.prefix_v[layer], self.k[layer], self.v[layer]]

    def step_slots(self, T: int):
        return self.prefix_len, [t[:, :, :T] for t in (*self.k, *self.v)]


def _off(t: torch.Tensor) -> bool:
    """Whether the kernels cannot read t [.., D] as it is: rows of 16-byte chunks."""
    return (t.stride(-1) != 1 or any(s < 0 or s % 8 for s in t.stride()[:-1]) or t.stride(-2) < t.shape[-1]
            or t.data_ptr() % 16 != 0)


class KVCacheWindow(_TwoParts):
    """The last ``window`` tokens of up to ``max_batch`` texts of any length, and their first ``sinks``.

    ``k``, ``v``: per layer ``[max_batch, n_kv_heads, sinks + ring, D]``: position p < sinks in slot p, any
    other in slot ``sinks + (p - sinks) % ring``, with ``ring`` the multiple of 64 that holds a window and a
    step of ``max_step`` tokens. Longer calls are done in steps of that.

    Tokens are written in order. A call may take back up to ``max_step`` tokens (a rejected draft): start at
    ``n - max_step`` or later, where ``n - 1`` is the furthest position written so far (tokens that were taken back
    count). Further back the window is gone. Positions are under 2^30.
    """

    def __init__(self, k: list, v: list, window: int, sinks: int, max_step: int) -> None:
        self.k, self.v = k, v
        self.window, self.sinks, self.max_step = window, sinks, max_step
        self.max_batch, self.n_kv_heads, n, self.head_dim = k[0].shape
        self.ring = n - sinks
        self.cur_len = 0
        self._parts = [[t[:, :, :sinks] for t in (a, b)] + [t[:, :, sinks:] for t in (a, b)] for a, b in zip(k, v)]

    @classmethod
    def alloc(cls, num_layers: int, window: int, *, sinks: int = 4, max_step: int = 256, max_batch: int = 1,
              n_kv_heads: int, head_dim: int, device) -> "KVCacheWindow":
        if num_layers < 1 or max_batch < 1 or n_kv_heads < 1:
            raise ValueError(f"KVCacheWindow: num_layers, max_batch and n_kv_heads must be at least 1, got "
                             f"{num_layers}, {max_batch}, {n_kv_heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"KVCacheWindow: heads of 64 or 128 are taken, got {head_dim}")
        if window < 1 or max_step < 1 or sinks < 0 or window + max_step + sinks > MAX_LEN - 64:
            raise ValueError(f"KVCacheWindow: window and max_step must be at least 1 and sinks at least 0, under 2^28 "
                             f"together, got {window}, {max_step}, {sinks}")
        ring = -(-(window + max_step - 1) // 64) * 64
        new = lambda: torch.zeros(max_batch, n_kv_heads, sinks + ring, head_dim, dtype=torch.bfloat16,  # noqa: E731
                                  device=device)
        return cls([new() for _ in range(num_layers)], [new() for _ in range(num_layers)], window, sinks, max_step)

    def parts(self, layer: int) -> list:
        return self._parts[layer]

    def _pieces(self, T: int):
        return [(lo, min(T, lo + self.max_step)) for lo in range(0, T, self.max_step)] if T > self.max_step else [(0, T)]

    def step_slots(self, T: int):
        if T > self.max_step:
            raise ValueError(f"KVCacheWindow: a step of {T} tokens, max_step is {self.max_step}")
        return 0, [t[:, :, :T] for t in (*self.k, *self.v)]


def _attend(fn, q, k, v, norms, cos, sin, cache, layer, start_pos, lengths):
    start, pos = _place(fn, start_pos, lengths)
    refuse_grad(fn, q, k, v)
    _check_tokens(fn, k, cache, start, pos)
    T, out = k.shape[1], []
    for lo, hi in cache._pieces(T):
        s, p, n = _at(lo, hi, T, start, pos, lengths)
        whole = hi - lo == T
        cut = lambda t: t if whole or t is None else t[..., lo:hi, :]  # noqa: E731
        qkv = (q, k, v) if whole else (t[:, lo:hi] for t in (q, k, v))
        out.append(_lib.ops().attention_seg(*qkv, *norms, cut(cos), cut(sin), *cache.parts(layer), cache.window, s, p, n))
    return out[0] if len(out) == 1 else torch.cat(out, 1)


def attention_shared(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KVCacheShared, layer: int, start_pos,
                     *, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Write the new keys and values of a batch of sequences that continue one text, and attend over
    the text and each sequence's own tokens.

    Args:
        q: ``[B, T, heads, D]`` bfloat16 on the cache's device; k, v: ``[B, T, n_kv_heads, D]``; normalised
            and rotated. heads is a multiple of ``n_kv_heads``.
        start_pos: the position of token 0, from the shared text's length on: an int, or an int64 tensor on
            the device, 0-dim or ``[B]`` for sequences of different lengths (a call captured in a HIP
            graph replays at any positions).
        lengths: how many of the T tokens each sequence has (int64 ``[B]`` on the device, default T): the
            others are not written.

    Returns:
        ``[B, T, heads, D]`` bfloat16: attention of the token at position p over positions 0 .. p. Rows past
        a sequence's length, and at device positions outside its own part (whose tokens are not
        written), are zero. Keys of the text are read once for all sequences while they have few tokens
        each (32 query rows per kv head).
    """
    return _attend("attention_shared", q, k, v, (None, None, 0.0, 0.0), None, None, cache, layer, start_pos, lengths)


def attention_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KVCacheWindow, layer: int, start_pos,
                     *, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Write the new keys and values into a cache with a window, and attend over it.

    Arguments and result as in :func:`attention_shared`, with positions from 0 on: the token at position p sees
    positions ``p - window + 1 .. p`` and the first ``sinks`` (up to p). Rows at device positions outside
    0 .. 2^30 - 1 are zero.
    """
    return _attend("attention_window", q, k, v, (None, None, 0.0, 0.0), None, None, cache, layer, start_pos, lengths)


def attention_core_seg(q, k, v, *, q_norm, k_norm, num_heads: int, cache: _TwoParts, layer: int, cos, sin,
                       start_pos) -> torch.Tensor:
    """What ``TritonAttention.forward`` does between its projections with a cache of two parts: QK-norm
    and RoPE of the flat projections ``[B, T, heads * D]`` in the kernel that writes the keys (in torch
    where a norm is not the plain one or a type is not bf16's), the cache write and attention. cos and sin
    are ``[T, D]``, or ``[B, T, D]`` for sequences at different positions. Returns ``[B, T, num_heads * D]``."""
    fn, D = "attention_window" if cache.window else "attention_shared", cache.head_dim
    B, T, _ = q.shape
    if any(t.shape not in ((T, D), (B, T, D)) for t in (cos, sin)):  # (one row would be every token's in torch)
        raise ValueError(f"{fn}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be {(T, D)} or {(B, T, D)}")
    fused = (plain_norm(q_norm) and plain_norm(k_norm) and not autocast()
             and all(t.dtype == torch.bfloat16 and t.shape == (D,) and t.is_contiguous() and t.data_ptr() % 16 == 0
                     for t in (q_norm.weight, k_norm.weight))
             and all(t.dtype == torch.bfloat16 and t.stride(-1) == 1
                     and t.device == q.device and (T == 1 or t.stride(-2) >= D) for t in (cos, sin))
             and not transformed(q_norm.weight, k_norm.weight, cos, sin))
    if not fused:
        from ._eager import rotate_half

        c, s = (t.unsqueeze(-2) for t in (cos, sin))  # [T, 1, D] or [B, T, 1, D]
        q4, k4, v4 = (t.view(B, T, -1, D) for t in (q, k, v))
        q4, k4 = (t * c + rotate_half(t) * s for t in (q_norm(q4), k_norm(k4)))
        return _attend(fn, q4, k4, v4, (None, None, 0.0, 0.0), None, None, cache, layer, start_pos, None).view(B, T, -1)
    return _attend(fn, q, k, v, (q_norm.weight, k_norm.weight, q_norm.eps, k_norm.eps), cos, sin, cache, layer,
                   start_pos, None)
