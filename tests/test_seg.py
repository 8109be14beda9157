"""Attention over a shared text and over a window with sinks against 64 bits, the caches, and
models that use them."""

from __future__ import annotations

import copy
import ctypes

import pytest
import torch

from llms_amd import _lib, harness
from llms_amd import kernels as fk

DEV = "cuda"
gpu = pytest.mark.gpu
HEADS = [(16, 8, 128), (8, 2, 64), (7, 1, 128), (3, 3, 64), (40, 8, 128)]


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).bfloat16()


def exact(q, k, v, q_pos, k_pos, window=0, sinks=0):
    """Of one sequence: q [T, Hq, D] at q_pos, k, v [n, Hk, D] at k_pos, on the GPU in 64 bits:
    (y, the weights' sum of |v|, which rows' columns see a value that is not finite)."""
    q, k, v = (t.to(DEV).double() for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    q_pos, k_pos = q_pos.to(DEV)[:, None], k_pos.to(DEV)[None]
    seen = k_pos <= q_pos
    if window:
        seen &= (k_pos > q_pos - window) | (k_pos < sinks)
    y, size, bad = (torch.zeros(q.shape, dtype=torch.double, device=DEV) for _ in range(3))
    fine = v.isfinite()
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // G].T / q.shape[2] ** 0.5
        w = s.masked_fill(~seen, -torch.inf).softmax(1)
        vh = torch.where(fine[:, h // G], v[:, h // G], 0.0)
        y[:, h], size[:, h] = w @ vh, w @ vh.abs()
        bad[:, h] = seen.double() @ (~fine[:, h // G]).double()
    return y, size, bad > 0


def check(y, e, parts, rows=None):
    """y [T, Hq, D] against exact()'s. One rounding to bf16 (2^-8 of the value at most). Each p enters in
    `parts` parts of bf16: off by 2^-8 of itself (one) or 2^-16 (two), in the products and in their
    sum, so twice that of the weighted |v|; 2^-17 of it more for fp32's scores (|q k| sums to
    under 2^7 here, each rounding 2^-24), exponentials and sums."""
    want, size, bad = e
    y = y.to(DEV).double()
    if rows is not None:
        y, want, size, bad = y[:rows], want[:rows], size[:rows], bad[:rows]
    err = (y - want).abs()
    tol = want.abs() * 2.0**-8 + size * (2 * 2.0 ** (-8 * parts) * (1 + 2.0**-8) + 2.0**-17) + 1e-30
    assert torch.equal(y.isnan(), bad), (y.isnan().sum(), bad.sum())
    ok = err <= tol
    assert (ok | bad).all(), float((err / tol)[~bad].max())


def parts(T, Hq, Hk, B=1):
    """Query rows per kv head that one kernel takes: over 64 of them p enters in one part. (A shared text is read
    for all sequences' rows together.)"""
    return 2 if B * T * Hq // Hk <= 64 else 1


# ------------------------------------------------------------- refusals (CPU)


def shared(H=2, P=10, D=64, B=3, n=8, dev="cpu", layers=1):
    t = [torch.zeros(H, P, D, dtype=torch.bfloat16, device=dev) for _ in range(2 * layers)]
    return fk.KVCacheShared(t[:layers], t[layers:], max_batch=B, max_new=n)


def test_refusals_on_the_cpu():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    w = fk.KVCacheWindow.alloc(1, 100, n_kv_heads=2, head_dim=64, device="cpu")
    assert w.ring == 384 and w.k[0].shape == (1, 2, 388, 64)  # 100 + 256 - 1 in whole 64
    for call, c, at in ((fk.attention_window, w, 0), (fk.attention_shared, shared(), 10)):
        q, k = z(1, 2, 4, 64), z(1, 2, 2, 64)
        with pytest.raises(ValueError, match="HIP"):
            call(q, k, k, c, 0, at)
        with pytest.raises(ValueError, match="must be"):
            call(q, k[..., :32], k[..., :32], c, 0, at)
        with pytest.raises(ValueError, match="must be"):
            call(q, z(1, 2), z(1, 2), c, 0, at)
        with pytest.raises(ValueError, match="and v"):
            call(q, k, k[:, :1], c, 0, at)
        with pytest.raises(TypeError, match="bfloat16"):
            call(q, k.float(), k.float(), c, 0, at)
        with pytest.raises(TypeError, match="start_pos"):
            call(q, k, k, c, 0, 1.5)
        with pytest.raises(ValueError, match="outside"):
            call(q, k, k, c, 0, at - 1)
        with pytest.raises(ValueError, match="outside"):
            call(q, k, k, c, 0, 1 << 30)
        with pytest.raises(ValueError, match="lengths"):
            call(q, k, k, c, 0, at, lengths=[1])
        with pytest.raises(ValueError, match="lengths"):
            call(q, k, k, c, 0, at, lengths=torch.zeros(2, dtype=torch.long))
        with pytest.raises(ValueError, match="sequences"):
            call(z(9, 2, 4, 64), z(9, 2, 2, 64), z(9, 2, 2, 64), c, 0, at)
        with pytest.raises(RuntimeError, match="no gradients"):
            call(q.float().requires_grad_().bfloat16(), k, k, c, 0, at)
        with pytest.raises(ValueError, match="HIP"):
            c.write(0, k, k, at)
        with pytest.raises(RuntimeError, match="no gradients"):
            c.write(0, k.float().requires_grad_().bfloat16(), k, at)
    c = shared()
    with pytest.raises(ValueError, match="outside"):
        fk.attention_shared(z(1, 9, 4, 64), z(1, 9, 2, 64), z(1, 9, 2, 64), c, 0, 10)
    for kw in (dict(window=0), dict(max_step=0), dict(sinks=-1), dict(head_dim=32), dict(n_kv_heads=0),
               dict(window=1 << 29)):
        with pytest.raises(ValueError, match="KVCacheWindow"):
            fk.KVCacheWindow.alloc(**(dict(num_layers=1, window=8, n_kv_heads=1, head_dim=64, device="cpu") | kw))
    for args in (([], []), ([z(2, 3, 64)], []), ([z(2, 3, 32)], [z(2, 3, 32)]), ([z(2, 0, 64)], [z(2, 0, 64)]),
                 ([z(2, 3, 64)], [z(2, 4, 64)]), ([z(2, 3, 64).float()], [z(2, 3, 64).float()])):
        with pytest.raises(ValueError, match="KVCacheShared"):
            fk.KVCacheShared(*args, max_batch=1, max_new=1)
    with pytest.raises(ValueError, match="KVCacheShared"):
        shared(B=0)
    model = harness.tiny_model(harness.Cfg(head_dim=64))
    with pytest.raises(ValueError, match="length"):
        fk.KVCacheShared.of(model.alloc_cache(8), 9, max_batch=1, max_new=1)
    for cache in (model.alloc_cache(8, window=4), fk.KVCacheShared.of(model.alloc_cache(8), 4, max_batch=1, max_new=4)):
        with pytest.raises(TypeError, match="apply_triton_kernels"):
            model(torch.zeros(1, 1, dtype=torch.long), cache, start_pos=4)
    with pytest.raises(ValueError, match="kv8"):
        model.alloc_cache(8, window=4, kv8=True)


class SegArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in "q k v".split()]
                + [(n, ctypes.c_int64) for n in "q_s_b q_s_t k_s_b k_s_t v_s_b v_s_t".split()]
                + [(n, ctypes.c_void_p) for n in "q_gamma k_gamma cos sin".split()]
                + [(n, ctypes.c_int64) for n in "cos_s_b cos_s_t sin_s_b sin_s_t".split()]
                + [(n, ctypes.c_void_p) for n in "fix_k fix_v".split()]
                + [(n, ctypes.c_int64) for n in "fix_s_b fix_s_h fix_s_p".split()]
                + [(n, ctypes.c_void_p) for n in "own_k own_v".split()]
                + [(n, ctypes.c_int64) for n in "own_s_b own_s_h own_s_p".split()]
                + [("y", ctypes.c_void_p), ("y_s_b", ctypes.c_int64)]
                + [(n, ctypes.c_int64) for n in
                   "B T n_heads n_kv_heads head_dim n_fixed own_len ring window pos".split()]
                + [("pos_dev", ctypes.c_void_p), ("pos_stride", ctypes.c_int64), ("lengths", ctypes.c_void_p),
                   ("q_eps", ctypes.c_float), ("k_eps", ctypes.c_float)])


def test_c_arguments():
    """Every refusal comes before a launch (there is no GPU here: a launch would not be FP_OK either)."""
    lib = _lib.capi()
    P, NULL, SHAPE, STRIDE, WS = 64, 1, 2, 3, 6

    def call(keys=100, ws=P, n=1 << 40, write=False, **kw):
        D, Hk, S, F = 64, 2, 128, 100
        a = dict(q=P, k=P, v=P, q_s_b=256, q_s_t=256, k_s_b=128, k_s_t=128, v_s_b=128, v_s_t=128, fix_k=P, fix_v=P,
                 fix_s_b=0, fix_s_h=F * D, fix_s_p=D, own_k=P, own_v=P, own_s_b=Hk * S * D, own_s_h=S * D, own_s_p=D,
                 y=P, y_s_b=256, B=3, T=1, n_heads=4, n_kv_heads=Hk, head_dim=D, n_fixed=F, own_len=S, pos=100)
        args = SegArgs(**(a | kw))
        return lib.fp_seg_write(ctypes.byref(args), None) if write else \
            lib.fp_seg_attention(ctypes.byref(args), keys, ws, n, None)

    for kw in (dict(B=0), dict(T=0), dict(n_heads=3), dict(head_dim=32), dict(n_fixed=-1), dict(own_len=0),
               dict(pos=99), dict(pos=228), dict(pos=1 << 40), dict(window=3), dict(ring=1), dict(keys=0),
               dict(ring=1, window=129), dict(ring=1, window=10, own_len=100), dict(ring=1, window=10, pos=-1),
               dict(ring=1, window=10, pos=1 << 30), dict(own_s_p=1 << 23), dict(q_eps=float("nan"))):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(q_s_t=255), dict(k_s_t=64), dict(own_s_p=60), dict(fix_s_p=60), dict(own_s_h=4), dict(q=P + 8),
               dict(y=P + 2), dict(own_s_b=-8), dict(pos_dev=P, pos_stride=2), dict(cos=P, sin=P, cos_s_t=63, sin_s_t=64)):
        assert call(**kw) == STRIDE, kw
    for kw in (dict(q=None), dict(k=None), dict(own_v=None), dict(fix_k=None), dict(y=None), dict(cos=P),
               dict(cos=P, sin=P, cos_s_t=64, sin_s_t=64, q_gamma=P)):
        assert call(**kw) == NULL, kw
    need = lib.fp_seg_workspace_bytes(3, 1, 4, 2, 64, 100, 100, 1, 0)
    assert need > 0 and call(n=need - 1) == WS and call(ws=None) == WS and call(ws=P + 4) == WS
    assert call(write=True, B=0) == SHAPE and call(write=True, k=None) == NULL and call(write=True, own_s_h=4) == STRIDE
    assert lib.fp_seg_attention(None, 1, P, 1, None) == NULL and lib.fp_seg_write(None, None) == NULL
    assert lib.fp_seg_workspace_bytes(0, 1, 4, 2, 64, 0, 1, 0, 0) == 0


# ------------------------------------------------------------- a shared text


def step_shared(g, c, hist, starts, counts, T, Hq, device_pos, lengths):
    """One call of all of a cache's sequences, whose histories (k, v lists, text first) it extends."""
    B, Hk, D, P = len(starts), c.n_kv_heads, c.head_dim, c.prefix_len
    q, k, v = randn(g, B, T, Hq, D, scale=1.5), randn(g, B, T, Hk, D), randn(g, B, T, Hk, D)
    at = P + torch.tensor(starts) if device_pos else P + starts[0]
    y = fk.attention_shared(q.to(DEV), k.to(DEV), v.to(DEV), c, 0, at.to(DEV) if device_pos else at,
                            lengths=torch.tensor(counts).to(DEV) if lengths else None)
    for b in range(B):
        n = counts[b]
        for name, x in (("k", k), ("v", v)):
            hist[b][name] = torch.cat([hist[b][name][: P + starts[b]], x[b, :n]])
        if n:
            e = exact(q[b, :n], hist[b]["k"], hist[b]["v"], P + starts[b] + torch.arange(n), torch.arange(P + starts[b] + n))
            check(y[b, :n], e, parts(T, Hq, Hk, B))
        assert (y[b, n:] == 0).all()
        own = c.k[0][b, :, : starts[b] + n].transpose(0, 1).cpu()
        assert torch.equal(own, hist[b]["k"][P:])
    return [s + n for s, n in zip(starts, counts)]


def new_shared(g, H, P, D, B, n):
    t = [randn(g, H, P, D) for _ in range(2)]
    c = fk.KVCacheShared([t[0].to(DEV)], [t[1].to(DEV)], max_batch=B, max_new=n)
    return c, [{"k": t[0].transpose(0, 1), "v": t[1].transpose(0, 1)} for _ in range(B)]


@gpu
@pytest.mark.parametrize("Hq,Hk,D", HEADS)
@pytest.mark.parametrize("B", [1, 2, 9, 40])
@pytest.mark.parametrize("P", [1, 31, 64, 333, 2500])
def test_shared_steps(Hq, Hk, D, B, P):
    """Tokens one by one and in steps, each sequence at its own position."""
    g = torch.Generator().manual_seed(B * P + Hq)
    c, hist = new_shared(g, Hk, P, D, B, 60)
    starts = [0] * B
    starts = step_shared(g, c, hist, starts, [1] * B, 1, Hq, False, False)
    counts = [1 + (b * 5) % 9 for b in range(B)]
    starts = step_shared(g, c, hist, starts, counts, 9, Hq, True, True)
    starts = step_shared(g, c, hist, starts, [1] * B, 1, Hq, True, False)
    starts = step_shared(g, c, hist, [s - 1 for s in starts], [3] * B, 3, Hq, True, False)  # one taken back
    step_shared(g, c, hist, starts, [0 if b % 3 == 1 else 2 for b in range(B)], 2, Hq, True, True)


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 128), (12, 4, 64), (7, 1, 128)])
@pytest.mark.parametrize("B,T,P", [(1, 200, 100), (3, 130, 70), (2, 65, 1000), (5, 33, 640), (2, 400, 3)])
def test_shared_prompts(Hq, Hk, D, B, T, P):
    """Questions of different lengths, padded to the longest, then a second round of them."""
    g = torch.Generator().manual_seed(T)
    c, hist = new_shared(g, Hk, P, D, B, 2 * T)
    counts = [T if b == 0 else 1 + (T * (b + 1)) // (B + 3) for b in range(B)]
    starts = step_shared(g, c, hist, [0] * B, counts, T, Hq, False, True)
    step_shared(g, c, hist, starts, counts[::-1], T, Hq, True, True)


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 128), (8, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("B", [1, 3, 20])
@pytest.mark.parametrize("P", [300, 1600])
def test_shared_drafts(Hq, Hk, D, B, P):
    """Steps of a few tokens: one to five groups of 16 rows, short and longer texts."""
    g = torch.Generator().manual_seed(B + P + Hq)
    c, hist = new_shared(g, Hk, P, D, B, 70)
    starts = [0] * B
    for i, T in enumerate((4, 8, 9, 16, 17)):
        counts = [T if (b + i) % 3 else (T * b) // B for b in range(B)]
        starts = step_shared(g, c, hist, starts, counts, T, Hq, True, True)


@gpu
def test_shared_positions_outside():
    """Rows at device positions before the own part or past it are zero and write nothing."""
    g = torch.Generator().manual_seed(5)
    c, _ = new_shared(g, 2, 50, 64, 5, 10)
    q, k = randn(g, 5, 3, 4, 64).to(DEV), randn(g, 5, 3, 2, 64).to(DEV)
    at = torch.tensor([49, 58, 60, -(1 << 62), 1 << 62], device=DEV)
    c.k[0].fill_(7), c.v[0].fill_(7)
    y = fk.attention_shared(q, k, k, c, 0, at)
    live = torch.tensor([[0, 1, 1], [1, 1, 0], [0, 0, 0], [0, 0, 0], [0, 0, 0]], dtype=torch.bool, device=DEV)
    assert (y[~live] == 0).all() and (y[live] != 0).any(-1).all()
    want = torch.full_like(c.k[0], 7)
    want[0, :, :2] = k[0, 1:].transpose(0, 1)
    want[1, :, 8:] = k[1, :2].transpose(0, 1)
    assert torch.equal(c.k[0], want) and torch.equal(c.v[0], want)


@gpu
@pytest.mark.parametrize("T", [1, 5, 100])
def test_shared_values_that_are_not_finite(T):
    """They spoil the rows that see them, in their columns; behind a row they do nothing."""
    g = torch.Generator().manual_seed(T)
    B, Hq, Hk, D, P = 3, 8, 2, 128, 200
    c, hist = new_shared(g, Hk, P, D, B, T + 40)
    c.k[0].fill_(float("nan")), c.v[0].fill_(float("inf"))  # nothing of what is not written counts
    starts = step_shared(g, c, hist, [0] * B, [20] * B, 20, Hq, False, False)
    step_shared(g, c, hist, starts, [T] * B, T, Hq, False, False)
    hist[1]["v"][P + 3, 1, 5] = float("inf")
    c.v[0][1, 1, 3, 5] = float("inf")
    c.k[0][2, 0, 20 + T - 1] = float("nan")  # overwritten by the call
    step_shared(g, c, hist, starts, [T] * B, T, Hq, False, False)
    for b in range(B):
        hist[b]["v"][7, 0, 9] = float("nan")
    c.prefix_v[0][0, 7, 9] = float("nan")
    step_shared(g, c, hist, starts, [T] * B, T, Hq, False, False)


@gpu
def test_shared_text_of_a_plain_cache_and_views():
    """The text in a larger cache's tensors (no copy), heads and tokens in strided tensors."""
    g = torch.Generator().manual_seed(9)
    H, D, P, B = 2, 64, 77, 3
    plain = harness.KVCache(k=[randn(g, 2, H, 100, D).to(DEV)], v=[randn(g, 2, H, 100, D).to(DEV)])
    c = fk.KVCacheShared.of(plain, P, max_batch=B, max_new=16)
    assert c.prefix_k[0].data_ptr() == plain.k[0].data_ptr() and c.cur_len == P
    d = fk.KVCacheShared([t[0, :, :P].contiguous() for t in plain.k], [t[0, :, :P].contiguous() for t in plain.v],
                         max_batch=B, max_new=16)
    qkv = randn(g, B, 4, (6 + 2 * H) * D).to(DEV)
    q, k, v = qkv.split([6 * D, H * D, H * D], -1)
    y = fk.attention_shared(q, k, v, c, 0, P)
    assert y.shape == (B, 4, 6 * D)
    heads = [t.reshape(B, 4, -1, D) for t in (q, k, v)]
    assert torch.equal(fk.attention_shared(*heads, d, 0, P).view(B, 4, -1), y)
    assert torch.equal(c.k[0], d.k[0]) and torch.equal(c.v[0], d.v[0])
    odd = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in heads]  # no unit stride: copied
    assert torch.equal(fk.attention_shared(*odd, d, 0, P).view(B, 4, -1), y)
    off = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in heads]  # off 16 bytes: copied
    assert torch.equal(fk.attention_shared(*off, d, 0, P).view(B, 4, -1), y)
    assert fk.attention_shared(*(t[:0] for t in heads), d, 0, P).shape == (0, 4, 6, D)
    assert fk.attention_shared(*(t[:, :0] for t in heads), d, 0, P).shape == (B, 0, 6, D)


# ------------------------------------------------------------- a window


def step_window(g, c, hist, starts, counts, T, Hq, device_pos, lengths):
    B, Hk, D = len(starts), c.n_kv_heads, c.head_dim
    q, k, v = randn(g, B, T, Hq, D, scale=1.5), randn(g, B, T, Hk, D), randn(g, B, T, Hk, D)
    at = torch.tensor(starts) if device_pos else starts[0]
    y = fk.attention_window(q.to(DEV), k.to(DEV), v.to(DEV), c, 0, at.to(DEV) if device_pos else at,
                            lengths=torch.tensor(counts).to(DEV) if lengths else None)
    for b in range(B):
        n, s = counts[b], starts[b]
        for name, x in (("k", k), ("v", v)):
            hist[b][name] = torch.cat([hist[b][name][:s], x[b, :n]])
        if n:
            e = exact(q[b, :n], hist[b]["k"], hist[b]["v"], s + torch.arange(n), torch.arange(s + n), c.window, c.sinks)
            check(y[b, :n], e, parts(min(T, c.max_step), Hq, Hk))
        assert (y[b, n:] == 0).all()
        # what the cache holds: the first and the last ones (behind the window, where tokens were taken back, theirs)
        end = s + n
        p = torch.cat([torch.arange(min(end, c.sinks)), torch.arange(max(c.sinks, end - c.window), max(c.sinks, end))])
        slot = torch.where(p < c.sinks, p, c.sinks + (p - c.sinks) % c.ring)
        assert torch.equal(c.v[0][b].transpose(0, 1).cpu()[slot], hist[b]["v"][p])
    return [s + n for s, n in zip(starts, counts)]


def new_window(window, sinks, Hk, D, B, max_step=64):
    c = fk.KVCacheWindow.alloc(1, window, sinks=sinks, max_step=max_step, max_batch=B, n_kv_heads=Hk, head_dim=D, device=DEV)
    return c, [{"k": torch.zeros(0, Hk, D).bfloat16(), "v": torch.zeros(0, Hk, D).bfloat16()} for _ in range(B)]


@gpu
@pytest.mark.parametrize("Hq,Hk,D", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (63, 0), (64, 4), (65, 70), (200, 1), (1000, 33)])
def test_window_steps(Hq, Hk, D, window, sinks):
    """From an empty cache through several rounds of the ring, in calls of all sizes."""
    g = torch.Generator().manual_seed(window + sinks + Hq)
    c, hist = new_window(window, sinks, Hk, D, 2)
    starts = [0, 0]
    for T in (1, 2, 1, 17, 9, 64, 300, 1, 5, 64, 30):
        starts = step_window(g, c, hist, starts, [T, T], T, Hq, False, False)
    starts = [s - 20 for s in starts]  # drafts taken back
    for T in (3, 1, 64, 130):
        starts = step_window(g, c, hist, starts, [T, T], T, Hq, False, False)


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 128), (8, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 2), (40, 4), (500, 0), (130, 100)])
@pytest.mark.parametrize("B", [1, 3, 12])
def test_window_ragged(Hq, Hk, D, window, sinks, B):
    g = torch.Generator().manual_seed(B + window)
    c, hist = new_window(window, sinks, Hk, D, B)
    starts = [0] * B
    for i, T in enumerate((40, 1, 200, 5, 1, 64, 1, 90, 2)):
        counts = [T if (b + i) % 4 == 0 else (T * (b % 5)) // 4 % (T + 1) for b in range(B)]
        starts = step_window(g, c, hist, starts, counts, T, Hq, True, True)


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 128), (8, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(300, 4), (1700, 0)])
@pytest.mark.parametrize("B", [1, 3])
def test_window_drafts(Hq, Hk, D, window, sinks, B):
    """Steps of a few tokens: one to five groups of 16 rows, short and longer windows."""
    g = torch.Generator().manual_seed(B + window + Hq)
    c, hist = new_window(window, sinks, Hk, D, B)
    starts = step_window(g, c, hist, [0] * B, [1750 - 30 * b for b in range(B)], 1750, Hq, True, True)
    for i, T in enumerate((4, 8, 9, 16, 17)):
        counts = [T if (b + i) % 3 else T // 2 for b in range(B)]
        starts = step_window(g, c, hist, starts, counts, T, Hq, True, True)


@gpu
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("Hq,Hk,D", [(16, 4, 128), (8, 2, 64)])
def test_norm_and_rope_in_the_call(Hq, Hk, D, window):
    """The same tokens in one call and in calls of all sizes: the same keys, bit for bit, and of each call the
    outputs for them. (The queries as the kernels normalise them: a cache's keys, with q in k's place.)"""
    g = torch.Generator().manual_seed(Hq + window)
    B, T, P, ops = 3, 60, 20, _lib.ops()
    gm, cos, sin = ((torch.rand(*s, generator=g) * 2 - 0.5).bfloat16().to(DEV) for s in ((D,), (B, T, D), (B, T, D)))
    q, k, v = (randn(g, B, T, h, D).to(DEV) for h in (Hq, Hk, Hk))
    text = [randn(g, Hq, P, D).to(DEV) for _ in range(2)]

    def new(heads):
        if window:
            return fk.KVCacheWindow.alloc(1, window, sinks=3, max_step=T, max_batch=B, n_kv_heads=heads, head_dim=D,
                                          device=DEV)
        return fk.KVCacheShared([text[0][:heads]], [text[1][:heads]], max_batch=B, max_new=T)

    def call(c, q, k, v, lo, hi):
        cut = [t[:, lo:hi] for t in (q, k, v, cos, sin)]
        at = torch.full((B,), (0 if window else P) + lo, device=DEV)
        return ops.attention_seg(*cut[:3], gm, gm, 1e-6, 1e-5, *cut[3:], *c.parts(0), window, 0, at, None)

    a, b, d = new(Hk), new(Hk), new(Hq)
    d_call = ops.attention_seg(q, q, q, gm, gm, 1e-6, 1e-6, cos, sin, *d.parts(0), window, 0 if window else P, None, None)
    assert d_call.shape == q.shape
    y = [call(a, q, k, v, 0, T)]
    ends = (1, 4, 12, 28, 45, 60)
    y.append(torch.cat([call(b, q, k, v, lo, hi) for lo, hi in zip((0, *ends), ends)], 1))
    assert torch.equal(a.k[0], b.k[0]) and torch.equal(a.v[0], b.v[0])
    for i in range(B):
        qn, kn = (c.k[0][i, :, :T].transpose(0, 1).cpu() for c in (d, a))
        vn = v[i].cpu()
        if not window:
            kn, vn = (torch.cat([t[:Hk].transpose(0, 1).cpu(), n]) for t, n in zip(text, (kn, vn)))
        at = torch.arange(T) + (0 if window else P)
        e = exact(qn, kn, vn, at, torch.arange(len(kn)), window, 3 if window else 0)
        check(y[0][i], e, 1)
        check(y[1][i], e, 1)


@gpu
@pytest.mark.parametrize("T", [1, 9, 300])
def test_window_far_positions(T):
    """Positions near 2^30 wrap as the near ones do; those outside are zero and write nothing."""
    g = torch.Generator().manual_seed(T)
    window, sinks, B, Hk, Hq, D = 100, 4, 3, 2, 8, 128
    c, _ = new_window(window, sinks, Hk, D, B)
    far = (1 << 30) - 700
    k, v = randn(g, B, 400 + T, Hk, D), randn(g, B, 400 + T, Hk, D)
    fk_, fv_ = randn(g, B, sinks, Hk, D), randn(g, B, sinks, Hk, D)
    c.write(0, fk_.to(DEV), fv_.to(DEV), 0)
    c.write(0, k[:, :400].to(DEV), v[:, :400].to(DEV), far)
    q = randn(g, B, T, Hq, D, scale=1.5)
    y = fk.attention_window(q.to(DEV), k[:, 400:].to(DEV), v[:, 400:].to(DEV), c, 0, far + 400)
    for b in range(B):
        at = torch.cat([torch.arange(sinks), far + torch.arange(400 + T)])
        e = exact(q[b], torch.cat([fk_[b], k[b]]), torch.cat([fv_[b], v[b]]), far + 400 + torch.arange(T), at, window, sinks)
        check(y[b], e, parts(min(T, 64), Hq, Hk))
    before = c.k[0].clone()
    at = torch.tensor([-5 - T, 1 << 30, 1 << 62], device=DEV)
    y = fk.attention_window(q.to(DEV), k[:, :T].to(DEV), v[:, :T].to(DEV), c, 0, at)
    assert (y == 0).all() and torch.equal(before, c.k[0])


@gpu
@pytest.mark.parametrize("T", [1, 5, 64, 200])
def test_window_values_that_are_not_finite(T):
    """What left the window, or was never written, does nothing; what a row sees spoils its column."""
    g = torch.Generator().manual_seed(T)
    c, hist = new_window(50, 4, 2, 64, 2, max_step=256)  # the steps below go back by T
    c.k[0].fill_(float("nan")), c.v[0].fill_(float("-inf"))
    starts = step_window(g, c, hist, [0, 0], [150, 150], 150, 6, False, False)
    slot = lambda p: 4 + (p - 4) % c.ring  # noqa: E731
    c.v[0][:, :, slot(90)] = float("nan")  # sixty before the step
    hist[0]["v"][90], hist[1]["v"][90] = float("nan"), float("nan")
    step_window(g, c, hist, starts, [T, T], T, 6, True, False)
    c.v[0][0, 1, slot(140), 7] = float("inf")  # in the first rows' windows
    hist[0]["v"][140, 1, 7] = float("inf")
    step_window(g, c, hist, starts, [T, T], T, 6, True, False)
    c.k[0][1, 0, slot(100)] = float("inf")  # outside every window of the step
    step_window(g, c, hist, starts, [T, T], T, 6, True, False)


@gpu
def test_window_scores_apart():
    """Scores that rise by far more than the exponential's range, and rows that see one key."""
    g = torch.Generator().manual_seed(0)
    c, hist = new_window(300, 2, 1, 128, 1)
    k, v = randn(g, 1, 320, 1, 128), randn(g, 1, 320, 1, 128)
    k = (k.float() * torch.linspace(0.01, 30, 320).view(1, -1, 1, 1)).bfloat16()
    q = randn(g, 1, 320, 4, 128, scale=4.0)
    for T in (320, 8):
        c.write(0, k.to(DEV), v.to(DEV), 0)
        y = fk.attention_window(q[:, -T:].to(DEV), k[:, -T:].to(DEV), v[:, -T:].to(DEV), c, 0, 320 - T)
        at = torch.arange(320)
        want, size, _ = exact(q[0, -T:], k[0], v[0], at[-T:], at, 300, 2)
        # fp32's scores reach 2^12: their roundings, 2^-24 of it in a few sums, move an exponential by 2^-10
        err = (y[0].double() - want).abs()
        assert (err <= want.abs() * 2.0**-8 + size * (2.0**-6.9 + 2.0**-9)).all()


@gpu
@pytest.mark.parametrize("B,T", [(1, 1), (4, 1), (2, 5)])
def test_graph_replays(B, T):
    """A captured step replays at any positions (and two graphs do not share what they work in)."""
    g = torch.Generator().manual_seed(T)
    Hq, Hk, D, P = 8, 2, 64, 300
    w, _ = new_window(100, 4, Hk, D, B)
    s, _ = new_shared(g, Hk, P, D, B, 400)
    k, v = randn(g, B, 350, Hk, D).to(DEV), randn(g, B, 350, Hk, D).to(DEV)
    w.write(0, k, v, 0), s.write(0, k, v, P)
    copies = copy.deepcopy((w.k, w.v, s.k, s.v))
    qs, ks, vs = (torch.zeros(B, T, h, D, dtype=torch.bfloat16, device=DEV) for h in (Hq, Hk, Hk))
    pos = torch.zeros(B, dtype=torch.long, device=DEV)
    run = lambda: (fk.attention_window(qs, ks, vs, w, 0, pos), fk.attention_shared(qs, ks, vs, s, 0, pos + P))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, out = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            out.append(run())
    for i in range(4):
        at = torch.tensor([350 - (7 * i + b) % 40 for b in range(B)], device=DEV)
        new = [randn(g, *t.shape).to(DEV) for t in (qs, ks, vs)]
        res = []
        for mode in range(3):
            for t, old in zip((w.k, w.v, s.k, s.v), copies):
                t[0].copy_(old[0])
            for t, x in zip((qs, ks, vs), new):
                t.copy_(x)
            pos.copy_(at)
            if mode == 2:
                res.append([t.clone() for t in run()])
            else:
                graphs[mode].replay()
                res.append([t.clone() for t in out[mode]])
            torch.cuda.synchronize()
        for a, b, e in zip(*res):
            assert torch.equal(a, b) and torch.equal(a, e)


@gpu
def test_streams():
    """Calls on two streams at once, each with its own cache."""
    g = torch.Generator().manual_seed(3)
    caches = [new_shared(g, 2, 3000, 128, 4, 16)[0] for _ in range(2)]
    q, k = randn(g, 4, 2, 8, 128).to(DEV), randn(g, 4, 2, 2, 128).to(DEV)
    want = [fk.attention_shared(q, k, k, c, 0, 3000) for c in caches]
    torch.cuda.synchronize()
    got = [[], []]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(fk.attention_shared(q, k, k, caches[i], 0, 3000))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# ------------------------------------------------------------- models


def model_of(**kw):
    c = harness.Cfg(vocab_size=211, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                    intermediate_size=512, max_position_embeddings=700)
    m = harness.tiny_model(c, state=harness.tiny_state(c, embed_scale=0.3), device=DEV)
    return m, fk.apply_triton_kernels(copy.deepcopy(m), **kw)


@gpu
@pytest.mark.parametrize("kw", [dict(), dict(int8=True, a8=True, linear_down_o=True, fuse_norm=True)])
def test_batch_generate(kw):
    """Several continuations of one text are what each would be by itself, up to ties that rounding decides; the
    step graph answers as the eager step does."""
    m, f = model_of(**kw)
    g = torch.Generator().manual_seed(2)
    text = torch.randint(0, 211, (150,), generator=g).tolist()
    tails = [torch.randint(0, 211, (n,), generator=g).tolist() for n in (1, 7, 30, 4)]
    out = harness.batch_generate(f, text, tails, 6, DEV)
    assert out == harness.batch_generate(f, text, tails, 6, DEV, graph=True)
    assert [len(o) for o in out] == [6] * 4
    with torch.inference_mode():
        for t, o in zip(tails, out):
            logits = harness.teacher_forced_logits(f, text + t + o, DEV)[len(text) + len(t) - 1 : -1]
            best = logits.max(-1).values
            took = logits.gather(1, torch.tensor(o, device=DEV)[:, None])[:, 0]
            # the other cache's kernel rounds p otherwise (and 8-bit codes move by one): near ties only
            assert (best - took <= 0.05 * logits.std()).all(), (best - took, logits.std())


@gpu
@pytest.mark.parametrize("window,sinks", [(32, 4), (400, 4)])
def test_window_model(window, sinks):
    """A window that holds all of the text is the plain cache; a short one is attention with that mask."""
    m, f = model_of()
    ids = torch.randint(0, 211, (1, 250), generator=torch.Generator().manual_seed(4)).to(DEV)
    with torch.inference_mode():
        cache = f.alloc_cache(300, window=window, sinks=sinks)
        a = torch.cat([f(p, cache) for p in ids.split([200, 1, 1, 40, 8], 1)], 1)
        if window > 250:
            b = f(ids, f.alloc_cache(300), start_pos=0)
            assert (a.float() - b.float()).abs().max() <= 0.05 * b.float().std()
        else:
            # a token's answer after all but the window and the sinks were other tokens: the first layer's
            # attention does not see them
            L = f.layers[0]
            x = torch.randn(1, 250, 256, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
            y = x.clone()
            y[:, sinks : 250 - window] = 0.5
            ys = []
            for t in (x, y):
                c = f.alloc_cache(300, window=window, sinks=sinks)
                ys.append(L.attn(t, kv_cache=c, layer_idx=0, cos=f.rope_cos[:250], sin=f.rope_sin[:250], start_pos=0))
            assert torch.equal(ys[0][:, -1], ys[1][:, -1]) and not torch.equal(ys[0][:, 100], ys[1][:, 100])
    prompt = ids[0, :100].tolist()
    out = harness.greedy_generate(f, prompt, 12, DEV, window=window)
    assert out == harness.graph_greedy_generate(f, prompt, 12, DEV, window=window)


@gpu
def test_rope_in_torch_is_the_same():
    """Where the norms carry hooks QK-norm and RoPE run in torch, on the same values."""
    m, f = model_of()
    ids = torch.randint(0, 211, (3, 5), generator=torch.Generator().manual_seed(4)).to(DEV)
    text = torch.randint(0, 211, (1, 40), generator=torch.Generator().manual_seed(5)).to(DEV)
    with torch.inference_mode():
        plain = f.alloc_cache(64)
        f(text, plain, start_pos=0)
        ys = []
        for hook in (False, True):
            if hook:
                for layer in f.layers:
                    layer.attn.q_norm.register_forward_hook(lambda *a: None)
            c = fk.KVCacheShared.of(plain, 40, max_batch=3, max_new=20)
            a = f(ids, c)
            ys.append((a, f(ids[:, :1], c, start_pos=torch.tensor([45, 44, 42], device=DEV))))
        for a, b in zip(*ys):
            assert torch.equal(a, b)
