"""The 8-bit key/value cache and attention over it against 64 bits."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from llms_amd import _lib
from llms_amd import kernels as fk

DEV = "cuda"
BLOCK = 64


def tokens(seed, B, T, H, D, spread=0.3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, H, D, generator=g) * (spread * torch.randn(H, D, generator=g)).exp()).bfloat16()


def pack(x):
    """[n * 64, H, D] tokens -> (codes, scales, values in fp32) of the whole blocks."""
    w = x.float().view(-1, BLOCK, *x.shape[1:])
    fin = w.isfinite()
    top = torch.where(fin, w.abs(), 0.0).amax((1, 3), keepdim=True)
    q = torch.where(top > 0, 127 * w.double() / top, 0.0).round().float()  # ties and sizes exact in 64 bits
    s = top / 127
    v = torch.where(fin, q * s, math.nan)
    return q, s, v.view(x.shape)


def held(x, length):
    """What a cache of `length` tokens x [P, H, D] holds, in fp32."""
    n = length // BLOCK * BLOCK
    return torch.cat([pack(x[:n])[2], x[n:length].float()]) if n else x[:length].float()


def attend(q, k, v, first):
    """[T, Hq, D] queries at first .. over values [P, H, D], in 64 bits: the output,
    sum p |v| and the largest score's sum of absolute products, for the tolerance."""
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    k, v = (t.double().repeat_interleave(G, 1) for t in (k, v))
    x = torch.einsum("thd,phd->htp", q.double(), k) * D**-0.5
    size = torch.einsum("thd,phd->htp", q.double().abs(), k.abs()).amax(-1) * D**-0.5
    hidden = torch.arange(k.shape[0])[None] > torch.arange(first, first + T)[:, None]
    x = x.masked_fill(hidden, -math.inf)
    p = x.softmax(-1)
    y = torch.einsum("htp,phd->thd", p, v)
    return y, torch.einsum("htp,phd->thd", p, v.abs()), size.T[..., None], v.abs().amax(0)[None], p.amax(-1).T[..., None]


def check(y, q, k, v, first):
    """y is rounded to bf16 (2^-8). Each p is off by 2^-12 of itself for fp16 (or by
    2^-25 of the row's largest, where it is under fp16's normal numbers: then a row's keys
    together are off by n 2^-25 of max |v| at its largest p) and by its score's fp32
    error, 2^-20 of the score's absolute products; its sum, in fp32, by the latter."""
    e, pv, size, vmax, top = attend(q, k, v, first)
    tol = e.abs() * 2.0**-8 + pv * (2.0**-11 + size * 2.0**-19) + k.shape[0] * 2.0**-25 * vmax * top + 1e-30
    err = (y.cpu().double() - e).abs()
    assert (err <= tol).all(), (err / tol).max()


def new(P, H, D, B=1, layers=1, garbage=True):
    """A cache whose buffers hold anything, as memory never written does."""
    c = fk.KVCache8.alloc(layers, P, max_batch=B, n_kv_heads=H, head_dim=D, device=DEV)
    if garbage:
        for i in range(layers):
            for t in c.parts(i)[:6]:
                t.random_(-128, 128) if t.dtype == torch.int8 else t.fill_(math.nan)
    return c


# ------------------------------------------------------------- refusals (CPU)


def test_refusals_on_the_cpu():
    c = fk.KVCache8.alloc(2, 100, max_batch=2, n_kv_heads=2, head_dim=64, device="cpu")
    assert c.parts(1)[0].shape == (2, 2, 2, 64, 64) and c.max_seq == 100 and len(c.tails()) == 2
    q, k = torch.zeros(1, 3, 4, 64).bfloat16(), torch.zeros(1, 3, 2, 64).bfloat16()
    with pytest.raises(ValueError, match="HIP"):
        fk.attention_kv8(q, k, k, c, 0, 0)
    with pytest.raises(ValueError, match="HIP"):
        c.write(0, k, k, 0)
    with pytest.raises(ValueError, match="HIP"):
        c.read(0, 0, 5)
    with pytest.raises(ValueError, match="must be"):
        fk.attention_kv8(q, k, k[:, :2], c, 0, 0)
    with pytest.raises(ValueError, match="must be"):
        c.write(0, k[..., :32], k[..., :32], 0)
    with pytest.raises(ValueError, match="holds 2"):
        c.write(0, k.expand(3, 3, 2, 64), k.expand(3, 3, 2, 64), 0)
    with pytest.raises(TypeError, match="bfloat16"):
        c.write(0, k.float(), k.float(), 0)
    for kw in (dict(head_dim=96), dict(max_seq=0), dict(max_seq=(1 << 23) + 1), dict(n_kv_heads=0), dict(max_batch=0),
               dict(num_layers=0)):
        a = dict(dict(num_layers=1, max_seq=64, n_kv_heads=1, head_dim=64, max_batch=1, device="meta"), **kw)
        with pytest.raises(ValueError, match="KVCache8"):
            fk.KVCache8.alloc(**a)
    with pytest.raises(ValueError, match="batch"):
        c.read(0, 0, 5, batch=3)
    for p in (98, -1, (1 << 63) - 1):
        with pytest.raises(ValueError, match="outside"):
            c.read(0, p, 3)
    from llms_amd import harness as h

    m = h.tiny_model(h.Cfg(head_dim=64))
    with pytest.raises(TypeError, match="apply_triton_kernels"):
        m(torch.zeros(1, 2, dtype=torch.long), m.alloc_cache(16, kv8=True))


class Args(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v")] + \
        [(n, ctypes.c_int64) for n in ("ldq", "ldk", "ldv")] + \
        [(n, ctypes.c_void_p) for n in ("q_gamma", "k_gamma", "cos", "sin")] + \
        [(n, ctypes.c_int64) for n in ("ld_cos", "ld_sin")] + \
        [(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "k_scale", "v_scale", "k_tail", "v_tail", "tail_block",
                                        "y")] + \
        [(n, ctypes.c_int64) for n in ("B", "T", "n_heads", "n_kv_heads", "head_dim", "cache_len", "pos")] + \
        [("pos_dev", ctypes.c_void_p), ("pos_stride", ctypes.c_int64), ("lengths", ctypes.c_void_p),
         ("q_eps", ctypes.c_float), ("k_eps", ctypes.c_float)]


def test_c_entry_refusals():
    lib = _lib.capi()
    P = 4096  # never dereferenced: every call below is refused before a launch
    need = lib.fp_kv8_workspace_bytes(2, 3, 4, 2, 128, 103, 1)
    assert need > 0 and lib.fp_kv8_workspace_bytes(2, 3, 4, 2, 96, 103, 1) == 0
    assert lib.fp_kv8_workspace_bytes(2, 3, 4, 2, 128, 103, 0) == 0
    assert lib.fp_kv8_workspace_bytes(2, 3, 4, 2, 128, 8000, 0) > 0

    def call(fn="attention", ws=P, nb=need, ko=P, **kw):
        a = dict(q=P, k=P, v=P, ldq=512, ldk=256, ldv=256, k_codes=P, v_codes=P, k_scale=P, v_scale=P, k_tail=P,
                 v_tail=P, tail_block=P, y=P, B=2, T=3, n_heads=4, n_kv_heads=2, head_dim=128, cache_len=200, pos=100)
        a.update(kw)
        s = Args(**a)
        if fn == "attention":
            return lib.fp_kv8_attention(ctypes.byref(s), ws, nb, None)
        if fn == "write":
            return lib.fp_kv8_write(ctypes.byref(s), None)
        return lib.fp_kv8_read(ctypes.byref(s), ko, P, None)

    NULL, SHAPE, STRIDE, WORKSPACE = 1, 2, 3, 6
    for fn in ("attention", "write", "read"):
        for kw in (dict(B=0), dict(T=0), dict(n_kv_heads=0), dict(head_dim=96), dict(cache_len=0), dict(pos=-1),
                   dict(pos=198), dict(pos=(1 << 63) - 1), dict(cache_len=(1 << 23) + 1), dict(pos_stride=2),
                   dict(T=1 << 30)):
            assert call(fn, **kw) == SHAPE, (fn, kw)
        for n in ("k_codes", "v_codes", "k_scale", "v_scale", "k_tail", "v_tail", "tail_block"):
            assert call(fn, **{n: None}) == NULL, (fn, n)
            assert call(fn, **{n: P + 2}) == STRIDE, (fn, n)
    for fn in ("attention", "write"):
        for kw in (dict(ldk=255), dict(ldv=252), dict(ldk=258), dict(k=P + 2), dict(v=P + 4)):
            assert call(fn, **kw) == STRIDE, (fn, kw)
        assert call(fn, k=None) == NULL and call(fn, v=None) == NULL
    for kw in (dict(n_heads=3), dict(n_heads=1), dict(cos=P, sin=P, ld_cos=128, ld_sin=128, q_eps=-1.0)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(ldq=511), dict(q=P + 2), dict(y=P + 4), dict(cos=P, sin=P, ld_cos=127, ld_sin=128),
               dict(pos_dev=P + 4), dict(lengths=P + 4)):
        assert call(**kw) == STRIDE, kw
    for kw in (dict(q=None), dict(y=None), dict(cos=P, ld_cos=128, ld_sin=128), dict(q_gamma=P),
               dict(q_gamma=P, k_gamma=P)):
        assert call(**kw) == NULL, kw
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=P + 8)):
        assert call(**kw, cos=P, sin=P, ld_cos=128, ld_sin=128) == WORKSPACE, kw
    assert call("read", ko=None) == NULL and call("read", ko=P + 4) == STRIDE


# ------------------------------------------------------------------- format


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [1, 63, 64, 65, 130, 384, 1000])
def test_what_the_cache_holds(P, D):
    """Exactly the packing's values, whatever the calls that wrote them."""
    H = 3
    k, v = tokens(P, 1, P, H, D), tokens(P + 1, 1, P, H, D)
    v[:, :, 1] *= 1e-3
    ek, ev = held(k[0], P), held(v[0], P)
    g = torch.Generator().manual_seed(P)
    for cuts in ([P], [1] * P if P <= 130 else [7] * (P // 7) + [P % 7],
                 torch.diff(torch.cat([torch.tensor([0]), torch.randperm(P, generator=g)[:5].sort().values,
                                       torch.tensor([P])])).tolist()):
        c = new(P + 3, H, D)
        at = 0
        for n in cuts:
            if n:
                c.write(0, k[:, at : at + n].to(DEV), v[:, at : at + n].to(DEV), at)
            at += n
        rk, rv = c.read(0, 0, P)
        assert rk.dtype == torch.float32 and rk.shape == (1, P, H, D)
        assert torch.equal(rk[0].cpu(), ek) and torch.equal(rv[0].cpu(), ev), cuts[:8]
        n = P // 2
        assert torch.equal(c.read(0, n, P - n)[1][0].cpu(), ev[n:])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("first,then", [(37, 91), (37, 100), (63, 65), (63, 66), (1, 191), (5, 250), (70, 129), (64, 130)])
def test_a_write_from_inside_a_block_over_the_next_ones(first, then, D):
    """Old rows are read from the ring slot that a later block of the same call goes to."""
    B, H, P = 8, 4, first + then + 70
    k, v = tokens(first, B, P, H, D), tokens(then, B, P, H, D)
    kd, vd = k.to(DEV), v.to(DEV)
    c = new(P, H, D, B)
    at = 0
    for n in (first, then, 1, 69):
        c.write(0, kd[:, at : at + n], vd[:, at : at + n], at)
        at += n
        rk, rv = (t.cpu() for t in c.read(0, 0, at))
        for b in range(B):
            assert torch.equal(rk[b], held(k[b], at)) and torch.equal(rv[b], held(v[b], at)), (b, at)


@pytest.mark.gpu
def test_packing_ties_zeros_and_sizes():
    x = torch.zeros(1, 256, 1, 64)
    x[0, 0, 0, 0], x[0, 1, 0] = 3.0, 1.5              # half of the largest: 63.5 is a tie
    x[0, 64:128] = 0                                  # a block of zeros
    x[0, 128, 0, :2] = torch.tensor([1e-38, 5e-39])   # at the edge of the normal numbers
    x[0, 192] = 3e38
    x = x.bfloat16()
    c = new(256, 1, 64)
    c.write(0, x.to(DEV), -x.to(DEV), 0)
    k, v = (t[0].cpu() for t in c.read(0, 0, 256))
    assert torch.equal(k, held(x[0], 256)) and torch.equal(v, -k)
    assert k[1, 0, 0] == 64 * (torch.tensor(3.0) / 127) and (k[64:128] == 0).all()


# ---------------------------------------------------------------- attention

CASES = [(1, 1, 0, 4, 2, 64), (1, 1, 63, 4, 2, 128), (1, 1, 64, 8, 1, 128), (2, 1, 333, 16, 8, 128),
         (1, 5, 60, 32, 8, 128), (1, 16, 100, 4, 1, 64), (1, 17, 47, 4, 1, 128), (1, 9, 1000, 7, 1, 64),
         (3, 2, 126, 6, 3, 128), (1, 64, 0, 2, 2, 64), (1, 64, 64, 1, 1, 128), (1, 65, 0, 1, 1, 128),
         (1, 100, 37, 8, 2, 128), (2, 130, 62, 6, 2, 64), (1, 700, 0, 4, 1, 128), (1, 300, 1001, 8, 8, 64),
         (1, 33, 3000, 8, 2, 128), (1, 3, 5000, 2, 1, 128), (4, 600, 5, 16, 8, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,pos,Hq,Hk,D", CASES)
def test_attention(B, T, pos, Hq, Hk, D):
    P = pos + T
    k, v, q = tokens(1, B, P, Hk, D), tokens(2, B, P, Hk, D), tokens(3, B, T, Hq, D) * 1.5
    c = new(P + 70, Hk, D, B + 1)
    kd, vd, qd = k.to(DEV), v.to(DEV), q.to(DEV)
    if pos:
        c.write(0, kd[:, :pos], vd[:, :pos], 0)
    y = fk.attention_kv8(qd, kd[:, pos:], vd[:, pos:], c, 0, pos)
    assert y.shape == (B, T, Hq, D) and y.dtype == torch.bfloat16
    again = fk.attention_kv8(qd, kd[:, pos:], vd[:, pos:], c, 0, torch.tensor(pos, device=DEV))
    for b in range(B):
        ek, ev = held(k[b], P), held(v[b], P)
        check(y[b], q[b], ek, ev, pos)
        check(again[b], q[b], ek, ev, pos)
        assert torch.equal(c.read(0, pos, T, batch=B)[0][b].cpu(), ek[pos:])


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(1, 128), (5, 64), (90, 128), (200, 64)])
def test_sequences_of_their_own_lengths(T, D):
    """Positions and lengths per sequence; sequences that are not there; rows behind a
    sequence's end are zero and other sequences' memory is left as it was."""
    B, Hq, Hk, S = 6, 8, 2, 700
    starts = [0, 63, 400, -3, S - 2, S + 5]
    lens = [T, max(T - 3, 0), T, T, T, T]
    lens[2] = 0
    k, v, q = tokens(1, B, S, Hk, D), tokens(2, B, S, Hk, D), tokens(3, B, T, Hq, D)
    c = new(S, Hk, D, B)
    place = torch.tensor(starts, device=DEV)
    before = place.clamp(0, S)
    c.write(0, k.to(DEV), v.to(DEV), 0, lengths=before)
    idx = [[min(max(p + t, 0), S - 1) for t in range(T)] for p in starts]
    nk, nv = (torch.stack([t[b, idx[b]] for b in range(B)]) for t in (k, v))
    kept = [t[5].clone() for t in c.parts(0)] + [t[2].clone() for t in c.parts(0)]
    y = fk.attention_kv8(q.to(DEV), nk.to(DEV), nv.to(DEV), c, 0, place, lengths=torch.tensor(lens, device=DEV)).cpu()
    for old, t in zip(kept, [t[5] for t in c.parts(0)] + [t[2] for t in c.parts(0)]):
        assert torch.equal(old.view(torch.uint8), t.view(torch.uint8))  # nothing of theirs was written
    for b in range(B):
        live = [t for t in range(lens[b]) if 0 <= starts[b] + t < S]
        dead = [t for t in range(T) if t not in live]
        assert (y[b, dead] == 0).all(), b
        if live:
            first, end = starts[b] + live[0], starts[b] + live[-1] + 1
            check(y[b, live], q[b, live], held(k[b], end), held(v[b], end), first)


@pytest.mark.gpu
@pytest.mark.parametrize("back", [190, 140, 127, 65, 64, 10, 0])
def test_going_back(back):
    """A step that takes tokens back: bf16 within the last two blocks, further back the
    packed values go on as the block's tokens."""
    P, H, D = 200, 2, 128
    k, v = tokens(1, 1, P, H, D), tokens(2, 1, P, H, D)
    c = new(400, H, D)
    c.write(0, k.to(DEV), v.to(DEV), 0)
    n = 150
    k2, v2, q = tokens(3, 1, n, H, D), tokens(4, 1, n, H, D), tokens(5, 1, n, 4, D)
    y = [fk.attention_kv8(q[:, t : t + m].to(DEV), k2[:, t : t + m].to(DEV), v2[:, t : t + m].to(DEV), c, 0, back + t)
         for t, m in ((0, 1), (1, 4), (5, 40), (45, 105))]

    def then(x, x2):
        x = x[0].clone()
        blk = back // BLOCK
        if blk < (P - 1) // BLOCK - 1:  # out of the ring: what the codes say
            x[blk * BLOCK : back] = pack(x[blk * BLOCK : (blk + 1) * BLOCK])[2][: back % BLOCK].bfloat16()
        return torch.cat([x[:back], x2[0]])

    ek, ev = then(k, k2), then(v, v2)
    at = back
    for out in y:
        m = out.shape[1]
        check(out[0], q[0, at - back : at - back + m], held(ek, at + m), held(ev, at + m), at)
        at += m
    rk, rv = c.read(0, 0, back + n)
    assert torch.equal(rk[0].cpu(), held(ek, back + n)) and torch.equal(rv[0].cpu(), held(ev, back + n))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70])
def test_non_finite_entries(T):
    """They are NaN in the cache, spoil the rows that see them (and, as 0 * NaN, none
    before them in another call), and leave the other entries of their block alone."""
    P, H, D = 200, 2, 64
    k, v = tokens(1, 1, P, H, D), tokens(2, 1, P, H, D)
    k[0, 70, 0, 3], k[0, 150, 1, 5], v[0, 80, 0, 7] = math.nan, math.inf, -math.inf
    c = new(P + T, H, D)
    c.write(0, k.to(DEV), v.to(DEV), 0)
    rk, rv = (t[0].cpu() for t in c.read(0, 0, P))
    ek, ev = held(k[0], P), held(v[0], P)
    for r, e in ((rk, ek), (rv, ev)):
        assert torch.equal(r.isnan(), e.isnan()) and torch.equal(r.nan_to_num(), e.nan_to_num())
    assert rk[70, 0, 3].isnan() and rv[80, 0, 7].isnan() and rk.isnan().sum() == 2
    q, k2, v2 = tokens(3, 1, T, 4, D), tokens(4, 1, T, H, D), tokens(5, 1, T, H, D)
    y = fk.attention_kv8(q.to(DEV), k2.to(DEV), v2.to(DEV), c, 0, 50).cpu()  # before all of them
    # (their block, long out of the ring, goes on from its packed values)
    kk, vv = (torch.cat([pack(a[0, :64])[2][:50].bfloat16(), b[0]]) for a, b in ((k, k2), (v, v2)))
    check(y[0], q[0], held(kk, 50 + T), held(vv, 50 + T), 50)
    c.write(0, k.to(DEV), v.to(DEV), 0)
    y = fk.attention_kv8(q.to(DEV), k2.to(DEV), v2.to(DEV), c, 0, P).cpu()
    assert y[0, :, :2].isnan().all() and y[0, :, 2:].isnan().all()  # both heads hold a bad key
    k[0, 70, 0, 3] = 0.5
    c.write(0, k.to(DEV), v.to(DEV), 0)
    y = fk.attention_kv8(q.to(DEV), k2.to(DEV), v2.to(DEV), c, 0, P).cpu()
    assert y[0, :, :2, 7].isnan().all() and y[0, :, :2].isnan().sum() == 2 * T  # the bad value's column


@pytest.mark.gpu
@pytest.mark.parametrize("rise", [1.0, 5.0, 7.9, 40.0, -5.0])
@pytest.mark.parametrize("T,D", [(100, 64), (70, 128), (3, 128)])
def test_a_maximum_that_rises_by_blocks(T, D, rise):
    """Scores that grow (or fall) by 2^rise from block to block: what p is relative to
    follows in steps or at once, and every row comes out the same."""
    P = 1300
    u = torch.ones(D) * D**-0.25
    at = (torch.arange(P) // BLOCK).float() * rise * math.log(2)
    k = (at[:, None, None] * u + 0.1 * tokens(1, 1, P, 1, D)[0].float()).bfloat16()[None]
    v, q = tokens(2, 1, P, 1, D), (u + 0.02 * tokens(3, 1, T, 2, D).float()).bfloat16()
    c = new(P, 1, D)
    c.write(0, k[:, : P - T].to(DEV), v[:, : P - T].to(DEV), 0)
    y = fk.attention_kv8(q.to(DEV), k[:, P - T :].to(DEV), v[:, P - T :].to(DEV), c, 0, P - T)
    check(y[0], q[0], held(k[0], P), held(v[0], P), P - T)


@pytest.mark.gpu
def test_values_of_all_sizes():
    """Blocks whose scales differ by many powers of two, tails far from one."""
    P, H, D = 300, 1, 128
    k, v = tokens(1, 1, P, H, D), tokens(2, 1, P, H, D).float()
    for b, f in enumerate((1e-30, 1e30, 1.0, 1e-12, 1e-38)):
        v[:, b * 64 : b * 64 + 64] *= f
    v = v.bfloat16()
    for P in (64, 100, 200, 260, 300):
        c = new(400, H, D)
        c.write(0, k[:, : P - 3].to(DEV), v[:, : P - 3].to(DEV), 0)
        for T in (3,):
            q = tokens(7, 1, T, 2, D)
            y = fk.attention_kv8(q.to(DEV), k[:, P - T : P].to(DEV), v[:, P - T : P].to(DEV), c, 0, P - T)
            check(y[0], q[0], held(k[0], P), held(v[0], P), P - T)


@pytest.mark.gpu
def test_long_cache():
    """65000 tokens: many ranges of keys, a step and a chunk of a prompt."""
    P, H, D = 65000, 2, 128
    k, v = tokens(1, 1, P + 80, H, D), tokens(2, 1, P + 80, H, D)
    c = new(P + 100, H, D)
    c.write(0, k[:, :P].to(DEV), v[:, :P].to(DEV), 0)
    for T in (1, 80):
        q = tokens(3, 1, T, 4, D)
        y = fk.attention_kv8(q.to(DEV), k[:, P : P + T].to(DEV), v[:, P : P + T].to(DEV), c, 0, P)
        check(y[0], q[0], held(k[0], P + T), held(v[0], P + T), P)


@pytest.mark.gpu
def test_strides_and_empty_calls():
    B, T, Hq, Hk, D = 2, 5, 4, 2, 64
    flat = tokens(1, B, T, Hq + 2 * Hk, D).view(B, T, -1).to(DEV)
    q, k, v = (t.view(B, T, -1, D) for t in flat.split([Hq * D, Hk * D, Hk * D], -1))
    c = new(50, Hk, D, B)
    y = fk.attention_kv8(q, k, v, c, 0, 0)
    for f in (lambda t: t.contiguous(), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
              lambda t: torch.stack([t, t], -1)[..., 0], lambda t: torch.cat([t[..., :1], t], -1)[..., 1:]):
        assert torch.equal(fk.attention_kv8(f(q), f(k), f(v), c, 0, 0), y)
    same = fk.attention_kv8(q[:1].expand(2, -1, -1, -1), k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), c, 0, 0)
    assert torch.equal(same[0], y[0]) and torch.equal(same[1], y[0])
    assert fk.attention_kv8(q[:, :0], k[:, :0], v[:, :0], c, 0, 3).shape == (B, 0, Hq, D)
    assert fk.attention_kv8(q[:0], k[:0], v[:0], c, 0, 3).shape == (0, T, Hq, D)
    c.write(0, k[:, :0], v[:, :0], 2)


@pytest.mark.gpu
def test_stream_and_graph():
    B, Hq, Hk, D, S = 2, 8, 2, 128, 400
    k, v, q = (tokens(i, B, S, h, D).to(DEV) for i, h in ((1, Hk), (2, Hk), (3, Hq)))
    c, e = new(S, Hk, D, B), new(S, Hk, D, B)
    T = 2
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in (c, e):
            x.write(0, k[:, :120], v[:, :120], 0)
        a = fk.attention_kv8(q[:, :T], k[:, 120 : 120 + T], v[:, 120 : 120 + T], c, 0, 120)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, fk.attention_kv8(q[:, :T], k[:, 120 : 120 + T], v[:, 120 : 120 + T], e, 0, 120))
    qs, ks, vs = (t[:, :T].clone() for t in (q, k, v))
    pos = torch.tensor([122, 60], device=DEV)
    warm = new(S, Hk, D, B)
    fk.attention_kv8(qs, ks, vs, warm, 0, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fk.attention_kv8(qs, ks, vs, c, 0, pos)
    at = torch.tensor([122, 60], device=DEV)
    for i in range(40):  # across the ends of blocks
        for dst, src in ((qs, q), (ks, k), (vs, v)):
            dst.copy_(src[:, 130 + i : 130 + i + T])
        pos.copy_(at)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fk.attention_kv8(qs, ks, vs, e, 0, at)), i
        at = at + T


@pytest.mark.gpu
def test_place_and_gradients_are_refused():
    c = new(64, 2, 64, 2, garbage=False)
    q, k = torch.zeros(2, 3, 4, 64, device=DEV).bfloat16(), torch.zeros(2, 3, 2, 64, device=DEV).bfloat16()
    for p in (-1, 62, torch.tensor([0], device=DEV), torch.tensor([0, 1], device=DEV).int(), torch.tensor(0),
              torch.zeros(4, device=DEV, dtype=torch.long)[::2]):
        with pytest.raises(ValueError):
            fk.attention_kv8(q, k, k, c, 0, p)
    for p in (1.0, True, None):
        with pytest.raises(TypeError):
            fk.attention_kv8(q, k, k, c, 0, p)
    for n in (torch.tensor([1], device=DEV), [1, 2], torch.tensor([1, 2])):
        with pytest.raises(ValueError, match="lengths"):
            fk.attention_kv8(q, k, k, c, 0, 0, lengths=n)
    with pytest.raises(ValueError, match="multiple"):
        fk.attention_kv8(q[:, :, :3], k, k, c, 0, 0)
    with pytest.raises(ValueError, match="must be"):
        fk.attention_kv8(q[..., :32], k, k, c, 0, 0)
    with pytest.raises(IndexError):
        c.write(1, k, k, 0)
    with pytest.raises(RuntimeError, match="gradients"):
        fk.attention_kv8(q.requires_grad_(), k, k, c, 0, 0)


# --------------------------------------------------------------------- model


def model(**kw):
    from llms_amd import harness as h

    c = h.Cfg(hidden_size=192, intermediate_size=320, head_dim=64, max_position_embeddings=512)
    m = h.tiny_model(c, state=h.tiny_state(c, seed=4, embed_scale=0.3), device=DEV)
    return h, fk.apply_triton_kernels(m, **kw)


@pytest.mark.gpu
def test_norm_and_rope_in_the_write():
    """The module's path (QK-norm and RoPE in the kernel) against the same steps in torch."""
    h, m = model()
    attn = m.layers[0].attn
    x = tokens(1, 2, 90, 1, 192).view(2, 90, 192).to(DEV)
    a, b = (m.alloc_cache(128, max_batch=2, kv8=True) for _ in range(2))
    from llms_amd.kernels._eager import apply_rope

    with torch.inference_mode():
        for lo, hi in ((0, 1), (1, 70), (70, 75), (75, 90)):
            cos, sin = m.rope_cos[lo:hi], m.rope_sin[lo:hi]
            y = attn(x[:, lo:hi], kv_cache=a, layer_idx=1, cos=cos, sin=sin, start_pos=lo)
            q, k, v = (t.view(2, hi - lo, -1, 64) for t in attn.project(x[:, lo:hi]))
            q, k = apply_rope(attn.q_norm(q).transpose(1, 2), attn.k_norm(k).transpose(1, 2), cos, sin)
            z = fk.attention_kv8(q.transpose(1, 2), k.transpose(1, 2), v, b, 1, lo)
            assert torch.equal(y, attn.o(z.view(2, hi - lo, -1)))
        for s, t in zip(a.read(1, 0, 90), b.read(1, 0, 90)):
            assert torch.equal(s, t)
        attn.q_norm.forward = lambda t: h.RMSNorm.forward(attn.q_norm, t) * 2  # not the plain norm any more
        w = attn(x[:, 75:], kv_cache=a, layer_idx=1, cos=cos, sin=sin, start_pos=75)
        assert not torch.equal(w, y)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(fuse_norm=True, linear_down_o=True),
                                dict(int4=True, w4_group=64, fuse_norm=True, linear_down_o=True)])
def test_model_over_the_cache(kw):
    """A model over the 8-bit cache, in one call, in chunks and token by token, against the
    same projections around 64-bit attention over what the cache holds. Both round
    to bf16 at the same points but for the attention's sums: a flipped rounding (2^-8) in a
    few of the ~30 roundings of two layers, sqrt(30) 2^-8 = 2e-2 of the logits' size."""
    h, m = model(**kw)
    g = torch.Generator().manual_seed(1)
    text = torch.randint(0, 32, (200,), generator=g).tolist()
    ids = torch.tensor([text], device=DEV)
    for cuts in ([200], [130, 1, 1, 1, 5, 62]):
        with torch.inference_mode():
            cache = m.alloc_cache(256, kv8=True)
            got = torch.cat([m(i, cache) for i in ids.split(cuts, 1)], 1).float()
        assert cache.cur_len == 200
        want = over_held_values(m, ids, cuts).float()
        assert (got - want).norm() <= 2e-2 * want.norm(), cuts
    scores = h.teacher_forced_logprobs(m, text, DEV, top_k=3, kv8=True)
    with torch.inference_mode():
        logits = m(ids, m.alloc_cache(256, kv8=True), start_pos=0)
        direct = fk.token_logprobs(logits[0, :-1], ids[0, 1:], 3)
    assert all(torch.equal(a, b) for a, b in zip(scores, direct))
    prompt = text[:70]
    assert h.greedy_generate(m, prompt, 20, DEV, kv8=True) == h.graph_greedy_generate(m, prompt, 20, DEV, kv8=True)


@torch.inference_mode()
def over_held_values(m, ids, cuts):
    """The swapped model's forward with torch attention over the values that an 8-bit
    cache holds after each chunk."""
    from llms_amd.kernels._eager import apply_rope

    seen = [([], []) for _ in m.layers]
    out, at = [], 0
    for chunk in ids.split(cuts, 1):
        T = chunk.shape[1]
        x = m.embed(chunk)
        for layer, (ks, vs) in zip(m.layers, seen):
            attn = layer.attn
            q, k, v = (t.view(1, T, -1, 64) for t in attn.project(layer.norm1(x)))
            q, k = apply_rope(attn.q_norm(q).transpose(1, 2), attn.k_norm(k).transpose(1, 2),
                              m.rope_cos[at : at + T], m.rope_sin[at : at + T])
            ks.append(k.transpose(1, 2)[0].cpu()), vs.append(v[0].cpu())
            y = attend(q.transpose(1, 2)[0].cpu(), held(torch.cat(ks), at + T), held(torch.cat(vs), at + T), at)[0]
            x = x + attn.o(y.bfloat16().to(DEV).reshape(1, T, -1))
            x = x + layer.ffn(layer.norm2(x))
        out.append(torch.nn.functional.linear(m.final_norm(x), m.embed.weight))
        at += T
    return torch.cat(out, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(1, 64), (6, 64), (6, 128), (80, 64), (80, 128)])
@pytest.mark.parametrize("gap", [12.0, 18.0, 21.0])
def test_one_key_far_above_the_rest(T, D, gap):
    """A first token of small values whose score is `gap` above every other one's: the others'
    probabilities, e^-gap of the largest, still make up the output. Each p is off by
    2^-12 of itself (fp16) down to 2^-24 of the row's largest, and by 2^-35 of that below.
    256 heads, so that no range of keys is so short that the sink is in another one."""
    B, Hk, G, P = 32, 8, 4, 12000
    u = torch.ones(D) * D**-0.5
    k = 0.05 * tokens(1, 1, P, 1, D, 0.0).float()
    k -= (k @ u)[..., None] * u              # scores of about zero ...
    k[0, 0, 0] = 4 * u                       # ... but for the first
    v = 1 + 0.5 * tokens(2, 1, P, 1, D, 0.0).float()
    v[0, 0] *= 1e-3
    k, v = k.bfloat16(), v.bfloat16()
    q = (u * gap * D**0.5 / 4).bfloat16().expand(1, T, G, D)
    c = new(P, Hk, D, B)
    kd, vd = (t.to(DEV).expand(B, P, Hk, D) for t in (k, v))
    c.write(0, kd[:, : P - T], vd[:, : P - T], 0)
    y = fk.attention_kv8(q.to(DEV).repeat(B, 1, Hk, 1), kd[:, P - T :], vd[:, P - T :], c, 0, P - T).cpu()
    assert torch.equal(y, y[:1, :, :1].expand_as(y))
    ek, ev = held(k[0], P), held(v[0], P)
    e, pv, size, vmax, top = attend(q[0, :, :1], ek, ev, P - T)
    tol = e.abs() * 2.0**-8 + pv * (2.0**-11 + size * 2.0**-19) + P * 2.0**-35 * vmax * top
    err = (y[0, :, :1].double() - e).abs()
    assert (err <= tol).all(), (err / tol).max()


def check_sizes(y, q, k, v, first):
    """check's bound without its absolute term: outputs down to the subnormal numbers, of
    which the smallest bf16 is 2^-133, and fp32 sums of them off by a few of 2^-149."""
    e, pv, size, vmax, top = attend(q, k, v, first)
    tol = e.abs() * 2.0**-8 + pv * (2.0**-11 + size * 2.0**-19) + k.shape[0] * 2.0**-25 * vmax * top + 2.0**-134 + 2.0**-142
    err = (y.cpu().double() - e).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("P", [40, 64, 100, 190])
@pytest.mark.parametrize("size", [1e30, 1e8, 1e-12, 1e-30, 2.0**-126, 2.0**-130, 0.0])
def test_a_cache_of_values_of_one_size(size, P, T):
    """Whole blocks and unfinished ones of values far from 1, at few and at many rows."""
    D = 128
    k, q = tokens(1, 1, P, 1, D), tokens(7, 1, T, 2, D)
    v = (tokens(2, 1, P, 1, D).double() * size).bfloat16()
    c = new(256, 1, D)
    if P > T:
        c.write(0, k[:, : P - T].to(DEV), v[:, : P - T].to(DEV), 0)
    y = fk.attention_kv8(q.to(DEV), k[:, P - T :].to(DEV), v[:, P - T :].to(DEV), c, 0, P - T)
    check_sizes(y[0], q[0], held(k[0], P), held(v[0], P), P - T)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("size", [2.0**14, 2.0**24, 2.0**60])
def test_a_large_channel_of_the_unfinished_block(size, T):
    """The unfinished block is held in bf16: a value channel far larger than the others takes
    nothing from them (as it would in a packed block)."""
    P, D = 60, 128
    k, q = tokens(1, 1, P, 1, D), tokens(7, 1, T, 2, D)
    v = tokens(2, 1, P, 1, D)
    v[..., 5] *= size
    c = new(128, 1, D)
    c.write(0, k[:, : P - T].to(DEV), v[:, : P - T].to(DEV), 0)
    y = fk.attention_kv8(q.to(DEV), k[:, P - T :].to(DEV), v[:, P - T :].to(DEV), c, 0, P - T)
    check_sizes(y[0], q[0], k[0].float(), v[0].float(), P - T)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
def test_infinities_of_the_unfinished_block(T):
    """They are NaN from the call that writes them on, not from the one that packs their
    block: a key's rows are NaN and do not lose that key, a value's column is."""
    P, H, D = 64, 2, 64
    k, v, q = tokens(1, 1, P, H, D), tokens(2, 1, P, H, D), tokens(3, 1, P, 4, D)
    k[0, 2, 0, 3], v[0, 4, 1, 7], v[0, 5, 1, 9] = -math.inf, math.inf, math.nan
    q[0, :, :2, 3] = 1.0  # the bad key's score would be -inf
    c = new(P, H, D)
    n = 20 + T
    for at in (0, 20):
        m = 20 if at == 0 else T
        y = fk.attention_kv8(q[:, at : at + m].to(DEV), k[:, at : at + m].to(DEV), v[:, at : at + m].to(DEV), c, 0, at)
    def spoilt(y):
        assert y[0, :, :2].isnan().all()
        assert y[0, :, 2:, [7, 9]].isnan().all() and y[0, :, 2:].isnan().sum() == y.shape[1] * 4
    spoilt(y.cpu())
    rk, rv = (t[0].cpu() for t in c.read(0, 0, n))
    assert rk[2, 0, 3].isnan() and rk.isnan().sum() == 1
    assert rv[4, 1, 7].isnan() and rv[5, 1, 9].isnan() and rv.isnan().sum() == 2
    y = fk.attention_kv8(q[:, n:].to(DEV), k[:, n:].to(DEV), v[:, n:].to(DEV), c, 0, n)  # packs the block
    spoilt(y.cpu())
    rk, rv = (t[0].cpu() for t in c.read(0, 0, P))
    assert rk[2, 0, 3].isnan() and rk.isnan().sum() == 1 and rv.isnan().sum() == 2


@pytest.mark.gpu
def test_rope_rows_that_share_memory():
    """cos and sin of tokens at one position, as an expanded row."""
    h, m = model()
    attn = m.layers[0].attn
    x = tokens(1, 1, 3, 1, 192).view(1, 3, 192).to(DEV)
    a, b = (m.alloc_cache(64, kv8=True) for _ in range(2))
    cos, sin = (t[5:6].expand(3, -1) for t in (m.rope_cos, m.rope_sin))
    with torch.inference_mode():
        y = attn(x, kv_cache=a, layer_idx=0, cos=cos, sin=sin, start_pos=0)
        z = attn(x, kv_cache=b, layer_idx=0, cos=cos.contiguous(), sin=sin.contiguous(), start_pos=0)
    assert torch.equal(y, z)


@pytest.mark.gpu
@pytest.mark.parametrize("pos,T,D", [(0, 63, 64), (64, 63, 128), (100, 27, 128), (63, 1, 64), (126, 1, 128), (127, 1, 64),
                                     (1000, 23, 64), (1, 62, 128)])
def test_calls_that_end_no_block_before_their_last_token_are_causal(pos, T, D):
    """Tokens after a row leave it bit for bit as it was."""
    P, Hk = pos + T, 2
    k, v, q = tokens(1, 1, P, Hk, D), tokens(2, 1, P, Hk, D), tokens(3, 1, T, 4, D)
    outs = []
    for t in sorted({0, T // 2, T - 1}):
        k2, v2 = k.clone(), v.clone()
        k2[:, pos + t + 1 :] *= 30
        v2[:, pos + t + 1 :] *= -30
        c = new(P, Hk, D)
        if pos:
            c.write(0, k[:, :pos].to(DEV), v[:, :pos].to(DEV), 0)
        y = fk.attention_kv8(q.to(DEV), k2[:, pos:].to(DEV), v2[:, pos:].to(DEV), c, 0, pos)
        outs.append((t, y))
    for t, y in outs:
        assert torch.equal(y[:, : t + 1], outs[-1][1][:, : t + 1]), t


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 63, 64, 65, 128, 200])
def test_causal_scores(n):
    """A text's scores up to a token do not depend on what follows it, and are a decode loop's
    but for the row counts of the projections (two layers' roundings, as in test_model_over_the_cache)."""
    h, m = model(fuse_norm=True, linear_down_o=True)
    g = torch.Generator().manual_seed(2)
    a = torch.randint(0, 32, (n,), generator=g).tolist()
    at = n // 2
    b = a[: at + 1] + [(t + 7) % 32 for t in a[at + 1 :]]
    x, y = (h.teacher_forced_logprobs(m, t, DEV, top_k=3, kv8=True, causal=True) for t in (a, b))
    for s, t in zip(x, y):
        assert s.shape[0] == n - 1 and torch.equal(s[:at], t[:at])
    with torch.inference_mode():
        cache, ids = m.alloc_cache(256, kv8=True), torch.tensor([a], device=DEV)
        step = torch.cat([m(i, cache) for i in ids.split(1, 1)], 1)[0, :-1].float()
        one = torch.cat([m(i, c) for c in [m.alloc_cache(256, kv8=True)]
                         for i in ids.split([63, 1] * (n // 64) + [n % 64] * (n % 64 > 0), 1)], 1)[0, :-1]
    assert (one.float() - step).norm() <= 2e-2 * step.norm()
    direct = fk.token_logprobs(one, ids[0, 1:], 3)
    assert all(torch.equal(s, t) for s, t in zip(x, direct))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_scores_of_the_shortest_texts(causal):
    h, m = model()
    for n in (0, 1):
        s = h.teacher_forced_logprobs(m, list(range(n)), DEV, top_k=2, kv8=True, causal=causal)
        assert s.logprob.shape == (0,) and s.top_ids.shape == (0, 2)
