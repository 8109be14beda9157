"""Caches of two parts at the ends of their range: scores that are far apart, precision by
the size of a call, positions at a window's and at a table's end."""

from __future__ import annotations

import ctypes

import pytest
import torch

from llms_amd import _lib, harness
from llms_amd import kernels as fk
from tests.test_seg import SegArgs, check, exact, new_shared, new_window, randn

DEV = "cuda"
gpu = pytest.mark.gpu


# ------------------------------------------------------------- scores far apart


def along(n, D, spikes):
    """Keys [n, 1, D]: 0 but for a first channel at some positions. With q = 32 there (heads of 128) a
    channel of x is a score of 4.0806 x in powers of two."""
    k = torch.zeros(n, 1, D, dtype=torch.bfloat16)
    for p, x in spikes.items():
        k[p, 0, 0] = x
    return k


def check_apart(y, e):
    """One rounding to bf16 (2^-8), p in two bf16 parts in products and in their sum (2 x 2^-16 of the weighted |v|),
    and scores of up to 2^7 powers of two: the factor log2(e) / sqrt(D) is three roundings off (2^-24 each) and the
    exponent one, so an exponential is off by 2^7 x 4 x 2^-24 x ln 2 < 2^-15, in the products and in their sum."""
    want, size, _ = e
    err = (y.to(DEV).double() - want).abs()
    tol = want.abs() * 2.0**-8 + size * (2 * 2.0**-16 + 2 * 2.0**-15) + 1e-30
    assert y.isfinite().all() and (err <= tol).all(), float((err / tol).max())


def window_apart(n, T, spikes):
    """The last T of n tokens of one head attend over all of them."""
    g = torch.Generator().manual_seed(n + T)
    c, _ = new_window(n, 0, 1, 128, 1, max_step=n)
    k, v = along(n, 128, spikes), randn(g, n, 1, 128)
    for p in spikes:
        v[p] = v[p].sign() / 2
    q = torch.zeros(T, 1, 128).bfloat16()
    q[:, :, 0] = 32
    c.write(0, k[None].to(DEV), v[None].to(DEV), 0)
    y = fk.attention_window(q[None].to(DEV), k[None, n - T :].to(DEV), v[None, n - T :].to(DEV), c, 0, n - T)
    at = torch.arange(n)
    check_apart(y[0], exact(q, k, v, at[n - T :], at))


@gpu
@pytest.mark.parametrize("late", [30.75, 31.0, 31.125, 31.25, 31.5, 40.0, 61.0, 62.25, 62.5, 80.0])
@pytest.mark.parametrize("early", [0.5, 15.0, 30.75, 31.25])
def test_a_score_far_above_those_before(early, late):
    """Of 200 keys one at position 100 counts beside a later one in the tile that the last rows see in part: sums of
    up to 2^127 meet a reference that rises by as much, or by more than an exponential can say."""
    window_apart(200, 200, {100: early, 195: late})


@gpu
@pytest.mark.parametrize("n,spikes", [
    (1065, {130: 30.75, 260: 31.125}),  # the first range's largest comes late, the second's early
    (1065, {130: 31.0, 260: 31.25, 700: 30.875}),
    (1065, {130: 31.25, 386: 31.25, 642: 31.25, 898: 31.25}),  # each range's sum is near the largest number
    (1065, {130: 31.25, 140: 45.0, 386: 31.25, 642: 45.0}),
    (16449, {320 * i + 130: 30.25 for i in range(51)}),  # and together they are past it
])
def test_scores_apart_in_ranges(n, spikes):
    """The same where a row's keys are cut into ranges."""
    window_apart(n, 65, spikes)


@gpu
@pytest.mark.parametrize("spikes", [{130: 30.75, 270: 31.125}, {256 * i + 130: 31.25 for i in range(8)}])
@pytest.mark.parametrize("B", [20, 40])
def test_scores_apart_in_a_shared_text(B, spikes):
    """And of rows of all sequences over one text."""
    g = torch.Generator().manual_seed(B)
    P, Hq = 2048, 8
    k, v, own = along(P, 128, spikes), randn(g, P, 1, 128), randn(g, B, 1, 1, 128)
    for p in spikes:
        v[p] = v[p].sign() / 2
    c = fk.KVCacheShared([k.transpose(0, 1).to(DEV)], [v.transpose(0, 1).to(DEV)], max_batch=B, max_new=4)
    q = torch.zeros(B, 1, Hq, 128).bfloat16()
    q[..., 0] = 32
    y = fk.attention_shared(q.to(DEV), torch.zeros_like(own).to(DEV), own.to(DEV), c, 0, P)
    for b in range(B):
        e = exact(q[b], torch.cat([k, torch.zeros_like(own[b])]), torch.cat([v, own[b]]), torch.tensor([P]),
                  torch.arange(P + 1))
        check_apart(y[b], e)


@gpu
@pytest.mark.parametrize("n,T", [(200, 5), (200, 100), (1065, 65)])
@pytest.mark.parametrize("x", [float("-inf"), torch.finfo(torch.bfloat16).min])
def test_first_keys_of_no_weight(n, T, x):
    """A whole tile whose scores are all the negative infinity comes before the others."""
    g = torch.Generator().manual_seed(n)
    c, _ = new_window(n, 0, 1, 128, 1, max_step=n)
    q, k, v = randn(g, T, 1, 128), randn(g, n, 1, 128), randn(g, n, 1, 128)
    k[:70, :, 0] = x
    q[:, :, 0] = q[:, :, 0].abs() + 32
    c.write(0, k[None].to(DEV), v[None].to(DEV), 0)
    y = fk.attention_window(q[None].to(DEV), k[None, n - T :].to(DEV), v[None, n - T :].to(DEV), c, 0, n - T)
    at = torch.arange(n)
    check_apart(y[0], exact(q, k, v, at[n - T :], at))


# ------------------------------------------------------------- precision


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(16, 8, 128), (8, 2, 64), (7, 1, 128)])
@pytest.mark.parametrize("B,T", [(1, 200), (2, 90), (1, 1000)])
def test_prompts_take_p_in_two_parts(Hq, Hk, D, B, T):
    g = torch.Generator().manual_seed(T + Hq)
    c, _ = new_window(400, 3, Hk, D, B, max_step=1000)
    s, text = new_shared(g, Hk, 333, D, B, T)
    q, k, v = randn(g, B, T, Hq, D, scale=1.5), randn(g, B, T, Hk, D), randn(g, B, T, Hk, D)
    on = [t.to(DEV) for t in (q, k, v)]
    y, z = fk.attention_window(*on, c, 0, 0), fk.attention_shared(*on, s, 0, 333)
    at = torch.arange(T)
    for b in range(B):
        check(y[b], exact(q[b], k[b], v[b], at, at, 400, 3), 2)
        kv = [torch.cat([text[b][n], t[b]]) for n, t in (("k", k), ("v", v))]
        check(z[b], exact(q[b], *kv, 333 + at, torch.arange(333 + T)), 2)


@gpu
@pytest.mark.parametrize("Hq,Hk,D", [(32, 8, 128), (8, 2, 64)])
@pytest.mark.parametrize("B", [2, 17, 33, 64])
def test_precision_of_a_sequence_does_not_depend_on_the_batch(Hq, Hk, D, B):
    g = torch.Generator().manual_seed(B)
    P, T = 700, 3
    s, text = new_shared(g, Hk, P, D, B, 8)
    q, k, v = randn(g, B, T, Hq, D, scale=1.5), randn(g, B, T, Hk, D), randn(g, B, T, Hk, D)
    y = fk.attention_shared(q.to(DEV), k.to(DEV), v.to(DEV), s, 0, P)
    at = torch.arange(T)
    for b in (0, 1, B - 1):
        kv = [torch.cat([text[b][n], t[b]]) for n, t in (("k", k), ("v", v))]
        check(y[b], exact(q[b], *kv, P + at, torch.arange(P + T)), 2)


@gpu
@pytest.mark.parametrize("Hq,Hk,D,B,T", [(32, 8, 128, 128, 9), (16, 8, 64, 70, 30), (12, 4, 128, 150, 16), (32, 8, 128, 64, 5)])
def test_few_rows_of_many_sequences(Hq, Hk, D, B, T):
    """More than 512 row tiles, each of 20 to 64 rows."""
    g = torch.Generator().manual_seed(B)
    c, _ = new_window(300, 4, Hk, D, B)
    q, k, v = randn(g, B, T, Hq, D, scale=1.5), randn(g, B, 400 + T, Hk, D), randn(g, B, 400 + T, Hk, D)
    c.write(0, k[:, :400].to(DEV), v[:, :400].to(DEV), 0)
    y = fk.attention_window(q.to(DEV), k[:, 400:].to(DEV), v[:, 400:].to(DEV), c, 0, 400)
    for b in (0, 1, B // 2, B - 1):
        check(y[b], exact(q[b], k[b], v[b], 400 + torch.arange(T), torch.arange(400 + T), 300, 4), 2)


# ------------------------------------------------------------- keys that are not finite


@gpu
@pytest.mark.parametrize("T", [1, 5, 100])
@pytest.mark.parametrize("x", [float("inf"), float("-inf"), float("nan")])
def test_keys_that_are_not_finite(T, x):
    """A row that sees one is NaN where its score is NaN or the positive infinity; a score of the negative one has no
    weight."""
    g = torch.Generator().manual_seed(T)
    n, Hq, Hk, D = 200, 4, 2, 64
    for dim in (1, D):
        c, _ = new_window(300, 2, Hk, D, 1, max_step=n)
        q, k, v = randn(g, T, Hq, D, scale=1.5), randn(g, n, Hk, D), randn(g, n, Hk, D)
        k[120, 0, :dim] = x
        k[n - 1, 1, :dim] = x  # seen by the last row alone
        c.write(0, k[None].to(DEV), v[None].to(DEV), 0)
        y = fk.attention_window(q[None].to(DEV), k[None, n - T :].to(DEV), v[None, n - T :].to(DEV), c, 0, n - T)
        at = torch.arange(n)
        want, size, _ = exact(q, k, v, at[n - T :], at, 300, 2)
        bad = want.isnan()
        assert torch.equal(y[0].isnan(), bad)
        err = (y[0].double() - want).abs()
        assert (err <= want.abs() * 2.0**-8 + size * (2 * 2.0**-16 * (1 + 2.0**-8) + 2.0**-17))[~bad].all()


# ------------------------------------------------------------- positions


@gpu
@pytest.mark.parametrize("window,max_step", [(65, 64), (1, 64), (1, 128), (129, 128)])
@pytest.mark.parametrize("again", [1, 5, 64])
def test_the_furthest_step_back(window, max_step, again):
    """max_step tokens taken back from a ring that has not a slot to spare, and written anew in steps of any size."""
    g = torch.Generator().manual_seed(window)
    Hq, Hk, D, n = 4, 2, 64, 500
    c, _ = new_window(window, 2, Hk, D, 1, max_step=max_step)
    assert c.ring == window + max_step - 1
    k, v = randn(g, n, Hk, D), randn(g, n, Hk, D)
    c.write(0, k[None].to(DEV), v[None].to(DEV), 0)
    at = torch.arange(n)
    for start in range(n - max_step, n, again):
        T = min(again, n - start)
        q, k[start : start + T], v[start : start + T] = randn(g, T, Hq, D), randn(g, T, Hk, D), randn(g, T, Hk, D)
        end = start + T
        y = fk.attention_window(q[None].to(DEV), *(t[None, start:end].to(DEV) for t in (k, v)), c, 0, start)
        check(y[0], exact(q, k[:end], v[:end], at[start:end], at[:end], window, 2), 2)


def model_of(**kw):
    c = harness.Cfg(vocab_size=211, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                    intermediate_size=512, max_position_embeddings=700)
    m = harness.tiny_model(c, state=harness.tiny_state(c, embed_scale=0.3), device=DEV)
    return fk.apply_triton_kernels(m, **kw)


@gpu
@pytest.mark.parametrize("kv8", [False, True])
def test_a_position_in_one_element(kv8):
    """One sequence's position as [1] is the one for all, over every cache."""
    f = model_of()
    ids = torch.randint(0, 211, (1, 40), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.inference_mode():
        ys = []
        for shape in ((), (1,)):
            c = f.alloc_cache(64, kv8=kv8)
            f(ids[:, :30], c)
            at = torch.full(shape, 30, device=DEV)
            ys.append((f(ids[:, 30:31], c, start_pos=at), f(ids[:, 31:], c, start_pos=at + 1)))
        for a, b in zip(*ys):
            assert a.shape == b.shape and (a.float() - b.float()).abs().max() <= 0.02 * a.float().std()


def small(device="cpu", **kw):
    c = harness.Cfg(vocab_size=40, hidden_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
                    head_dim=64, intermediate_size=64, **{"max_position_embeddings": 20, **kw})
    return harness.tiny_model(c, device=device)


def test_positions_past_the_rope_table():
    """Host positions are refused; device ones read no row that is not there (here the eager attention's refusal of the
    cache, not an index out of range, ends the call)."""
    m = small()
    ids = torch.zeros(1, 3, dtype=torch.long)
    with torch.inference_mode():
        assert m(ids, m.alloc_cache(30), start_pos=17).shape == (1, 3, 40)
        for at in (18, 19, 20, 1000, -1):
            with pytest.raises(ValueError, match="RoPE table of 20"):
                m(ids, m.alloc_cache(30), start_pos=at)
        cache = m.alloc_cache(30, window=4)
        for at in ([18], [-1], [1 << 40]):
            with pytest.raises(TypeError, match="apply_triton_kernels"):
                m(ids, cache, start_pos=torch.tensor(at))
        # within the table a device position is the host's
        a, b = m.alloc_cache(20), m.alloc_cache(20)
        for c, at in ((a, 0), (b, torch.tensor(0))):
            m(ids, c, start_pos=at)
        for n in (1, 2):
            y, z = m(ids[:, :n], a, start_pos=3), m(ids[:, :n], b, start_pos=torch.tensor(3))
            assert (y - z).abs().max() <= 0.02 * y.float().std()


def test_rope_rows_of_another_length():
    """cos and sin must have a row for each token, whatever computes the rotation."""
    norm = small().layers[0].attn.q_norm
    c = fk.KVCacheWindow.alloc(1, 8, n_kv_heads=1, head_dim=64, device="cpu")
    q, k = torch.zeros(1, 3, 128).bfloat16(), torch.zeros(1, 3, 64).bfloat16()
    for n in (1, 2, 4):
        for t in (torch.ones(n, 64).bfloat16(), torch.ones(n, 64), torch.ones(1, n, 64)):
            with pytest.raises(ValueError, match=r"must be \(3, 64\)"), torch.inference_mode():
                fk.seg.attention_core_seg(q, k, k, q_norm=norm, k_norm=norm, num_heads=2, cache=c, layer=0, cos=t, sin=t,
                                          start_pos=0)


@gpu
def test_a_window_model_at_its_table_s_end():
    f = model_of()
    ids = torch.randint(0, 211, (1, 698), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.inference_mode():
        c = f.alloc_cache(900, window=100)
        f(ids, c)
        with pytest.raises(ValueError, match="RoPE table"):
            f(ids[:, :3], c)
        step = harness.StepGraph(f, c, T=2)
        with pytest.raises(ValueError, match="RoPE table"):
            step(ids[:, :2], 699)
        y = step(ids[:, :2], 698).clone()
        assert torch.equal(y, f(ids[:, :2], c))
        s = harness.StepGraph(f, c, T=1, per_sequence=True)
        s(ids[:, :1], torch.tensor([700], device=DEV))  # past the table: its last row
        s(ids[:, :1], torch.tensor([-3], device=DEV))
    with pytest.raises(ValueError, match="RoPE table"):
        harness.greedy_generate(f, ids[0].tolist(), 8, DEV, window=100)


@pytest.mark.parametrize("kw", [dict(), dict(sinks=0), dict(sinks=9, max_step=100)])
def test_a_model_s_window_has_all_of_the_operator_s_sizes(kw):
    c = small().alloc_cache(50, window=30, max_batch=2, **kw)
    assert (c.window, c.sinks, c.max_step) == (30, kw.get("sinks", 4), kw.get("max_step", 256))
    with pytest.raises(ValueError, match="KVCacheWindow"):
        small().alloc_cache(50, window=30, max_step=0)


@gpu
def test_generation_over_a_window_of_any_sizes():
    """Steps of another size are the same attention; sinks are not."""
    f = model_of()
    prompt = torch.randint(0, 211, (300,), generator=torch.Generator().manual_seed(7)).tolist()
    kw = dict(window=64, sinks=7)
    out = harness.greedy_generate(f, prompt, 20, DEV, **kw)
    assert out == harness.graph_greedy_generate(f, prompt, 20, DEV, **kw)
    with torch.inference_mode():
        ids = torch.tensor([prompt], device=DEV)
        a, b, c = (f(ids, f.alloc_cache(300, window=64, **k)).float() for k in (dict(sinks=7), dict(sinks=7, max_step=300),
                                                                               dict(sinks=0)))
        assert (a - b).abs().max() <= 0.05 * a.std() < (a - c).abs().max()


def test_a_shared_text_is_taken_from_a_plain_cache():
    m = small()
    text = fk.KVCacheShared.of(m.alloc_cache(30), 10, max_batch=2, max_new=20)
    for cache in (m.alloc_cache(30, window=16), text):
        with pytest.raises(TypeError, match="plain cache"):
            fk.KVCacheShared.of(cache, 5, max_batch=1, max_new=1)


def test_key_counts_beyond_any_cache():
    """The C entry plans for at most as many keys as a cache may hold (2^28), whatever it is told."""
    need = _lib.capi().fp_seg_workspace_bytes
    for B, T, Hq, Hk, shared in ((1, 1, 4, 2, 0), (3, 5, 4, 2, 1), (2, 100, 4, 4, 0)):
        most = need(B, T, Hq, Hk, 64, 100, 1 << 28, shared, 0)
        assert most > 0
        for keys in ((1 << 28) + 1, 1 << 40, 1 << 61, (1 << 63) - 300, (1 << 63) - 1):
            assert need(B, T, Hq, Hk, 64, 100, keys, shared, 0) == most, keys
        for fixed in ((1 << 28) + 1, 1 << 60, (1 << 63) - 1):
            assert need(B, T, Hq, Hk, 64, fixed, 100, shared, 0) == 0


def test_sizes_that_overflow_are_refused():
    """Before a launch (there is no GPU here: a launch would not be FP_ERR_SHAPE either)."""
    a = dict(q=64, k=64, v=64, q_s_b=256, q_s_t=256, k_s_b=128, k_s_t=128, v_s_b=128, v_s_t=128, own_k=64, own_v=64,
             own_s_b=2 * 128 * 64, own_s_h=128 * 64, own_s_p=64, y=64, y_s_b=256, B=3, T=1, n_heads=4, n_kv_heads=2,
             head_dim=64, n_fixed=0, own_len=128)
    fixed = dict(fix_k=64, fix_v=64, fix_s_h=6400, n_fixed=100, pos=100)
    for kw in (dict(ring=1, window=(1 << 63) - 1), dict(ring=1, window=(1 << 63) - 129, T=128), dict(own_s_p=1 << 60),
               dict(own_s_p=1 << 62), dict(fixed, fix_s_p=1 << 61), dict(fixed, fix_s_p=(1 << 63) - 8)):
        for call in (lambda p: _lib.capi().fp_seg_attention(p, 100, 64, 1 << 40, None),
                     lambda p: _lib.capi().fp_seg_write(p, None)):
            assert call(ctypes.byref(SegArgs(**(a | kw)))) == 2, kw


@gpu
@pytest.mark.parametrize("T", [200, 129, 64])
def test_a_call_in_steps_past_the_last_position_writes_nothing(T):
    g = torch.Generator().manual_seed(0)
    c, _ = new_window(50, 4, 2, 64, 1)
    q, k = randn(g, 1, T, 4, 64).to(DEV), randn(g, 1, T, 2, 64).to(DEV)
    start = (1 << 30) - T + 1
    for call in (lambda: fk.attention_window(q, k, k, c, 0, start), lambda: c.write(0, k, k, start)):
        with pytest.raises(ValueError, match="outside"):
            call()
    assert not c.k[0].any() and not c.v[0].any()
    fk.attention_window(q, k, k, c, 0, start - 1)
    assert c.k[0].any()
