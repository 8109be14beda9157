"""Log-probabilities of tokens, entropy and top alternatives against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from llms_amd import _lib
from llms_amd import kernels as fk

DEV = "cuda"


def reference(logits, tokens, k):
    """The definition in 64 bits on the CPU; top k by value, ties to the lowest token."""
    x = logits.detach().cpu().double()
    V = x.shape[-1]
    lp = x.log_softmax(-1)
    t = tokens.cpu()
    at = lp.gather(-1, t.clamp(0, V - 1)[..., None])[..., 0]
    at = torch.where(t < 0, torch.zeros_like(at), torch.where(t >= V, torch.full_like(at, math.nan), at))
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    h = torch.where(lp.isnan().any(-1), torch.full_like(h, math.nan), h)
    key = torch.where(x.isnan(), math.inf, x)  # a NaN row is checked apart
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :k]
    return at, h, ids, lp.gather(-1, ids)


def check(logits, tokens, k, got=None):
    """Sums in 32 bits: a row's l has terms off by the rounding of z log2(e) (half a
    step of up to 1.45 spread), of exp2 (a step) and of at most 64 + 8 + 64 additions,
    so log l is off by at most 2^-24 (138 + 3 spread); x - m and the differences
    add steps of the spread. The entropy has that error in log l, and u / l, at most
    log V, off by twice the relative error."""
    got = got if got is not None else fk.token_logprobs(logits, tokens, k)
    at, h, ids, top = reference(logits, tokens, k)
    x = logits.detach().cpu().double()
    fin = torch.where(x.isfinite(), x, torch.nan)
    spread = (torch.nan_to_num(fin, nan=-1e300).amax(-1) - torch.nan_to_num(fin, nan=1e300).amin(-1)).clamp(min=0)
    tol = 2.0**-24 * (160 + 8 * spread)
    V = x.shape[-1]
    for name, g, e, t in (("logprob", got.logprob, at, tol), ("entropy", got.entropy, h, tol * (2 + 2 * math.log(V))),
                          ("top", got.top_logprobs, top, tol[..., None])):
        assert g.dtype == torch.float32 and g.shape == e.shape, name
        g = g.cpu().double()
        same = (g == e) | (g.isnan() & e.isnan())
        assert (same | ((g - e).abs() <= t)).all(), (name, (g - e).abs().max())
    assert got.top_ids.dtype == torch.int64
    assert torch.equal(got.top_ids.cpu(), ids)


def make(M, V, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, V, generator=g) * scale).to(dtype)
    return x.to(DEV), torch.randint(0, V, (M,), generator=g).to(DEV)


# ------------------------------------------------------------- refusals (CPU)


def test_refusals_on_the_cpu():
    x, t = torch.zeros(3, 50, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.long)
    with pytest.raises(ValueError, match="HIP"):
        fk.token_logprobs(x, t)
    with pytest.raises(ValueError, match="without its last dim"):
        fk.token_logprobs(x, t[:2])
    with pytest.raises(TypeError, match="float32"):
        fk.token_logprobs(x.double(), t)
    with pytest.raises(TypeError, match="int64"):
        fk.token_logprobs(x, t.int())
    for k in (-1, 51, 65):
        with pytest.raises(ValueError, match="top_k"):
            fk.token_logprobs(x, t, k)
    with pytest.raises(ValueError, match="top_k"):
        fk.token_logprobs(torch.zeros(3, 100), t, 65)
    with pytest.raises(ValueError, match="1 to"):
        fk.token_logprobs(torch.zeros(3, 0), t)
    with pytest.raises(ValueError, match="1 to"):
        fk.token_logprobs(torch.zeros(1, (1 << 20) + 1), t[:1])


def test_c_entry_refusals():
    lib = _lib.capi()
    P = 4096  # never dereferenced: every call below is refused before a launch
    ok = dict(x=P, dt=0, ld=100, t=P, lp=P, h=P, ids=P, top=P, M=4, V=100, k=5, ws=P, nb=1 << 20)

    def call(**kw):
        a = dict(ok, **kw)
        return lib.fp_token_logprobs(a["x"], a["dt"], a["ld"], a["t"], a["lp"], a["h"], a["ids"], a["top"],
                                     a["M"], a["V"], a["k"], a["ws"], a["nb"], None)

    NULL, SHAPE, STRIDE, WORKSPACE = 1, 2, 3, 6
    for kw in (dict(dt=3), dict(dt=-1), dict(M=-1), dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21), dict(k=-1),
               dict(k=65), dict(k=101), dict(M=1 << 25)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(ld=99), dict(x=P + 1), dict(dt=2, x=P + 2), dict(t=P + 4), dict(lp=P + 2)):
        assert call(**kw) == STRIDE, kw
    for kw in (dict(x=None), dict(t=None), dict(lp=None), dict(h=None), dict(ids=None), dict(top=None)):
        assert call(**kw) == NULL, kw
    need = lib.fp_logprob_workspace_bytes(4, 100000, 5)
    assert need > 0
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=P + 8)):
        assert call(V=100000, ld=100000, **dict(dict(nb=need), **kw)) == WORKSPACE, kw
    assert call(M=0) == 0
    assert lib.fp_logprob_workspace_bytes(4, 100, 5) == 0  # one piece per row
    assert lib.fp_logprob_workspace_bytes(4, 100, 101) == 0


# ------------------------------------------------------------------- numerics


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (2, 7, 0), (3, 50, 50), (5, 64, 64), (1, 348, 20), (2, 4096, 3),
                                   (3, 4097, 20), (4, 16384, 5), (2, 32003, 8), (600, 16391, 6), (1, 151936, 20),
                                   (530, 2001, 33), (1, 262145, 64), (1, 1 << 20, 64)])
def test_against_64_bits(M, V, k, dtype):
    x, t = make(M, V, dtype, seed=M + V)
    check(x, t, k)


@pytest.mark.gpu
def test_large_offsets():
    """Element offsets beyond 2^31 (rows of 4.5 GB together)."""
    M, V = 15000, 151936
    x = torch.zeros(M, V, dtype=torch.bfloat16, device=DEV)
    rows = [0, 7065, 14134, 14999]
    some, t = make(len(rows), V, torch.bfloat16, seed=1)
    x[rows] = some
    tokens = torch.zeros(M, dtype=torch.long, device=DEV)
    tokens[rows] = t
    got = fk.token_logprobs(x, tokens, 5)
    check(some, t, 5, fk.TokenLogprobs(*(o[rows] for o in got)))
    assert torch.allclose(got.entropy[1:7000].cpu(), torch.tensor(math.log(V)), rtol=1e-5)
    assert (got.top_ids[1:7000].cpu() == torch.arange(5)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 3000, 16384, 151936])
def test_ties_and_equal_rows(V):
    g = torch.Generator().manual_seed(V)
    x = torch.zeros(4, V)
    x[1] = torch.randint(0, 3, (V,), generator=g).float()          # a third of the row ties at the top
    x[2, :] = torch.arange(V).float() % 5 * -0.0                   # zeros of both signs
    x[3] = torch.linspace(0, 20, V)                                # the best in one place
    t = torch.tensor([0, V - 1, V // 2, 1])
    for dtype in (torch.bfloat16, torch.float32):
        check(x.to(dtype).to(DEV), t.to(DEV), 20)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [60, 5000, 151936])
def test_masked_infinite_and_nan_logits(V):
    x, _ = make(8, V, torch.bfloat16, seed=3)
    t = torch.arange(8, device=DEV)
    x[0, 11:] = -math.inf                # most tokens forbidden: fewer left than top_k
    x[1, 1:] = -math.inf                 # one left
    x[2] = -math.inf                     # none left
    x[3, 5] = math.inf
    x[4, 50] = math.nan
    x[5, : V // 2] = -math.inf
    x[6] = -math.inf
    x[6, V - 1] = -3.0
    got = fk.token_logprobs(x, t, 20)
    keep = [0, 1, 5, 6, 7]
    check(x[keep], t[keep], 20, fk.TokenLogprobs(*(o[keep] for o in got)))
    for r in (2, 3, 4):
        assert got.logprob[r].isnan() and got.entropy[r].isnan(), r
    assert got.top_ids[2].tolist() == list(range(20))
    assert got.top_ids[3, 0] == 5
    assert got.top_ids[4, 0] == 50 and got.top_logprobs[4].isnan().all()
    assert got.entropy[1] == 0 and got.logprob[1] == -math.inf


@pytest.mark.gpu
def test_tokens_that_are_none():
    x, _ = make(4, 700, torch.bfloat16)
    t = torch.tensor([-1, -100, 700, 1 << 40], device=DEV)
    got = fk.token_logprobs(x, t)
    assert got.logprob[:2].tolist() == [0.0, 0.0] and got.logprob[2:].isnan().all()
    assert got.top_ids.shape == (4, 0)


@pytest.mark.gpu
def test_strides_and_shapes():
    x, _ = make(12, 3003, torch.bfloat16, seed=5)
    t = torch.randint(0, 3000, (3, 4), device=DEV)
    check(x.view(3, 4, 3003), t, 4)
    check(x.view(3, 4, 3003)[:, 1:, 1:3001], t[:, 1:], 4)         # odd row starts, rows that do not collapse
    check(x[:, ::2], t.view(-1) // 2, 4)                          # strided last dim
    check(x[:1].expand(5, 3003), t.view(-1)[:5], 4)               # rows that share memory
    check(x.t()[:12, :3].t().contiguous().t().t(), t.view(-1)[:3] % 12, 2)
    check(x[0], t[0, 0], 3)                                       # one row without a leading dim
    got = fk.token_logprobs(x[:0], t.view(-1)[:0], 2)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 2)


@pytest.mark.gpu
def test_stream_graph_and_inputs_left():
    x, t = make(9, 20011, torch.bfloat16, seed=6)
    before = x.clone()
    eager = fk.token_logprobs(x, t, 7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = fk.token_logprobs(x, t, 7)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fk.token_logprobs(x, t, 7)
    for seed in (6, 7, 8, 9):
        y, u = make(9, 20011, torch.bfloat16, seed=seed)
        x.copy_(y), t.copy_(u)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, fk.token_logprobs(y, u, 7)):
            assert torch.equal(a, b)
    x.copy_(before)
    assert torch.equal(x, before)


@pytest.mark.gpu
def test_gradients_and_transforms_are_refused():
    x, t = make(2, 100, torch.float32)
    with pytest.raises(RuntimeError, match="gradients"):
        fk.token_logprobs(x.requires_grad_(), t)
    with torch.no_grad():
        fk.token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="gradients"):
        torch.func.vmap(lambda a, b: fk.token_logprobs(a, b).logprob)(x.detach()[None], t[None])


@pytest.mark.gpu
def test_scoring_a_text_with_a_model():
    from llms_amd import harness as h

    m = h.tiny_model(h.Cfg(vocab_size=300), seed=2, device=DEV)
    tokens = [5, 9, 250, 7, 7, 31, 299, 0]
    got = h.teacher_forced_logprobs(m, tokens, DEV, top_k=4)
    logits = h.teacher_forced_logits(m, tokens, DEV)[:-1]
    check(logits, torch.tensor(tokens[1:], device=DEV), 4, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [60, 5000, 151936])
@pytest.mark.parametrize("mask", [-1e5, -1e9, -1e10, -1e20, -1e30, "lowest"])
def test_finite_masks(mask, V, dtype):
    """Forbidden tokens at a large finite value instead of -inf: whole pieces of a row, all
    but one token, the whole row, all but a token as far above zero. What is not masked
    spreads over less than 32 (check's tolerance there); a masked token's distance is a
    difference of fp32 values, and a second one with log l (2^-23 of it)."""
    low = torch.finfo(dtype).min if mask == "lowest" else mask
    x, _ = make(5, V, torch.float32, seed=9)
    x[0, : V // 2] = low
    x[1] = low
    x[1, V - 1] = 1.0
    x[2] = low
    x[3] = low
    x[3, 0] = -low
    x[4, V // 3 :] = low
    x, t = x.to(dtype), torch.tensor([V - 1, V - 1, 3, 0, 0], device=DEV)
    got = fk.token_logprobs(x, t, 5)
    at, h, ids, top = reference(x, t, 5)
    tol = 2.0**-24 * (160 + 8 * 32)
    assert ((got.logprob.cpu().double() - at).abs() <= tol).all()
    assert ((got.entropy.cpu().double() - h).abs() <= tol * (2 + 2 * math.log(V))).all()
    top = top.float().double()  # (twice the largest number is -inf in 32 bits)
    g = got.top_logprobs.cpu().double()
    assert ((g == top) | ((g - top).abs() <= tol + top.abs() * 2.0**-23)).all()
    assert torch.equal(got.top_ids.cpu(), ids)
