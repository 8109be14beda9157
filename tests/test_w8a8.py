"""Projections in 8-bit integers against 64 bits, and the swapped model."""

from __future__ import annotations

import copy

import pytest
import torch

from llms_amd import _lib, harness
from llms_amd import kernels as fk

DEV = "cuda"


def pack(w):
    s = w.float().abs().amax(1) / 127
    return torch.where(s[:, None] > 0, w.float() / s[:, None], 0.0).round().clamp(-127, 127).to(torch.int8), s


def make(seed, M, K, N, n=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, seed % K] *= 10
    x = x.bfloat16()
    # tokens whose quotients hold ties of the rounding: 127 x / top with top = 254 2^j
    if K >= 4 and M > 1:
        top = x[1].float().abs().max().log2().ceil().exp2() * (254 / 256)
        x[1, 0], x[1, 1], x[1, 2] = top, top * (3 / 254), -top * (101 / 254)
    ws = [pack((torch.randn(N, K, generator=g) * 0.02).bfloat16()) for _ in range(n)]
    return x, ws


def on(x, ws):
    return x.to(DEV), [(q.to(DEV), s.to(DEV)) for q, s in ws]


def codes(x):
    """Whole numbers (in 64 bits) and scales of tokens: ties to even."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(x * 127 / top.clamp(min=1e-300)), 0.0), top / 127


def exact(x, qs):
    c, sx = codes(x)
    return (c @ qs[0].double().T) * sx * qs[1].double()


def check_linear(y, x, qs):
    """The sum is exact; then fp32 rounds it, the token's scale and two products (2^-24 of the value
    each), and bf16 once (2^-8 of the value at most)."""
    e = exact(x, qs)
    err = (y.cpu().double() - e).abs()
    tol = e.abs() * (2.0**-8 + 2.0**-21) + 1e-38
    assert (err <= tol).all(), (err / tol).max()


def check_gate_up(y, x, g, u):
    """g and u off by four roundings of 2^-24; silu by its slope's share of that (|g silu'| <=
    (1 + |g|) silu) and fewer than 12 + 2 |g| roundings more (the exponential's argument is
    rounded to 2^-24 of |g|); the product's, and bf16's once."""
    eg, eu = exact(x, g), exact(x, u)
    y0 = eg * torch.sigmoid(eg) * eu
    tol = y0.abs() * (2.0**-8 + 2.0**-24 * (24 + 8 * eg.abs())) + 1e-37 * (1 + eu.abs())
    err = (y.cpu().double() - y0).abs()
    assert (err <= tol).all(), (err / tol).max()


# ------------------------------------------------------------- refusals (CPU)


def test_refusals_on_the_cpu():
    x, ((q, s),) = make(0, 3, 256, 40)
    with pytest.raises(ValueError, match="HIP"):
        fk.fused_linear_w8a8(x, q, s)
    with pytest.raises(TypeError, match="x must be bfloat16"):
        fk.fused_linear_w8a8(x.float(), q, s)
    with pytest.raises(TypeError, match="q must be int8"):
        fk.fused_linear_w8a8(x, q.to(torch.uint8), s)
    with pytest.raises(TypeError, match="s must be float32"):
        fk.fused_linear_w8a8(x, q, s.double())
    with pytest.raises(ValueError, match="s shape"):
        fk.fused_linear_w8a8(x, q, s[:-1])
    with pytest.raises(ValueError, match="q shape"):
        fk.fused_linear_w8a8(x[:, :-1], q, s)
    with pytest.raises(ValueError, match="n_q"):
        fk.fused_qkv_w8a8(x, q, s, n_q=8, n_k=8)
    with pytest.raises(ValueError, match="qg shape"):
        fk.fused_gate_up_silu_w8a8(x, q, s, q[:-1], s)
    with pytest.raises(ValueError, match="norm weight"):
        fk.fused_rmsnorm_qkv_w8a8(x, torch.ones(255).bfloat16(), 1e-6, q, s, n_q=20, n_k=10)
    with pytest.raises(ValueError, match="eps"):
        fk.fused_rmsnorm_gate_up_silu_w8a8(x, torch.ones(256).bfloat16(), -1.0, q, s, q, s)
    with pytest.raises(RuntimeError, match="no gradients"):
        fk.fused_linear_w8a8(x.requires_grad_(), q, s)


def test_swap_refusals():
    m = harness.tiny_model(harness.Cfg())
    with pytest.raises(ValueError, match="a8"):
        fk.apply_triton_kernels(m, a8=True)
    with pytest.raises(ValueError, match="exclude"):
        fk.apply_triton_kernels(m, int8=True, int4=True, a8=True)


def test_c_arguments():
    lib = _lib.capi()
    P, OK, NULL, SHAPE, STRIDE, WS = 64, 0, 1, 2, 3, 6
    wb = lib.fp_w8a8_workspace_bytes

    def lin(x=P, ldx=64, g=None, eps=0.0, q=P, ldq=64, s=P, y=P, ldy=96, M=40, N=96, K=64, ws=P, n=1 << 30):
        return lib.fp_linear_w8a8(x, ldx, g, eps, q, ldq, s, y, ldy, M, N, K, ws, n, None)

    def gu(qu=P, ldqu=64, su=P, M=40, N=96, K=64, n=1 << 30):
        return lib.fp_gate_up_silu_w8a8(P, 64, None, 0.0, P, 64, P, qu, ldqu, su, P, 96, M, N, K, P, n, None)

    assert lin(M=0) == OK and gu(M=0) == OK
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(K=(1 << 17) + 1, ldx=1 << 18, ldq=1 << 18),
               dict(N=1 << 23, ldy=1 << 23), dict(M=1 << 24), dict(g=P, eps=-1.0), dict(g=P, eps=float("nan"))):
        assert lin(**kw) == SHAPE, kw
    for kw in (dict(ldx=63), dict(ldq=63), dict(ldy=95), dict(x=P + 1), dict(s=P + 2), dict(y=P + 1), dict(ldq=1 << 23)):
        assert lin(**kw) == STRIDE, kw
    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(y=None)):
        assert lin(**kw) == NULL, kw
    assert gu(qu=None) == NULL and gu(su=None) == NULL and gu(ldqu=63) == STRIDE
    need = wb(40, 96, 64, 0)
    assert need >= 40 * 128 and lin(n=need - 1) == WS and lin(ws=None) == WS and lin(ws=P + 8) == WS
    assert wb(0, 96, 64, 0) == 0 and wb(40, 0, 64, 0) == 0


# ------------------------------------------------------------- products

gpu = pytest.mark.gpu

SHAPES = [  # M, K, N
    (1, 1, 1), (1, 1, 3), (2, 7, 2), (1, 16, 1), (3, 100, 40), (1, 1024, 4096), (2, 2560, 300), (4, 4096, 96),
    (1, 2541, 970), (5, 2560, 1000), (5, 2541, 97), (8, 128, 64), (9, 129, 65), (16, 9728, 40), (16, 300, 2560),
    (17, 1000, 17), (33, 1024, 129), (64, 4096, 600), (65, 2541, 200), (100, 64, 1000), (128, 256, 256),
    (129, 512, 513), (300, 2541, 970), (300, 2560, 1024), (257, 12288, 96), (1000, 1024, 700), (520, 4096, 3000),
    (2100, 640, 2600), (7, 20000, 33), (40, 20001, 64), (3, 131072, 10), (2, 4360, 40), (1, 12296, 20), (4, 4104, 50), (6, 4264, 30),
]


@gpu
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_and_qkv(M, K, N):
    x, ws = make(M + K + N, M, K, N)
    xd, (w,) = on(x, ws)
    y = fk.fused_linear_w8a8(xd, *w)
    assert y.shape == (M, N)
    check_linear(y, x, ws[0])
    if N >= 3:
        n_k = N // 3
        q, k, v = fk.fused_qkv_w8a8(xd, *w, n_q=N - 2 * n_k, n_k=n_k)
        assert torch.equal(torch.cat([q, k, v], -1), y)


@gpu
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gate_up(M, K, N):
    x, ws = make(M + K + N, M, K, N, n=2)
    xd, (g, u) = on(x, ws)
    y = fk.fused_gate_up_silu_w8a8(xd, *g, *u)
    assert y.shape == (M, N)
    check_gate_up(y, x, *ws)


@gpu
@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 16, 17, 64, 130, 300])
@pytest.mark.parametrize("K,N", [(1024, 512), (2541, 130), (2560, 640)])
def test_rows_do_not_depend_on_the_call(M, K, N):
    """A token's outputs are the same bits in any call, by itself or among others."""
    x, ws = make(M, M, K, N, n=2)
    xd, (g, u) = on(x, ws)
    y, z = fk.fused_linear_w8a8(xd, *g), fk.fused_gate_up_silu_w8a8(xd, *g, *u)
    assert torch.equal(y, fk.fused_linear_w8a8(xd, *g)) and torch.equal(z, fk.fused_gate_up_silu_w8a8(xd, *g, *u))
    for m in {0, M // 2, M - 1}:
        assert torch.equal(fk.fused_linear_w8a8(xd[m : m + 1], *g)[0], y[m])
        assert torch.equal(fk.fused_gate_up_silu_w8a8(xd[m : m + 1], *g, *u)[0], z[m])


@gpu
@pytest.mark.parametrize("M", [1, 3, 4, 5, 12, 40, 200])
@pytest.mark.parametrize("K", [1024, 2541, 2560, 11000])
def test_norm(M, K):
    """The norm rounds as the framework's norm does, so the call on its result is the same."""
    x, ws = make(M + K, M, K, 96, n=2)
    xd, (g, u) = on(x, ws)
    gamma = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(K))).bfloat16().to(DEV)
    f = xd.double()
    t = (f * (f.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).to(torch.bfloat16)
    xn = (t.float() * gamma.float()).bfloat16()
    q, k, v = fk.fused_rmsnorm_qkv_w8a8(xd, gamma, 1e-6, *g, n_q=32, n_k=32)
    y, e = torch.cat([q, k, v], -1).double(), exact(xn.cpu(), ws[0]).to(DEV)
    z = fk.fused_rmsnorm_gate_up_silu_w8a8(xd, gamma, 1e-6, *g, *u).double()
    eg, eu = e, exact(xn.cpu(), ws[1]).to(DEV)
    # a norm's value next to a rounding of bf16 may fall to either side: a code off by one or two (the row's
    # largest: the scale by 2^-8 and the codes with it) in a few of K places
    size = (codes(xn.cpu())[1] * ws[0][1].double() * 127).to(DEV)
    assert ((y - e).abs() <= e.abs() * 2.0**-7 + size * (4 + 0.02 * K**0.5)).all()
    size_u = (codes(xn.cpu())[1] * ws[1][1].double() * 127).to(DEV)
    off = 1.1 * size * (4 + 0.02 * K**0.5) * eu.abs() + (eg.abs() + size) * size_u * (4 + 0.02 * K**0.5)
    assert ((z - eg * torch.sigmoid(eg) * eu).abs() <= (eg * eu).abs() * 2.0**-6 + off).all()
    if M <= 64:  # one norm for every row count
        one = fk.fused_rmsnorm_qkv_w8a8(xd[M - 1 :], gamma, 1e-6, *g, n_q=32, n_k=32)
        assert torch.equal(torch.cat(one, -1)[0], torch.cat([q, k, v], -1)[M - 1])


@gpu
@pytest.mark.parametrize("M", [1, 4, 6, 20, 150])
@pytest.mark.parametrize("K", [64, 1000, 2560])
def test_special_tokens(M, K):
    """Zeros, the smallest and the largest numbers, infinities and NaN stay with their token."""
    x, ws = make(M * K, M, K, 130, n=2)
    want = x.clone()
    rows = torch.arange(M)
    x[rows % 6 == 1] = 0
    x[rows % 6 == 2] *= 2.0**-130
    x[rows % 6 == 3] *= 2.0**120
    x[rows % 6 == 4, K // 2] = float("inf")
    x[rows % 6 == 5, K - 1] = float("nan")
    xd, (g, u) = on(x, ws)
    y = fk.fused_linear_w8a8(xd, *g).cpu()
    z = fk.fused_gate_up_silu_w8a8(xd, *g, *u).cpu()
    bad = (rows % 6 == 4) | (rows % 6 == 5)
    assert y[bad].isnan().all() and z[bad].isnan().all()
    zero = rows % 6 == 1
    assert (y[zero] == 0).all() and (z[zero] == 0).all()
    fine = (rows % 6 == 0) | (rows % 6 == 3)
    check_linear(y[fine], x[fine], ws[0])
    tiny = rows % 6 == 2  # the scale is a denormal number: 2^-149 of itself off, and so are the outputs
    if tiny.any():
        e = exact(x[tiny], ws[0])
        step = codes(x[tiny])[0] @ ws[0][0].double().T * ws[0][1].double() * 2.0**-149
        assert ((y[tiny].double() - e).abs() <= e.abs() * 2.0**-8 + step.abs() + 2.0**-133).all()
    assert not want.isnan().any()


@gpu
def test_strides_and_views():
    x, ws = make(3, 24, 512, 128, n=2)
    big = torch.zeros(24, 700, dtype=torch.bfloat16)
    big[:, 3:515] = x
    xd, (g, u) = on(x, ws)
    want = fk.fused_linear_w8a8(xd, *g)
    view = big.to(DEV)[:, 3:515]
    assert torch.equal(fk.fused_linear_w8a8(view, *g), want)
    assert torch.equal(fk.fused_linear_w8a8(xd.T.contiguous().T, *g), want)
    assert torch.equal(fk.fused_linear_w8a8(xd.view(2, 3, 4, 512), *g).view(24, 128), want)
    q = torch.zeros(128, 601, dtype=torch.int8, device=DEV)
    for at in (0, 1, 7, 64):  # weight rows at any stride and alignment
        q[:, at : at + 512] = g[0]
        assert torch.equal(fk.fused_linear_w8a8(xd, q[:, at : at + 512], g[1]), want)
        assert torch.equal(fk.fused_linear_w8a8(xd[:3], q[:, at : at + 512], g[1]), want[:3])
    s = torch.zeros(256, device=DEV)
    s[::2] = g[1]
    assert torch.equal(fk.fused_linear_w8a8(xd, g[0], s[::2]), want)
    assert fk.fused_linear_w8a8(xd[:0], *g).shape == (0, 128)
    assert torch.equal(fk.fused_gate_up_silu_w8a8(xd, *g, *g), fk.fused_gate_up_silu_w8a8(view, *g, *g))


@gpu
@pytest.mark.parametrize("M", [1, 3, 5, 17, 70, 300])
@pytest.mark.parametrize("K,step", [(1000, 1008), (2541, 2560), (130, 1024)])
def test_padded_weight_rows(M, K, step):
    """Rows of any length at a stride of whole 16 bytes: what lies between them has no part."""
    x, ws = make(M + K, M, K, 130, n=2)
    xd = x.to(DEV)
    pad = []
    for q, s in ws:
        b = torch.full((130, step), 127, dtype=torch.int8)
        b[:, :K] = q
        pad.append((b.to(DEV)[:, :K], s.to(DEV)))
    check_linear(fk.fused_linear_w8a8(xd, *pad[0]), x, ws[0])
    check_gate_up(fk.fused_gate_up_silu_w8a8(xd, *pad[0], *pad[1]), x, *ws)


@gpu
@pytest.mark.parametrize("M,K", [(1, 1024), (3, 2541), (12, 2560), (70, 1024), (70, 2541)])
def test_graph_replays(M, K):
    x, ws = make(M, M, K, 320, n=2)
    xd, (g, u) = on(x, ws)
    static = torch.zeros_like(xd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fk.fused_gate_up_silu_w8a8(static, *g, *u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = fk.fused_linear_w8a8(static, *g), fk.fused_gate_up_silu_w8a8(static, *g, *u)
    for i in range(3):
        xi = (xd * (i + 1)).roll(i, 1)
        static.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fk.fused_linear_w8a8(xi, *g)) and torch.equal(z, fk.fused_gate_up_silu_w8a8(xi, *g, *u))


@gpu
def test_two_streams():
    """Calls on two streams at once do not share what they work in."""
    x, ws = make(1, 600, 1024, 1024)
    xd, (w,) = on(x, ws)
    want = [fk.fused_linear_w8a8(xd * (i + 1), *w) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fk.fused_linear_w8a8(xd * (i + 1), *w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# ------------------------------------------------------------- the swapped model


@gpu
@pytest.mark.parametrize("fuse_norm", [False, True])
@pytest.mark.parametrize("rows", [1, 7, 90])
def test_swapped_model(fuse_norm, rows):
    """The swapped modules are the calls on the packed weights, and near the weight-only form."""
    c = harness.Cfg(vocab_size=300, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                    intermediate_size=512, max_position_embeddings=128)
    model = harness.tiny_model(c, state=harness.tiny_state(c, embed_scale=0.3), device=DEV)
    a = fk.apply_triton_kernels(copy.deepcopy(model), int8=True, linear_down_o=True, fuse_norm=fuse_norm)
    b = fk.apply_triton_kernels(copy.deepcopy(model), int8=True, a8=True, linear_down_o=True, fuse_norm=fuse_norm)
    fk.prewarm_triton_kernels(b)
    ids = torch.randint(0, 300, (1, rows), generator=torch.Generator().manual_seed(rows)).to(DEV)
    with torch.inference_mode():
        h = torch.randn(rows, 256, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
        ffn, attn = b.layers[0].ffn, b.layers[0].attn
        if fuse_norm:
            n1, n2 = attn.prenorm, ffn.prenorm
            want = fk.fused_rmsnorm_gate_up_silu_w8a8(h, n2.weight, n2.eps, ffn.qg, ffn.sg, ffn.qu, ffn.su)
            qkv = fk.fused_rmsnorm_qkv_w8a8(h, n1.weight, n1.eps, attn.q_qkv, attn.s_qkv, n_q=256, n_k=128)
        else:
            want = fk.fused_gate_up_silu_w8a8(h, ffn.qg, ffn.sg, ffn.qu, ffn.su)
            qkv = fk.fused_qkv_w8a8(h, attn.q_qkv, attn.s_qkv, n_q=256, n_k=128)
        assert torch.equal(ffn.gate_up(h), want) and all(map(torch.equal, attn.project(h), qkv))
        assert torch.equal(ffn.down(want), fk.fused_linear_w8a8(want, ffn.down.q, ffn.down.s))
        y = [m(ids, m.alloc_cache(rows + 4), start_pos=0).float() for m in (a, b)]
    assert torch.nn.functional.cosine_similarity(y[0].flatten(), y[1].flatten(), 0) > 0.99


@gpu
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_modules_of_odd_sizes(rows):
    """Weights whose rows are no whole 16 bytes are kept at a stride that is."""
    lin = torch.nn.Linear(201, 77, bias=False, device=DEV, dtype=torch.bfloat16)
    f = fk.FusedLinear.from_linear(lin, int8=True, a8=True)
    assert f.q.shape == (77, 201) and f.q.stride(0) == 208
    x = make(rows, rows, 201, 1)[0]
    with torch.inference_mode():
        check_linear(f(x.to(DEV)), x, (f.q.cpu(), f.s.cpu()))


@gpu
def test_swapped_model_generates():
    c = harness.Cfg(vocab_size=64, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                    intermediate_size=256)
    m = harness.tiny_model(c, state=harness.tiny_state(c, embed_scale=0.3), device=DEV)
    fk.apply_triton_kernels(m, int8=True, a8=True, linear_down_o=True)
    prompt = [1, 2, 3, 4, 5]
    assert harness.greedy_generate(m, prompt, 8, DEV) == harness.graph_greedy_generate(m, prompt, 8, DEV)
