"""Projections on 4-bit weights against 64 bits, their packing and the swapped model."""

from __future__ import annotations

import math

import pytest
import torch

from llms_amd import _lib
from llms_amd import kernels as fk

DEV = "cuda"
GROUPS = [32, 64, 128]


def pack(w, group):
    """The packing's definition (32-bit arithmetic with correctly rounded division)."""
    N, K = w.shape
    G = -(-K // group)
    x = torch.zeros(N, G * group)
    x[:, :K] = w.float()
    x = x.view(N, G, group)
    m, e = torch.frexp(x.abs().amax(2) / 7)
    s = torch.ldexp((m * 32).round() / 32, e)
    q = torch.where(s[..., None] > 0, x / s[..., None], 0.0).round().clamp(-7, 7)
    u = (q + 8).to(torch.uint8).view(N, -1)[:, : K + K % 2].reshape(N, -1, 2)
    return u[..., 0] | (u[..., 1] << 4), s.to(torch.bfloat16)


def make(seed, M, K, N, group, n=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).bfloat16()
    ws = [pack((torch.randn(N, K, generator=g) * 0.02).bfloat16(), group) for _ in range(n)]
    return x, ws


def exact(x, qs, group):
    K = x.shape[-1]
    q, s = (t.cpu() for t in qs)
    w = torch.stack([q & 15, q >> 4], 2).view(q.shape[0], -1)[:, :K].double() - 8
    return x.cpu().double() @ (w * s.double().repeat_interleave(group, 1)[:, :K]).T, \
        x.cpu().double().abs() @ ((w.abs() + 136) * s.double().repeat_interleave(group, 1)[:, :K].abs()).T


def check_linear(y, x, qs, group):
    """One rounding to bf16 (2^-8 of the value at most: half a step is 2^-9 of the next
    power of two) on an fp32 sum whose terms, with the 136 that the codes carry, are off
    by 2^-24 of their size in each of at most ~64 sequential additions and the last
    ones of the groups and waves."""
    e, size = exact(x, qs, group)
    K = x.shape[-1]
    tol = e.abs() * 2.0**-8 + size * 2.0**-24 * (8 + math.sqrt(K))
    err = (y.cpu().double() - e).abs()
    assert (err <= tol).all(), (err / tol).max()


def check_gate_up(y, x, g, u, group):
    """One rounding of the product to bf16. Before it: g and u off by their fp32 sums'
    errors, silu's slope under 1.1, and a dozen fp32 operations of 2^-24 each (the
    exponential and the division of silu, the product)."""
    (eg, sg), (eu, su) = exact(x, g, group), exact(x, u, group)
    K = x.shape[-1]
    silu = eg * torch.sigmoid(eg)
    f32 = 2.0**-24 * (8 + math.sqrt(K))
    dg, du = sg * f32, su * f32
    ds = 1.1 * dg + (silu.abs() + 1.1 * dg) * 12 * 2.0**-24
    tol = ds * (eu.abs() + du) + silu.abs() * du
    tol = tol + ((silu * eu).abs() + tol) * 2.0**-8 + 1e-30
    err = (y.cpu().double() - silu * eu).abs()
    assert (err <= tol).all(), (err / tol).max()


# ------------------------------------------------------------- refusals (CPU)


def test_refusals_on_the_cpu():
    x, ((q, s),) = make(0, 3, 256, 40, 128)
    with pytest.raises(ValueError, match="HIP"):
        fk.fused_linear_w4(x, q, s)
    with pytest.raises(ValueError, match="group"):
        fk.fused_linear_w4(x, q, s, group=16)
    with pytest.raises(ValueError, match="s shape"):
        fk.fused_linear_w4(x, q, s, group=64)
    with pytest.raises(ValueError, match="does not hold"):
        fk.fused_linear_w4(x[:, :100], q, s)
    with pytest.raises(TypeError, match="uint8"):
        fk.fused_linear_w4(x, q.to(torch.int8), s)
    with pytest.raises(TypeError, match="bfloat16"):
        fk.fused_linear_w4(x, q, s.float())
    with pytest.raises(TypeError, match="bfloat16"):
        fk.fused_linear_w4(x.float(), q, s)
    with pytest.raises(ValueError, match="n_q"):
        fk.fused_qkv_w4(x, q, s, n_q=20, n_k=11)
    with pytest.raises(ValueError, match="n_q"):
        fk.fused_qkv_w4(x, q, s, n_q=0, n_k=20)
    with pytest.raises(ValueError, match="qu shape"):
        fk.fused_gate_up_silu_w4(x, q, s, q[:20], s[:20])
    with pytest.raises(ValueError, match="eps"):
        fk.fused_rmsnorm_qkv_w4(x, torch.ones(256).bfloat16(), -1.0, q, s, n_q=20, n_k=10)
    with pytest.raises(ValueError, match="norm weight"):
        fk.fused_rmsnorm_gate_up_silu_w4(x, torch.ones(255).bfloat16(), 1e-6, q, s, q, s)
    with pytest.raises(ValueError, match="2D"):
        fk.quantize_w4(x[0])
    with pytest.raises(ValueError, match="group"):
        fk.quantize_w4(x, 48)
    with pytest.raises(ValueError, match="at least one"):
        fk.quantize_w4(x[:, :0])
    with pytest.raises(ValueError, match="HIP"):
        fk.quantize_w4(x)
    with pytest.raises(ValueError, match="exclude"):
        fk.apply_triton_kernels(torch.nn.Module(), int8=True, int4=True)
    for group in (0, 48):
        with pytest.raises(ValueError, match="w4_group"):
            fk.apply_triton_kernels(torch.nn.Module(), int4=True, w4_group=group)


def test_c_entry_refusals():
    lib = _lib.capi()
    P = 4096  # never dereferenced: every call below is refused before a launch
    assert lib.fp_w4_workspace_bytes(4, 96, 256, 0, 0) == 0
    need = lib.fp_w4_workspace_bytes(20, 96, 256, 0, 0)
    assert need > 0 and lib.fp_w4_workspace_bytes(0, 96, 256, 0, 1) == 0
    assert lib.fp_w4_workspace_bytes(65, 96, 256, 1, 0) >= 65 * 256 * 2  # x as the tiles read it
    assert lib.fp_w4_workspace_bytes(65, 96, 256, 1, 1) >= 2 * 65 * 256 * 2  # and as the norm wrote it
    assert lib.fp_w4_workspace_bytes(2, 2, 5, 1, 0) > 0  # weights of under 16 bytes
    ok = dict(x=P, ldx=256, gamma=None, eps=0.0, q=P, ldq=128, s=P, lds=2, group=128, y=P, ldy=96,
              M=20, N=96, K=256, ws=P, nb=need)

    def call(**kw):
        a = dict(ok, **kw)
        one = lib.fp_linear_w4(a["x"], a["ldx"], a["gamma"], a["eps"], a["q"], a["ldq"], a["s"], a["lds"],
                               a["group"], a["y"], a["ldy"], a["M"], a["N"], a["K"], a["ws"], a["nb"], None)
        nb = a["nb"] if "nb" in kw else lib.fp_w4_workspace_bytes(20, 96, 256, 1, 0)
        two = lib.fp_gate_up_silu_w4(a["x"], a["ldx"], a["gamma"], a["eps"], P, 128, P, 2, a["q"], a["ldq"],
                                     a["s"], a["lds"], a["group"], a["y"], a["ldy"], a["M"], a["N"], a["K"],
                                     a["ws"], nb, None)
        assert one == two, kw
        return one

    NULL, SHAPE, STRIDE, WORKSPACE = 1, 2, 3, 6
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(group=16), dict(group=0), dict(gamma=P, eps=-1.0),
               dict(gamma=P, eps=math.nan), dict(M=1 << 40)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(ldx=255), dict(ldq=127), dict(lds=1), dict(ldy=95), dict(ldq=1 << 26),
               dict(lds=1 << 26), dict(ldx=1 << 26),
               dict(x=P + 1), dict(s=P + 1), dict(y=P + 1)):
        assert call(**kw) == STRIDE, kw
    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(y=None)):
        assert call(**kw) == NULL, kw
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=P + 8)):
        assert call(**kw) == WORKSPACE, kw
    assert call(M=0) == 0

    def quant(**kw):
        a = dict(dict(w=P, ldw=256, q=P, ldq=128, s=P, lds=2, N=96, K=256, group=128), **kw)
        return lib.fp_quantize_w4(a["w"], a["ldw"], a["q"], a["ldq"], a["s"], a["lds"], a["N"], a["K"],
                                  a["group"], None)

    assert quant(group=100) == SHAPE and quant(K=0) == SHAPE and quant(N=-1) == SHAPE
    assert quant(ldw=255) == STRIDE and quant(ldq=127) == STRIDE and quant(lds=1) == STRIDE
    assert quant(w=None) == NULL and quant(N=0) == 0


# ------------------------------------------------------------------- packing


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("N,K", [(1, 1), (3, 7), (16, 128), (40, 200), (7, 2541), (300, 1024)])
def test_packing(N, K, group):
    g = torch.Generator().manual_seed(N + K)
    w = torch.randn(N, K, generator=g) * torch.exp(4 * torch.randn(N, 1, generator=g))
    w[0, : K // 2] = 0
    w[N // 2, K // 3 :] *= 1e-6
    w = w.bfloat16()
    q, s = fk.quantize_w4(w.to(DEV), group)
    eq, es = pack(w, group)
    assert torch.equal(s.cpu(), es) and torch.equal(q.cpu(), eq)
    back = fk.dequantize_w4(q, s, K, group=group).cpu()
    code = torch.stack([eq & 15, eq >> 4], 2).view(N, -1)[:, :K].double() - 8
    value = code * es.double().repeat_interleave(group, 1)[:, :K]
    assert torch.equal(back.double(), value)  # exact in bf16
    # half a step of s, and up to 7.25 s where the scale was rounded down
    assert ((value - w.double()).abs() <= 0.5 * es.double().repeat_interleave(group, 1)[:, :K]).all()
    wide = torch.randn(N, K + 5, generator=g).bfloat16().to(DEV)
    for t in (wide[:, 3 : K + 3], wide.t().contiguous().t()[:, :K]):
        a, b = fk.quantize_w4(t, group)
        assert torch.equal(a.cpu(), pack(t.cpu(), group)[0])


@pytest.mark.gpu
def test_packing_of_non_finite_and_tiny_groups():
    w = torch.full((4, 256), 0.5, dtype=torch.bfloat16)
    w[0, 5], w[1, 200] = math.inf, math.nan
    w[2, :128] = 1e-38
    w[3, 0] = torch.finfo(torch.bfloat16).max
    q, s = (t.cpu() for t in fk.quantize_w4(w.to(DEV), 128))
    assert s[0, 0].isnan() and not s[0, 1].isnan() and s[1, 1].isnan()
    assert s[2, 0] == 0 and (q[2, :64] == 0x88).all()
    assert s[3, 0].isfinite() and (7 * s[3, 0].double()) <= torch.finfo(torch.bfloat16).max
    x = torch.ones(2, 256, dtype=torch.bfloat16, device=DEV)
    for M in (2, 70):
        y = fk.fused_linear_w4(x[:1].repeat(M, 1), q.to(DEV), s.to(DEV)).cpu()
        assert y[:, :2].isnan().all() and y[:, 2].isfinite().all()


# ------------------------------------------------------------------- numerics

SHAPES = [(1, 1, 1), (1, 33, 17), (1, 128, 16), (2, 130, 5), (3, 1024, 64), (5, 2541, 50), (16, 512, 100),
          (17, 640, 33), (33, 384, 130), (64, 1000, 20), (65, 513, 70), (130, 256, 300), (1, 9728, 48),
          (4, 12288, 32), (64, 4100, 97), (20, 40, 37), (70, 96, 20), (40, 3, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(M, K, N, group):
    x, (w,) = make(M + K + N, M, K, N, group)
    y = fk.fused_linear_w4(x.to(DEV), w[0].to(DEV), w[1].to(DEV), group=group)
    assert y.shape == (M, N) and y.dtype == torch.bfloat16
    check_linear(y, x, w, group)


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gate_up(M, K, N, group):
    x, (g, u) = make(M + K + N + 1, M, K, N, group, 2)
    y = fk.fused_gate_up_silu_w4(x.to(DEV), *(t.to(DEV) for t in g), *(t.to(DEV) for t in u), group=group)
    check_gate_up(y, x, g, u, group)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 64, 100])
@pytest.mark.parametrize("K", [1024, 1001])
def test_offsets_of_x_cancel(M, K):
    """x far from zero: the 136 on every code has to leave the sum again."""
    x, (w,) = make(7, M, K, 40, 64)
    x = (x.float() + 20).bfloat16()
    y = fk.fused_linear_w4(x.to(DEV), w[0].to(DEV), w[1].to(DEV), group=64)
    check_linear(y, x, w, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 40, 80])
def test_qkv_norm_and_views(M):
    K, n_q, n_k = 640, 96, 40
    x, (w,) = make(M, M, K, n_q + 2 * n_k, 128)
    gamma = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(1))).bfloat16()
    wd, xd = [t.to(DEV) for t in w], x.to(DEV)
    y = fk.fused_linear_w4(xd, *wd)
    q, k, v = fk.fused_qkv_w4(xd.view(1, M, K), *wd, n_q=n_q, n_k=n_k)
    assert torch.equal(torch.cat([q, k, v], -1)[0], y) and k.data_ptr() == q.data_ptr() + 2 * n_q
    from llms_amd.kernels._eager import RMSNorm

    norm = RMSNorm(K).to(DEV, torch.bfloat16)
    with torch.no_grad():
        norm.weight.copy_(gamma)
        xn = norm(xd)
    a = fk.fused_rmsnorm_qkv_w4(xd, gamma.to(DEV), norm.eps, *wd, n_q=n_q, n_k=n_k)
    check_linear(torch.cat(a, -1), xn.cpu(), w, 128)
    spread = gamma.repeat_interleave(2).to(DEV)[::2]
    b = fk.fused_rmsnorm_qkv_w4(xd, spread, norm.eps, *wd, n_q=n_q, n_k=n_k)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    g = fk.fused_rmsnorm_gate_up_silu_w4(xd, gamma.to(DEV), norm.eps, *wd, *wd)
    check_gate_up(g, xn.cpu(), w, w, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 20, 64, 90])
def test_strides(M):
    """Rows off the 16-byte grid, spread rows, strided inner dims: the same sums."""
    K, N = 512, 70
    x, (w,) = make(M, M, K, N, 64)
    wide = torch.full((M, K + 40), math.nan, dtype=torch.bfloat16, device=DEV)
    qw = torch.zeros(N, K // 2 + 31, dtype=torch.uint8, device=DEV)
    sw = torch.full((N, K // 64 + 3), math.nan, dtype=torch.bfloat16, device=DEV)
    wide[:, 3 : K + 3], qw[:, 5 : K // 2 + 5], sw[:, 1 : K // 64 + 1] = x.to(DEV), w[0].to(DEV), w[1].to(DEV)
    xs = [x.to(DEV), wide[:, 3 : K + 3], x.t().contiguous().t().to(DEV)]
    qs = [w[0].to(DEV), qw[:, 5 : K // 2 + 5]]
    ss = [w[1].to(DEV), sw[:, 1 : K // 64 + 1]]
    for xi in xs:
        for qi, si in zip(qs, ss):
            check_linear(fk.fused_linear_w4(xi, qi, si, group=64), x, w, 64)
    same = fk.fused_linear_w4(xs[0][:1].expand(M, K), qs[0], ss[0], group=64)
    check_linear(same, x[:1].expand(M, K), w, 64)
    assert fk.fused_linear_w4(xs[0][:0], qs[0], ss[0], group=64).shape == (0, N)


@pytest.mark.gpu
def test_rows_do_not_mix():
    """A NaN or an infinity in one row of x stays in that row."""
    x, (w,) = make(5, 20, 512, 48, 128)
    x[3, 100], x[7, 30] = math.nan, math.inf
    y = fk.fused_linear_w4(x.to(DEV), w[0].to(DEV), w[1].to(DEV)).cpu()
    assert y[3].isnan().all() and not y[7].isfinite().any()
    keep = [r for r in range(20) if r not in (3, 7)]
    check_linear(y[keep], x[keep], w, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 33, 100])
def test_stream_and_graph(M):
    x, (g, u) = make(M, M, 1024, 96, 128, 2)
    xd, gd, ud = x.to(DEV), [t.to(DEV) for t in g], [t.to(DEV) for t in u]
    eager = fk.fused_gate_up_silu_w4(xd, *gd, *ud)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = fk.fused_gate_up_silu_w4(xd, *gd, *ud)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(eager, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fk.fused_gate_up_silu_w4(xd, *gd, *ud)
    for seed in range(4):
        xd.copy_(make(seed, M, 1024, 1, 128)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fk.fused_gate_up_silu_w4(xd, *gd, *ud))


@pytest.mark.gpu
def test_gradients_are_refused():
    x, (w,) = make(0, 2, 256, 16, 128)
    with pytest.raises(RuntimeError, match="gradients"):
        fk.fused_linear_w4(x.to(DEV).requires_grad_(), w[0].to(DEV), w[1].to(DEV))


# --------------------------------------------------------------------- model


@pytest.mark.gpu
@pytest.mark.parametrize("group,fuse_norm,linear", [(32, False, False), (64, True, True), (128, True, True)])
def test_swapped_model(group, fuse_norm, linear):
    """A model on 4-bit weights against the same model in bf16 on the values that
    the packed weights stand for."""
    from llms_amd import harness as h

    c = h.Cfg(hidden_size=192, intermediate_size=320, head_dim=64)
    state = h.tiny_state(c, seed=4, embed_scale=0.3)
    packed = dict(state)
    kinds = ["q", "k", "v", "gate", "up"] + (["o", "down"] if linear else [])
    for name, w in state.items():
        if name.split(".")[-2] in kinds:
            K = w.shape[1]
            packed[name] = fk.dequantize_w4(*pack(w.bfloat16(), group), K, group=group).float()
    plain = h.tiny_model(c, state=packed, device=DEV)
    m = h.tiny_model(c, state=state, device=DEV)
    fk.apply_triton_kernels(m, int4=True, w4_group=group, fuse_norm=fuse_norm, linear_down_o=linear)
    fk.prewarm_triton_kernels(m, m_values=(1, 4))
    for T in (1, 7, 40):
        tokens = torch.randint(0, 32, (T,), generator=torch.Generator().manual_seed(T)).tolist()
        a, b = (h.teacher_forced_logits(i, tokens, DEV) for i in (m, plain))
        # both round at the same points: they differ by bf16 steps in few places
        assert (a - b).norm() <= 2e-2 * b.norm()
    assert h.greedy_generate(m, [1, 2, 3], 6, DEV) == h.graph_greedy_generate(m, [1, 2, 3], 6, DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("M", [1, 5, 16, 30, 64, 100])
def test_outliers_of_x(M, group):
    """An input far above the others, as the inputs of a down projection have: outputs whose
    code there is zero lose nothing. Whole numbers and scales of 1, and what a code
    carries in the sums (16 + code + 8, at most 31) keeps every partial sum under 2^24: all of
    them are exact, and so is the output but for its rounding."""
    K, N = 1000, 48
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-3, 4, (M, K), generator=g).float()
    x[:, 77], x[:, 801] = 2.0**18, -(2.0**18)
    q = torch.randint(1, 16, (N, K), generator=g)
    q[::2, 77], q[::2, 801] = 8, 8
    packed = (q[:, 0::2] | q[:, 1::2] << 4).to(torch.uint8)
    s = torch.ones(N, -(-K // group), dtype=torch.bfloat16)
    e = x.double() @ (q.double() - 8).T
    y = fk.fused_linear_w4(x.bfloat16().to(DEV), packed.to(DEV), s.to(DEV), group=group)
    assert torch.equal(y.cpu(), e.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("M", [1, 5, 30, 100])
def test_very_large_x(M, group):
    """Finite as long as a group's inputs stay under 2^123 together (31 times that is finite)."""
    K, N = 512, 32
    x, (w,) = make(M, M, K, N, group)
    x = (x.float() * 2.0**100).bfloat16()
    x[:, 7] = 2.0**122
    x[:, 300] = -(2.0**122)
    y = fk.fused_linear_w4(x.to(DEV), w[0].to(DEV), w[1].to(DEV), group=group)
    assert y.isfinite().all()
    check_linear(y, x, w, group)


def test_large_calls_are_taken():
    """Row counts and widths that the bf16 and int8 projections take, too: the grids of the
    larger tiles that such calls run on are far from 2^32 threads."""
    lib = _lib.capi()
    for M, N, K, gate_up in ((90000, 12288, 4096, 1), (8192, 151936, 4096, 0), (1 << 17, 4096, 2560, 0),
                             (349000, 12288, 64, 1)):
        assert lib.fp_w4_workspace_bytes(M, N, K, gate_up, 0) >= M * K * 2, (M, N, K)
    for M, N, K in ((1 << 25, 16, 64), (1 << 24, 1 << 22, 64), (16, 65535 * 64 + 1, 64), (1 << 24, 64, 1 << 20)):
        assert lib.fp_w4_workspace_bytes(M, N, K, 0, 0) == 0, (M, N, K)


@pytest.mark.gpu
def test_a_large_output():
    """More than 2^30 outputs in one call (2.2 GB)."""
    M, K, N = 33000, 64, 33000
    x, (w,) = make(1, M, K, N, 64)
    y = fk.fused_linear_w4(x.to(DEV), w[0].to(DEV), w[1].to(DEV), group=64)
    rows = [0, 63, 64, 16387, 32639, 32999]
    check_linear(y[rows], x[rows], w, 64)
