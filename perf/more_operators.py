"""Operators for serving many or endless texts, measured against plain torch forms.

Three families, as a serving loop of a Qwen3 model uses them:

- ``w8a8``: projections in 8-bit integers: weights with a scale for each output,
  activations with one for each token (``fused_linear_w8a8``, ``fused_qkv_w8a8``,
  ``fused_gate_up_silu_w8a8``).
- ``shared``: a step of a batch of sequences that all continue one long text, whose
  keys and values are held once (``attention_shared`` over a ``KVCacheShared``).
- ``window``: a step over a cache that keeps a window of the last tokens and the
  first few (``attention_window`` over a ``KVCacheWindow``).

Formats
  Weights in 8 bits: q in -127 .. 127 and a scale per row. Activations: with
  top = max|x| of a token, the codes are round(127 x / top), ties to even, and the
  scale is top / 127. The product is scale * scale * the codes' sum.
  The caches are bf16. A window's cache holds position p < sinks in slot p, any other
  in slot sinks + (p - sinks) % ring, with the ring a multiple of 64 that holds the window
  and a step of max_step tokens.
  The token at position p sees positions 0 .. p, with a window those of the last
  ``window`` positions (its own counts) and of the first ``sinks``.

Keys and values are N(0, 1) with a spread of channel sizes (what normalised keys
and x.Wv give), queries alike, so a few keys carry most of a row's weight;
activations N(0, 1) with a few channels of ten times that size, weights N(0, 0.02).
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"

# (hidden, query heads, key/value heads, head size, FFN width)
SHAPES = {
    "0.6b": (1024, 16, 8, 128, 3072),
    "4b": (2560, 32, 8, 128, 9728),
    "8b": (4096, 32, 8, 128, 12288),
}


def listed():
    return [
        # The smallest product: one token's QKV projection of the smallest model.
        {"name": "w8a8-qkv-one-token", "op": "w8a8", "fn": "qkv", "M": 1, "K": 1024, "N": 4096},
        # Verification of a 4-token draft: the widest projection of a layer.
        {"name": "w8a8-gate-up-verify", "op": "w8a8", "fn": "gate_up", "M": 5, "K": 2560, "N": 9728},
        # A batch of 64 sequences decoding together on the largest model.
        {"name": "w8a8-gate-up-batch64", "op": "w8a8", "fn": "gate_up", "M": 64, "K": 4096, "N": 12288},
        # A prompt on rows that no vector width divides.
        {"name": "w8a8-linear-ragged", "op": "w8a8", "fn": "linear", "M": 300, "K": 2541, "N": 9700},
        # A long prompt on the largest model (the largest product).
        {"name": "w8a8-gate-up-prompt", "op": "w8a8", "fn": "gate_up", "M": 4096, "K": 4096, "N": 12288},
        # Four answers to one question on the smallest model. Launches and latency count.
        {"name": "shared-four-answers", "op": "shared", "B": 4, "T": 1, "P": 1000, "pos": 40,
         "Hq": 16, "Hk": 8, "D": 128, "ragged": False},
        # 64 chats under one long system text, of different lengths.
        {"name": "shared-batch64", "op": "shared", "B": 64, "T": 1, "P": 16000, "pos": 700,
         "Hq": 32, "Hk": 8, "D": 128, "ragged": True},
        # Drafts of four tokens verified for eight readers of one book.
        {"name": "shared-verify", "op": "shared", "B": 8, "T": 5, "P": 50001, "pos": 150,
         "Hq": 32, "Hk": 8, "D": 128, "ragged": False},
        # Eight questions of up to 300 tokens about one document, padded to the longest.
        {"name": "shared-questions", "op": "shared", "B": 8, "T": 300, "P": 9000, "pos": 0,
         "Hq": 32, "Hk": 8, "D": 128, "ragged": True},
        # One token of an endless chat on the smallest model.
        {"name": "window-one-token", "op": "window", "B": 1, "T": 1, "pos": 100000, "window": 1024, "sinks": 4,
         "max_step": 64, "Hq": 16, "Hk": 8, "D": 128, "ragged": False},
        # 16 endless chats decoding together, some of them still short.
        {"name": "window-batch16", "op": "window", "B": 16, "T": 1, "pos": 7000, "window": 4096, "sinks": 4,
         "max_step": 64, "Hq": 32, "Hk": 8, "D": 128, "ragged": True},
        # A later chunk of a long prompt.
        {"name": "window-prompt", "op": "window", "B": 1, "T": 4000, "pos": 5001, "window": 2048, "sinks": 4,
         "max_step": 4096, "Hq": 32, "Hk": 8, "D": 128, "ragged": False},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["w8a8", "shared", "window"])
    if op == "w8a8":
        c = {"op": op, "fn": rng.choice(["linear", "qkv", "gate_up"]),
             "M": rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 4096)])}
        hidden, hq, hk, d, inter = SHAPES[rng.choice(list(SHAPES))]
        if rng.random() < 0.35:
            return dict(c, K=_log(rng, 65, 9000), N=_log(rng, 64, 10000))
        if c["fn"] == "qkv":
            return dict(c, K=hidden, N=(hq + 2 * hk) * d)
        if c["fn"] == "gate_up":
            return dict(c, K=hidden, N=inter)
        return dict(c, K=inter, N=hidden) if rng.random() < 0.5 else dict(c, K=hq * d, N=hidden)
    Hq, Hk = rng.choice([(16, 8), (32, 8), (32, 8), (8, 8), (12, 4), (7, 1), (40, 8)])
    c = {"op": op, "Hq": Hq, "Hk": Hk, "D": rng.choice([64, 128, 128])}
    if op == "shared":
        if rng.random() < 0.65:  # decoding and verification
            B = _log(rng, 1, 64)
            return dict(c, B=B, T=rng.choice([1, 1, 1, 2, 3, 5, 9]), P=_log(rng, 10, 50000),
                        pos=rng.choice([0, _log(rng, 1, 700)]), ragged=B > 1 and rng.random() < 0.6)
        return dict(c, B=_log(rng, 1, 8), T=_log(rng, 16, 300), P=_log(rng, 10, 9000),
                    pos=rng.choice([0, 0, _log(rng, 1, 200)]), ragged=rng.random() < 0.5)
    c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice([0, 1, 4, 4, 16, _log(rng, 1, 100)])
    if rng.random() < 0.65:
        B = _log(rng, 1, 16)
        return dict(c, B=B, T=rng.choice([1, 1, 1, 2, 3, 5, 9]), pos=_log(rng, 1, 200000), max_step=64,
                    ragged=B > 1 and rng.random() < 0.6)
    T = _log(rng, 16, 2048)
    return dict(c, B=1, T=T, pos=rng.choice([0, 0, _log(rng, 1, 20000)]), max_step=2048, ragged=False)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _pack8(w):
    """(codes, scales) of a weight in 8 bits."""
    s = w.float().abs().amax(1) / 127
    return (w.float() / s[:, None]).round().clamp(-127, 127).to(torch.int8), s


def _w8a8_inputs(c, seed):
    g = _gen(seed)
    x = _randn(g, c["M"], c["K"])
    x[:, torch.randint(0, c["K"], (3,), generator=g, device=DEV)] *= 10
    n = 2 if c["fn"] == "gate_up" else 1
    return {"x": x.bfloat16(), "w": [_pack8(_randn(g, c["N"], c["K"], scale=0.02).bfloat16()) for _ in range(n)]}


def _ring(c):
    """Slots of a window's cache behind the sinks."""
    return -(-(c["window"] + c["max_step"] - 1) // 64) * 64


def _attention_inputs(c, seed):
    """q, k, v of the new tokens; the own tokens of each sequence before them (those that a
    window's ring holds); the shared text or the sinks; where each sequence goes
    on (``start``, counted behind the shared text) and how many tokens it has (``count``)."""
    g = _gen(seed)
    B, T, D, Hk = c["B"], c["T"], c["D"], c["Hk"]
    start = torch.full((B,), c["pos"], dtype=torch.long, device=DEV)
    count = torch.full((B,), T, dtype=torch.long, device=DEV)
    if c["ragged"]:
        low = torch.randint(c["pos"] // 2, c["pos"] + 1, (B,), generator=g, device=DEV)
        start[1:] = low[1:]
        if T > 9:  # questions of different lengths
            count[1:] = torch.randint(T // 4, T + 1, (B,), generator=g, device=DEV)[1:]
    spread = (0.3 * _randn(g, 2, Hk, D)).exp()
    window = c["op"] == "window"
    d = {"start": start, "count": count, "q": (1.5 * _randn(g, B, T, c["Hq"], D)).bfloat16()}
    n = min(c["pos"], _ring(c)) if window else c["pos"]
    for i, name in enumerate("kv"):
        fixed = (B, c["sinks"]) if window else (c["P"],)
        d["fix_" + name] = (_randn(g, *fixed, Hk, D) * spread[i]).bfloat16()
        d["hist_" + name] = (_randn(g, B, n, Hk, D) * spread[i]).bfloat16()
        d[name] = (_randn(g, B, T, Hk, D) * spread[i]).bfloat16()
    if window:  # the sinks are the first tokens of a history that begins there
        d["first"] = (start - n).clamp(min=0)
        for name in "kv":
            for j in range(min(c["sinks"], n)):
                here = (d["first"] == 0) & (j < start)
                d["hist_" + name][:, j] = torch.where(here[:, None, None], d["fix_" + name][:, j], d["hist_" + name][:, j])
    return d


def prepare(c, seed):
    if c["op"] == "w8a8":
        return dict(_w8a8_inputs(c, seed), c=c)
    d = dict(_attention_inputs(c, seed), c=c)
    k, v, start, count = d.pop("hist_k"), d.pop("hist_v"), d["start"], d["count"]
    fix_k, fix_v = d.pop("fix_k"), d.pop("fix_v")
    n = k.shape[1]
    d["lengths"] = count if c["ragged"] and c["T"] > 9 else None
    if c["op"] == "shared":
        text = [t.transpose(0, 1).contiguous() for t in (fix_k, fix_v)]  # [Hk, P, D]
        if own:
            from llms_amd import kernels as fk

            d["cache"] = fk.KVCacheShared([text[0]], [text[1]], max_batch=c["B"], max_new=c["pos"] + c["T"])
            if n:
                d["cache"].write(0, k, v, c["P"], lengths=start)
            d["at"] = c["P"] + start if c["ragged"] else c["P"] + c["pos"]
        else:
            d["text"] = text
            d["k_own"], d["v_own"] = (_plain_own(t, start, c["pos"] + c["T"]) for t in (k, v))
        return d
    first = d.pop("first")
    if own:
        from llms_amd import kernels as fk

        d["cache"] = fk.KVCacheWindow.alloc(1, c["window"], sinks=c["sinks"], max_step=c["max_step"],
                                            max_batch=c["B"], n_kv_heads=c["Hk"], head_dim=c["D"], device=DEV)
        if c["sinks"]:
            d["cache"].write(0, fix_k, fix_v, 0, lengths=start.clamp(max=c["sinks"]))
        if n:
            d["cache"].write(0, k, v, first, lengths=start - first)
        d["at"] = start if c["ragged"] else c["pos"]
    else:
        at = first[:, None] + torch.arange(n, device=DEV)
        for name, sink, hist in (("k_own", fix_k, k), ("v_own", fix_v, v)):
            buf = torch.zeros(c["B"], c["Hk"], c["sinks"] + _ring(c), c["D"], dtype=hist.dtype, device=DEV)
            buf[:, :, : c["sinks"]] = sink.transpose(1, 2)
            buf[:, :, : c["sinks"]].masked_fill_(
                (torch.arange(c["sinks"], device=DEV) >= start[:, None])[:, None, :, None], 0)
            d[name] = _plain_put(buf, hist, _slots(c, at), at < start[:, None])
    return d


# ------------------------------------------------------------ plain forms


def _unpacked_product(x, w):
    """x [M, K] in 8-bit codes times w (codes, scales), in 32 bits."""
    top = x.abs().amax(1, keepdim=True)
    # 127 x is exact and so is its quotient at a tie: every tie is seen as one
    codes = torch.where(top > 0, 127 * x / top, 0.0).round()
    return (codes @ w[0].float().T) * (top / 127) * w[1]


def _heads(c):
    """Rows of a QKV weight that are queries, keys and values."""
    n_k = c["N"] // 4
    return [c["N"] - 2 * n_k, n_k, n_k]


def _plain_w8a8(d):
    c = d["c"]
    y = [_unpacked_product(d["x"].float(), w) for w in d["w"]]
    if c["fn"] == "gate_up":
        return (y[0] / (1 + (-y[0]).exp()) * y[1]).bfloat16()
    return y[0].bfloat16().split(_heads(c), 1) if c["fn"] == "qkv" else y[0].bfloat16()


def _plain_own(hist, start, size):
    """[B, n, H, D] tokens as a cache [B, H, size, D], those before ``start`` of each sequence."""
    B, n, H, D = hist.shape
    buf = torch.zeros(B, H, size, D, dtype=hist.dtype, device=DEV)
    live = torch.arange(n, device=DEV) < start[:, None]
    buf[:, :, :n] = torch.where(live[:, :, None, None], hist, 0).transpose(1, 2)
    return buf


def _slots(c, p):
    s = c["sinks"]
    return torch.where(p < s, p, s + (p - s) % _ring(c))


def _plain_put(buf, x, slot, live):
    """buf [B, H, size, D] with x [B, T, H, D] at ``slot`` [B, T] where ``live``, in place."""
    b, t = live.nonzero(as_tuple=True)
    buf.transpose(1, 2)[b, slot[b, t]] = x[b, t]
    return buf


def _plain_scatter(buf, x, slot, live):
    """x [B, T, H, D] in the cache buf [B, H, size, D] at ``slot`` where ``live``; the cache as 32 bits."""
    idx = slot[:, None, :, None].expand(-1, buf.shape[1], -1, buf.shape[3])
    buf.scatter_(2, idx, torch.where(live[:, None, :, None], x.transpose(1, 2), buf.gather(2, idx)))
    return buf.float()


def _plain_new(d, slot):
    """The step's keys and values put into the cache, and which tokens there are."""
    live = torch.arange(d["c"]["T"], device=DEV) < d["count"][:, None]
    return (_plain_scatter(d["k_own"], d["k"], slot, live), _plain_scatter(d["v_own"], d["v"], slot, live), live)


def _plain_shared(d):
    c, start = d["c"], d["start"]
    B, T, Hk, D, P, G = c["B"], c["T"], c["Hk"], c["D"], c["P"], c["Hq"] // c["Hk"]
    pos = start[:, None] + torch.arange(T, device=DEV)
    k, v, live = _plain_new(d, pos)
    q = d["q"].float().view(B, T, Hk, G, D).permute(2, 0, 3, 1, 4)  # [Hk, B, G, T, D]
    S = k.shape[2]
    far = torch.matmul(q.reshape(Hk, B * G * T, D), d["text"][0].float().transpose(1, 2).contiguous())
    near = torch.matmul(q.transpose(0, 1).reshape(B, Hk, G * T, D), k.transpose(2, 3).contiguous())
    hidden = torch.arange(S, device=DEV) > pos[:, :, None]
    near = near.view(B, Hk, G, T, S).masked_fill(hidden[:, None, None], -math.inf)
    far = far.view(Hk, B, G, T, P).transpose(0, 1)
    x = torch.cat([far, near], -1) * D ** -0.5
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    y = torch.matmul(p[..., :P].transpose(0, 1).reshape(Hk, B * G * T, P), d["text"][1].float())
    y = y.view(Hk, B, G, T, D).transpose(0, 1) + torch.matmul(p[..., P:].reshape(B, Hk, G * T, S), v).view(B, Hk, G, T, D)
    y = y.permute(0, 3, 1, 2, 4).reshape(B, T, c["Hq"], D)
    return {"y": torch.where(live[:, :, None, None], y, 0.0).bfloat16(), "k": d["k_own"], "v": d["v_own"]}


def _plain_window(d):
    c, start = d["c"], d["start"]
    B, T, Hk, D, G, R = c["B"], c["T"], c["Hk"], c["D"], c["Hq"] // c["Hk"], _ring(c)
    pos = start[:, None] + torch.arange(T, device=DEV)
    k, v, live = _plain_new(d, _slots(c, pos))
    # the position in each slot: the last one up to the step's end that falls there
    s = c["sinks"]
    last = (start + d["count"] - 1)[:, None]
    ring = torch.arange(R, device=DEV)
    at = torch.cat([torch.arange(s, device=DEV).expand(B, s), last - (last - s - ring) % R], 1)
    at = torch.where(at < 0, torch.iinfo(torch.long).max, at)[:, None]
    own_pos = pos[:, :, None]
    seen = (at <= own_pos) & ((at > own_pos - c["window"]) | (at < s))
    seen &= (at >= s) | (torch.arange(s + R, device=DEV) < s)
    q = d["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    x = x.view(B, Hk, G, T, s + R).masked_fill(~seen[:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(B, Hk, G * T, s + R)
    y = torch.matmul(p, v).view(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, c["Hq"], D)
    return {"y": torch.where(live[:, :, None, None], y, 0.0).bfloat16(), "k": d["k_own"], "v": d["v_own"]}


_PLAIN = {"w8a8": _plain_w8a8, "shared": _plain_shared, "window": _plain_window}


# ---------------------------------------------------- the framework's calls


def _own_w8a8(d):
    from llms_amd import kernels as fk

    c, w = d["c"], d["w"]
    if c["fn"] == "gate_up":
        return fk.fused_gate_up_silu_w8a8(d["x"], *w[0], *w[1])
    if c["fn"] == "qkv":
        n_q, n_k, _ = _heads(c)
        return fk.fused_qkv_w8a8(d["x"], *w[0], n_q=n_q, n_k=n_k)
    return fk.fused_linear_w8a8(d["x"], *w[0])


def _own_attention(d):
    from llms_amd import kernels as fk

    call = fk.attention_shared if d["c"]["op"] == "shared" else fk.attention_window
    y = call(d["q"], d["k"], d["v"], d["cache"], 0, d["at"], lengths=d["lengths"])
    return {"y": y, "k": d["cache"].k[0], "v": d["cache"].v[0]}


_OWN = {"w8a8": _own_w8a8, "shared": _own_attention, "window": _own_attention}


def run(d):
    return (_OWN if own else _PLAIN)[d["c"]["op"]](d)


# ------------------------------------------------------------------- work


def work(c):
    if c["op"] == "w8a8":
        n = (2 if c["fn"] == "gate_up" else 1) * c["N"]
        return {"bytes": n * (c["K"] + 4) + 2 * c["M"] * (c["K"] + c["N"]), "flops": 2.0 * c["M"] * n * c["K"]}
    B, T, Hq, Hk, D, pos = (c[i] for i in ("B", "T", "Hq", "Hk", "D", "pos"))
    io = B * T * D * (4 * Hq + 8 * Hk)  # q and y, the new keys and values in and into the cache
    some = 1 + 0.75 * (B - 1) if c["ragged"] else B  # of all sequences together
    rows = T * (1 + 0.625 * (B - 1)) if c["ragged"] and T > 9 else T * B
    if c["op"] == "shared":
        pairs = rows * (c["P"] + T / 2) + T * some * pos
        return {"bytes": 4 * Hk * D * (c["P"] + some * pos) + io, "flops": 4.0 * Hq * D * pairs}
    old = min(pos, c["window"] - 1 + c["sinks"])
    seen = min(pos + T / 2, c["window"] + c["sinks"])
    return {"bytes": 4 * Hk * D * old * B + io, "flops": 4.0 * Hq * D * B * T * seen}


# ------------------------------------------------------------------ exact


def _exact_w8a8(c, seed):
    d = _w8a8_inputs(c, seed)
    x = d["x"].double()
    top = x.abs().max(1, keepdim=True).values
    xq = torch.round(x * 127 / top.clamp(min=1e-300)) * top / 127
    y = [xq @ (q.double() * s.double()[:, None]).T for q, s in d["w"]]
    if c["fn"] == "gate_up":
        return y[0] * torch.sigmoid(y[0]) * y[1]
    return y[0].split(_heads(c), 1) if c["fn"] == "qkv" else y[0]


def _exact_attention(c, seed):
    d = _attention_inputs(c, seed)
    T, Hk, D, G = c["T"], c["Hk"], c["D"], c["Hq"] // c["Hk"]
    window = c["op"] == "window"
    size = c["sinks"] + _ring(c) if window else c["pos"] + T
    out = {"y": torch.zeros(d["q"].shape, dtype=torch.double, device=DEV)}
    for name in "kv":
        out[name] = torch.zeros(c["B"], Hk, size, D, dtype=torch.double, device=DEV)
    for b, (p, n) in enumerate(zip(d["start"].tolist(), d["count"].tolist())):
        kv = {}
        for name in "kv":
            hist, new = d["hist_" + name][b], d[name][b, :n]
            if window:
                lo = max(0, p - hist.shape[0])  # the position of hist[0]
                fixed = d["fix_" + name][b, : min(c["sinks"], p)]
                rows = torch.cat([fixed[: min(lo, c["sinks"])], hist[: p - lo], new]).double()
                at = torch.cat([torch.arange(min(lo, c["sinks"]), device=DEV), torch.arange(lo, p + n, device=DEV)])
                keep = at >= max(0, p + n - _ring(c))
                keep |= at < c["sinks"]
                s = at[keep]
                s = torch.where(s < c["sinks"], s, c["sinks"] + (s - c["sinks"]) % _ring(c))
                out[name][b, :, s] = rows[keep].transpose(0, 1)
            else:
                rows = torch.cat([d["fix_" + name], hist[:p], new]).double()
                at = torch.arange(c["P"] + p + n, device=DEV)
                out[name][b, :, : p + n] = rows[c["P"] :].transpose(0, 1)
            kv[name] = rows.transpose(0, 1).contiguous()  # [Hk, n, D]
        me = torch.arange(p, p + n, device=DEV)[:, None] + (0 if window else c["P"])
        hidden = at > me
        if window:
            hidden |= (at <= me - c["window"]) & (at >= c["sinks"])
        for h in range(c["Hq"]):
            q = d["q"][b, :n, h].double() / math.sqrt(D)
            w = (q @ kv["k"][h // G].T).masked_fill(hidden, -math.inf).softmax(1)
            out["y"][b, :n, h] = w @ kv["v"][h // G]
    return out


def exact(c, seed):
    return _exact_w8a8(c, seed) if c["op"] == "w8a8" else _exact_attention(c, seed)
