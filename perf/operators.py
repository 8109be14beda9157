"""Operators of low-bit serving, measured against plain torch forms.

Three families, as a decode or scoring loop of a Qwen3 model uses them:

- ``kv8``: the tokens of a step are put into a key/value cache that is held in
  8 bits with one scale for each block of 64 tokens and head, and attend over it
  (``attention_kv8``). Outputs: the attention output, and the values that the
  cache now holds at the step's positions.
- ``w4``: projections on 4-bit weights with a scale for each group of inputs
  (``fused_linear_w4``, ``fused_qkv_w4``, ``fused_gate_up_silu_w4``).
- ``logprob``: log-probabilities of given tokens, the entropy and the most
  likely tokens of each row of logits (``token_logprobs``).

Formats
  8-bit cache: with m = max|x| over a block's 64 tokens and the head's D entries,
  its scale is m / 127 and its codes round(127 x / m), ties to even. Only whole
  blocks are packed: the tokens of the last, unfinished block count as they came,
  in bf16.
  4-bit weights: the scale of a row's group of G inputs is max|w| / 7 rounded to
  five significant bits, the codes q = round(w / s) in -7 .. 7; byte j of a row
  holds q + 8 of inputs 2j (low half) and 2j + 1; the last byte of an odd row is
  padded with code 0.

Keys and values are N(0, 1) with a spread of channel sizes (what normalised keys
and x.Wv give), queries alike, so a few keys carry most of a row's weight;
activations N(0, 1), weights N(0, 0.02); logits N(0, 2.5) with a few strong
tokens per row.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 64

# (hidden, query heads, key/value heads, head size, FFN width)
SHAPES = {
    "0.6b": (1024, 16, 8, 128, 3072),
    "4b": (2560, 32, 8, 128, 9728),
    "8b": (4096, 32, 8, 128, 12288),
}


def listed():
    return [
        # The smallest step: one token of the smallest model early in a chat.
        # Launches and latency count.
        {"name": "kv8-one-token", "op": "kv8", "B": 1, "T": 1, "pos": 333, "Hq": 16, "Hk": 8,
         "D": 128, "ragged": False},
        # A batch of chats of different lengths decoding together.
        {"name": "kv8-batch16", "op": "kv8", "B": 16, "T": 1, "pos": 4000, "Hq": 32, "Hk": 8,
         "D": 128, "ragged": True},
        # Verification of a 4-token draft far into a long document.
        {"name": "kv8-long-verify", "op": "kv8", "B": 1, "T": 5, "pos": 65001, "Hq": 32, "Hk": 8,
         "D": 128, "ragged": False},
        # The second chunk of a prompt, off the block borders.
        {"name": "kv8-prompt", "op": "kv8", "B": 1, "T": 1000, "pos": 1037, "Hq": 32, "Hk": 8,
         "D": 128, "ragged": False},
        # The smallest product: one token's QKV projection of the smallest model.
        {"name": "w4-qkv-one-token", "op": "w4", "fn": "qkv", "M": 1, "K": 1024, "N": 4096,
         "group": 128},
        # Greedy decoding: the widest projection of a layer at one token.
        {"name": "w4-gate-up-one-token", "op": "w4", "fn": "gate_up", "M": 1, "K": 2560, "N": 9728,
         "group": 128},
        # Verification of a 4-token draft: the longest rows of a layer, finer groups.
        {"name": "w4-down-verify", "op": "w4", "fn": "linear", "M": 5, "K": 9728, "N": 2560,
         "group": 64},
        # A batch of 64 sequences decoding together on the largest model.
        {"name": "w4-gate-up-batch64", "op": "w4", "fn": "gate_up", "M": 64, "K": 4096, "N": 12288,
         "group": 128},
        # A prompt on rows that no vector width divides.
        {"name": "w4-gate-up-ragged", "op": "w4", "fn": "gate_up", "M": 300, "K": 2541, "N": 9700,
         "group": 32},
        # One decode step's answer, with the alternatives that an interface shows.
        {"name": "logprob-one-token", "op": "logprob", "M": 1, "V": 151936, "k": 20,
         "dtype": "bfloat16"},
        # Eight drafts of five tokens, logits kept in 32 bits, a vocabulary of odd size.
        {"name": "logprob-verify-fp32", "op": "logprob", "M": 40, "V": 32003, "k": 8,
         "dtype": "float32"},
        # Scoring a document of 2048 tokens (the largest).
        {"name": "logprob-scoring", "op": "logprob", "M": 2048, "V": 151936, "k": 5,
         "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["kv8", "w4", "logprob"])
    if op == "kv8":
        Hq, Hk = rng.choice([(16, 8), (32, 8), (32, 8), (8, 8), (12, 4), (7, 1), (40, 8)])
        c = {"op": op, "Hq": Hq, "Hk": Hk, "D": rng.choice([64, 128, 128])}
        if rng.random() < 0.65:  # decoding and verification
            B = _log(rng, 1, 24)
            return dict(c, B=B, T=rng.choice([1, 1, 1, 2, 3, 5, 9]),
                        pos=_log(rng, 1, 60000 // B), ragged=B > 1 and rng.random() < 0.6)
        T = _log(rng, 16, 1000)  # prompts and later chunks of one
        return dict(c, B=1, T=T, pos=rng.choice([0, 0, _log(rng, 1, 1000)]), ragged=False)
    if op == "w4":
        c = {"op": op, "fn": rng.choice(["linear", "qkv", "gate_up"]),
             "M": rng.choice([1, 1, _log(rng, 1, 300)]), "group": rng.choice([32, 64, 128, 128])}
        hidden, hq, hk, d, inter = SHAPES[rng.choice(list(SHAPES))]
        if rng.random() < 0.35:
            return dict(c, K=_log(rng, 65, 9000), N=_log(rng, 64, 10000))
        if c["fn"] == "qkv":
            return dict(c, K=hidden, N=(hq + 2 * hk) * d)
        if c["fn"] == "gate_up":
            return dict(c, K=hidden, N=inter)
        return dict(c, K=inter, N=hidden) if rng.random() < 0.5 else dict(c, K=hq * d, N=hidden)
    V = rng.choice([151936, 32000, _log(rng, 100, 151936)])
    return {"op": op, "M": _log(rng, 1, max(1, 150_000_000 // V)) if rng.random() < 0.4 else _log(rng, 1, 64),
            "V": V, "k": rng.choice([0, 1, 5, 20, _log(rng, 1, 32)]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float32", "float16"])}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _positions(c, g):
    """The first position of each sequence's new tokens: pos for the first, from
    half of it on for the others of a ragged batch."""
    start = torch.full((c["B"],), c["pos"], dtype=torch.long, device=DEV)
    if c["ragged"]:
        low = torch.randint(c["pos"] // 2, c["pos"] + 1, (c["B"],), generator=g, device=DEV)
        start[1:] = low[1:]
    return start


def _kv8_inputs(c, seed):
    g = _gen(seed)
    B, T, D, Hk = c["B"], c["T"], c["D"], c["Hk"]
    start = _positions(c, g)
    spread = (0.3 * _randn(g, 2, Hk, D)).exp()
    d = {"start": start, "q": (1.5 * _randn(g, B, T, c["Hq"], D)).bfloat16()}
    for i, name in enumerate("kv"):
        d["hist_" + name] = (_randn(g, B, c["pos"], Hk, D) * spread[i]).bfloat16()
        d[name] = (_randn(g, B, T, Hk, D) * spread[i]).bfloat16()
    return d


def _pack4(w, group):
    """(bytes, scales) of a weight in 4 bits, as the module's head defines them."""
    N, K = w.shape
    G = -(-K // group)
    x = torch.zeros(N, G * group, device=w.device)
    x[:, :K] = w.float()
    x = x.view(N, G, group)
    m, e = torch.frexp(x.abs().amax(2) / 7)
    s = torch.ldexp((m * 32).round() / 32, e)  # five significant bits: m in [1/2, 1)
    q = torch.where(s[..., None] > 0, x / s[..., None], 0.0).round().clamp(-7, 7)
    u = (q + 8).to(torch.uint8).view(N, -1)[:, : K + K % 2].reshape(N, -1, 2)
    return u[..., 0] | (u[..., 1] << 4), s.bfloat16()


def _w4_inputs(c, seed):
    g = _gen(seed)
    n = 2 if c["fn"] == "gate_up" else 1
    d = {"x": _randn(g, c["M"], c["K"]).bfloat16(), "w": []}
    for _ in range(n):
        d["w"].append(_pack4(_randn(g, c["N"], c["K"], scale=0.02).bfloat16(), c["group"]))
    return d


def _logprob_inputs(c, seed):
    g = _gen(seed)
    M, V = c["M"], c["V"]
    x = _randn(g, M, V, scale=2.5)
    strong = torch.randint(0, V, (M, 4), generator=g, device=DEV)
    x.scatter_(1, strong, 9.0 + 3.0 * _randn(g, M, 4))
    rare = torch.randint(0, V, (M,), generator=g, device=DEV)
    pick = torch.rand(M, generator=g, device=DEV) < 0.7
    return {"logits": x.to(getattr(torch, c["dtype"])), "tokens": torch.where(pick, strong[:, 0], rare)}


_INPUTS = {"kv8": _kv8_inputs, "w4": _w4_inputs, "logprob": _logprob_inputs}


def prepare(c, seed):
    d = dict(_INPUTS[c["op"]](c, seed), c=c)
    if c["op"] == "kv8":
        # the cache as the steps before this one left it
        k, v, start = d.pop("hist_k"), d.pop("hist_v"), d["start"]
        if own:
            from llms_amd import kernels as fk

            d["cache"] = fk.KVCache8.alloc(1, c["pos"] + c["T"], max_batch=c["B"],
                                           n_kv_heads=c["Hk"], head_dim=c["D"], device=DEV)
            if c["pos"]:
                d["cache"].write(0, k, v, 0, lengths=start)
            d["at"] = start if c["ragged"] else c["pos"]
        else:
            d["old"] = [_plain_cache(t, start) for t in (k, v)]
    return d


# ------------------------------------------------------------ plain forms


def _codes(x):
    """Values of whole blocks [..., 64, D] as 8 bits hold them: (codes, scales)."""
    top = x.abs().amax((-2, -1))[..., None, None]
    # 127 x is exact and so is its quotient at a tie: every tie is seen as one
    return torch.where(top > 0, 127 * x / top, 0.0).round(), (top / 127)[..., 0, 0]


def _plain_cache(hist, start):
    """[B, P, H, D] tokens as a cache: codes and scales of the whole blocks, and
    the block that position ``start`` falls in, unpacked."""
    B, P, H, D = hist.shape
    nb = P // BLOCK
    x = hist[:, : nb * BLOCK].float().view(B, nb, BLOCK, H, D).permute(0, 3, 1, 2, 4)
    q, s = _codes(x)
    row = (start // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device=DEV)
    tail = hist[torch.arange(B, device=DEV)[:, None], row.clamp(max=max(P - 1, 0))] if P else \
        hist.new_zeros(B, BLOCK, H, D)
    return q.to(torch.int8), s, tail.transpose(1, 2).contiguous()


def _plain_kv8(d):
    c, start = d["c"], d["start"]
    B, T, Hk, D = c["B"], c["T"], c["Hk"], c["D"]
    off = start % BLOCK                      # new tokens before row `off` of their block
    R = -(-(BLOCK - 1 + T) // BLOCK) * BLOCK
    row = torch.arange(R, device=DEV)
    at = off[:, None] + torch.arange(T, device=DEV)
    both, new = [], []
    for (q, s, tail), x in zip(d["old"], (d["k"], d["v"])):
        old = (q.float() * s[..., None, None]).view(B, Hk, -1, D)
        buf = torch.zeros(B, Hk, R, D, device=DEV)
        buf[:, :, :BLOCK] = tail.float()
        idx = at[:, None, :, None].expand(B, Hk, T, D)
        buf = buf.scatter(2, idx, x.float().transpose(1, 2))
        nq, ns = _codes(buf.view(B, Hk, -1, BLOCK, D))
        packed = (nq * ns[..., None, None]).view(B, Hk, R, D)
        whole = row[None] < ((off + T) // BLOCK * BLOCK)[:, None]
        buf = torch.where(whole[:, None, :, None], packed, buf)
        both.append(torch.cat([old, buf], 2))
        new.append(buf.gather(2, idx).transpose(1, 2))
    k, v = both
    base = start - off
    n_old = k.shape[2] - R
    qpos = start[:, None] + torch.arange(T, device=DEV)
    old_pos = torch.arange(n_old, device=DEV)[None].expand(B, -1)
    far = torch.iinfo(torch.long).max
    kpos = torch.cat([torch.where(old_pos < base[:, None], old_pos, far), base[:, None] + row], 1)
    G = c["Hq"] // Hk
    q = d["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    x = x.view(B, Hk, G, T, -1).masked_fill(kpos[:, None, None, None] > qpos[:, None, None, :, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(B, Hk, G * T, -1)
    y = torch.matmul(p, v).view(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, c["Hq"], D)
    return {"y": y.bfloat16(), "k": new[0], "v": new[1]}


def _unpack4(qs, K, group):
    q, s = qs
    u = torch.stack([q & 15, q >> 4], 2).view(q.shape[0], -1)[:, :K].float() - 8
    return u * s.float().repeat_interleave(group, 1)[:, :K]


def _heads(c):
    """Rows of a QKV weight that are queries, keys and values."""
    n_k = c["N"] // 4
    return [c["N"] - 2 * n_k, n_k, n_k]


def _plain_w4(d):
    c = d["c"]
    x = d["x"].float()
    y = [x @ _unpack4(w, c["K"], c["group"]).T for w in d["w"]]
    if c["fn"] == "gate_up":
        return (y[0] / (1 + (-y[0]).exp()) * y[1]).bfloat16()
    return y[0].bfloat16().split(_heads(c), 1) if c["fn"] == "qkv" else y[0].bfloat16()


def _plain_logprob(d):
    c = d["c"]
    x = d["logits"].float()
    z = x - x.amax(1, keepdim=True)
    e = z.exp()
    l = e.sum(1)
    lse = l.log()
    out = {"logprob": z.gather(1, d["tokens"][:, None])[:, 0] - lse, "entropy": lse - (z * e).sum(1) / l}
    # by value, ties to the lowest token: an order-preserving whole number, then the token
    b = x.view(torch.int32).long()
    key = torch.where(b < 0, -(b & 0x7FFFFFFF), b) * (1 << 20) + ((1 << 20) - 1 - torch.arange(c["V"], device=DEV))
    ids = (1 << 20) - 1 - key.topk(min(c["k"], c["V"]), 1).values % (1 << 20)
    out["top_ids"] = ids
    out["top_logprobs"] = z.gather(1, ids) - lse[:, None]
    return out


_PLAIN = {"kv8": _plain_kv8, "w4": _plain_w4, "logprob": _plain_logprob}


# ---------------------------------------------------- the framework's calls


def _own_kv8(d):
    from llms_amd import kernels as fk

    y = fk.attention_kv8(d["q"], d["k"], d["v"], d["cache"], 0, d["at"])
    k, v = d["cache"].read(0, d["at"], d["c"]["T"])
    return {"y": y, "k": k, "v": v}


def _own_w4(d):
    from llms_amd import kernels as fk

    c, w = d["c"], d["w"]
    if c["fn"] == "gate_up":
        return fk.fused_gate_up_silu_w4(d["x"], *w[0], *w[1], group=c["group"])
    if c["fn"] == "qkv":
        n_q, n_k, _ = _heads(c)
        return fk.fused_qkv_w4(d["x"], *w[0], n_q=n_q, n_k=n_k, group=c["group"])
    return fk.fused_linear_w4(d["x"], *w[0], group=c["group"])


def _own_logprob(d):
    from llms_amd import kernels as fk

    return fk.token_logprobs(d["logits"], d["tokens"], top_k=d["c"]["k"])._asdict()


_OWN = {"kv8": _own_kv8, "w4": _own_w4, "logprob": _own_logprob}


def run(d):
    return (_OWN if own else _PLAIN)[d["c"]["op"]](d)


# ------------------------------------------------------------------- work


def work(c):
    if c["op"] == "kv8":
        B, T, Hq, Hk, D = (c[i] for i in ("B", "T", "Hq", "Hk", "D"))
        pos = (c["pos"] * (1 + 0.75 * (B - 1)) if c["ragged"] else c["pos"] * B)  # all sequences
        cache = 2 * pos * Hk * D + 8 * pos / BLOCK * Hk
        # q, y, the new keys and values: in, into the cache and read back as 32 bits
        io = B * T * D * (4 * Hq + 2 * Hk * (2 + 2 + 4))
        return {"bytes": cache + io, "flops": 4.0 * Hq * D * (T * pos + B * T * (T + 1) / 2)}
    if c["op"] == "w4":
        n = (2 if c["fn"] == "gate_up" else 1) * c["N"]
        return {"bytes": n * (-(-c["K"] // 2) + 2 * -(-c["K"] // c["group"])) + 2 * c["M"] * (c["K"] + c["N"]),
                "flops": 2.0 * c["M"] * n * c["K"]}
    size = 4 if c["dtype"] == "float32" else 2
    return {"bytes": c["M"] * (c["V"] * size + 16 + 12 * c["k"]), "flops": 6.0 * c["M"] * c["V"]}


# ------------------------------------------------------------------ exact


def _exact_blocks(x, n):
    """Tokens [P, H, D] in 64 bits, the first n (whole blocks) as 8 bits hold them."""
    out = x.double().clone()
    w = out[:n].reshape(-1, BLOCK, *x.shape[1:])
    top = w.abs().amax((1, 3), keepdim=True)
    out[:n] = (torch.round(w * 127 / top.clamp(min=1e-300)) * top / 127).reshape(n, *x.shape[1:])
    return out


def _exact_kv8(c, seed):
    d = _kv8_inputs(c, seed)
    T, Hk = c["T"], c["Hk"]
    ys, ks, vs = [], [], []
    for b, p in enumerate(d["start"].tolist()):
        end = p + T
        k, v = (_exact_blocks(torch.cat([d["hist_" + i][b, :p], d[i][b]]), end // BLOCK * BLOCK) for i in "kv")
        q = d["q"][b].double() / math.sqrt(c["D"])  # [T, Hq, D]
        hidden = torch.arange(end, device=DEV)[None] > torch.arange(p, end, device=DEV)[:, None]
        y = torch.empty_like(q)
        for h in range(c["Hq"]):
            i = h // (c["Hq"] // Hk)
            y[:, h] = (q[:, h] @ k[:, i].T).masked_fill(hidden, -math.inf).softmax(1) @ v[:, i]
        ys.append(y), ks.append(k[p:]), vs.append(v[p:])
    return {"y": torch.stack(ys), "k": torch.stack(ks), "v": torch.stack(vs)}


def _exact_w4(c, seed):
    d = _w4_inputs(c, seed)
    x = d["x"].double()
    y = []
    for q, s in d["w"]:
        w = torch.empty(c["N"], 2 * q.shape[1], dtype=torch.double, device=DEV)
        w[:, 0::2], w[:, 1::2] = (q % 16).double() - 8, (q // 16).double() - 8
        col = torch.arange(c["K"], device=DEV) // c["group"]
        y.append(x @ (w[:, : c["K"]] * s.double()[:, col]).T)
    if c["fn"] == "gate_up":
        return y[0] * torch.sigmoid(y[0]) * y[1]
    return y[0].split(_heads(c), 1) if c["fn"] == "qkv" else y[0]


def _exact_logprob(c, seed):
    d = _logprob_inputs(c, seed)
    rows = {"logprob": [], "entropy": [], "top_ids": [], "top_logprobs": []}
    for i in range(0, c["M"], 256):
        x = d["logits"][i : i + 256].double()
        lp = x.log_softmax(1)
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : c["k"]]
        rows["logprob"].append(lp.gather(1, d["tokens"][i : i + 256, None])[:, 0])
        rows["entropy"].append(-(lp.exp() * lp).sum(1))
        rows["top_ids"].append(ids)
        rows["top_logprobs"].append(lp.gather(1, ids))
    return {k: torch.cat(v) for k, v in rows.items()}


_EXACT = {"kv8": _exact_kv8, "w4": _exact_w4, "logprob": _exact_logprob}


def exact(c, seed):
    return _EXACT[c["op"]](c, seed)
