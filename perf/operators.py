"""Attention over a KV cache held in 4 bits: what a program serving a long-context or batched
Qwen3-Next / Qwen3.6 model calls for its full-attention blocks, between the projections.

Kinds of case (``case["kind"]``):

  append  new k, v rows normalised, rotated, quantised and written, then read back as values
  step    one token per sequence: its row appended, attention over the rows of its sequence,
          the output gate; with ``weights`` also the attention that each row has gathered
  prefill several tokens per sequence, causal after the rows that are there
  evict   the heaviest rows of a cache moved to a smaller one, then read as values

The cache holds per (sequence, kv head) `R` rows (a multiple of 32), all in one buffer:
  k codes  int32 [B, KVH, R, hd / 8]      word j of a row: dims 8 j .. 8 j + 7, lowest bits first
  v codes  int32 [B, KVH, R / 8, hd]      word d of a block: dim d of rows 8 i .. 8 i + 7
  params   f16   [B, KVH, 4, hd / 64, R]  k scale, k bias, v scale, v bias of each 64 dims
with value = scale * code + bias; scale = (max - min) / 15 and bias = min of the 64 values,
each rounded to f32 and then to f16, code = (value - bias) / scale rounded to the nearest.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e7
GROUP = 64

# query heads, kv heads, head size, rotated dims
HEADS = {"35b": (16, 2, 256, 64), "gqa128": (32, 8, 128, 128), "mha64": (8, 8, 64, 0)}


def listed():
    return [
        # a short chat, one conversation: latency
        {"name": "step-b1-500", "kind": "step", "heads": "35b", "sequences": 1, "rows": 500, "dtype": "f32", "weights": False},
        # a long document, one conversation, its cache about to be pruned
        {"name": "step-b1-33k-weights", "kind": "step", "heads": "35b", "sequences": 1, "rows": 33000, "dtype": "f32", "weights": True},
        # a batch of conversations of every length
        {"name": "step-b16-8k-ragged", "kind": "step", "heads": "35b", "sequences": 16, "rows": 8191, "dtype": "bf16", "weights": False},
        # a wide batch with more kv heads: the cache is what it reads
        {"name": "step-b32-16k", "kind": "step", "heads": "gqa128", "sequences": 32, "rows": 16384, "dtype": "bf16", "weights": False},
        # a short turn, its length as it comes, f32 activations
        {"name": "prefill-77", "kind": "prefill", "heads": "35b", "sequences": 1, "tokens": 77, "rows": 0, "dtype": "f32", "weights": False},
        # several prompts in one call, lengths as they come
        {"name": "prefill-b4-ragged", "kind": "prefill", "heads": "gqa128", "sequences": 4, "tokens": 1000, "rows": 129, "dtype": "bf16", "weights": False},
        # a chunk of a long prompt, gathering the weights to prune by
        {"name": "prefill-512-at-8k-weights", "kind": "prefill", "heads": "35b", "sequences": 1, "tokens": 512, "rows": 8192, "dtype": "bf16", "weights": True},
        # a long prompt in one call
        {"name": "prefill-4096", "kind": "prefill", "heads": "35b", "sequences": 1, "tokens": 4096, "rows": 0, "dtype": "bf16", "weights": False},
        # the rows of a decode batch, for a layer whose cache other layers read
        {"name": "append-b16", "kind": "append", "heads": "35b", "sequences": 16, "tokens": 1, "rows": 4097, "dtype": "f32"},
        # the rows of a long prompt
        {"name": "append-4096", "kind": "append", "heads": "gqa128", "sequences": 2, "tokens": 4096, "rows": 77, "dtype": "bf16"},
        # a long document's cache cut to an eighth
        {"name": "evict-b1-33k", "kind": "evict", "heads": "35b", "sequences": 1, "rows": 33000, "budget": 4096, "sink": 4, "recent": 512},
        # a batch's caches cut to a common size
        {"name": "evict-b8-8k", "kind": "evict", "heads": "gqa128", "sequences": 8, "rows": 8193, "budget": 2047, "sink": 4, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "step", "step", "prefill", "prefill", "evict"])
    heads = rng.choice(sorted(HEADS))
    _, kvh, hd, _ = HEADS[heads]
    B = _log(rng, 1, 32)
    # the rows of all sequences together, kv heads and dims included, stay within the largest listed step's
    most = 32 * 16384 * 8 * 128 // (B * kvh * hd)
    dtype = rng.choice(["bf16", "f32"])
    if kind == "step":
        return {"kind": kind, "heads": heads, "sequences": B, "rows": _log(rng, 1, min(most, 100000)), "dtype": dtype,
                "weights": rng.random() < 0.4}
    if kind == "evict":
        rows = _log(rng, 64, min(most // 4, 50000))
        sink, recent = rng.choice([0, 4, 5]), rng.choice([0, 1, 32, 100])
        budget = rng.randint(min(rows, sink + recent + 1), rows)
        return {"kind": kind, "heads": heads, "sequences": B, "rows": rows, "budget": max(budget, sink + recent), "sink": sink, "recent": recent}
    B = min(B, 8)
    if kind == "append":
        return {"kind": kind, "heads": heads, "sequences": B, "tokens": _log(rng, 1, 4096 // B), "rows": _log(rng, 1, 9000), "dtype": dtype}
    rows = rng.choice([0, 0, _log(rng, 1, 2500)])
    return {"kind": kind, "heads": heads, "sequences": B, "tokens": _log(rng, 2, 2048 // B), "rows": rows, "dtype": dtype,
            "weights": rng.random() < 0.3}


def _lengths(case):
    """Rows that each sequence has before the call, and the tokens that it brings."""
    B = case["sequences"]
    rows = [case["rows"] * (2 * b + 1) // (2 * B) if B > 1 else case["rows"] for b in range(B)]
    if B > 1:
        rows[-1] = case["rows"]
    kind = case["kind"]
    if kind == "evict":
        return rows, [0] * B
    tokens = case.get("tokens", 1)
    if kind == "prefill" and B > 1:
        return rows, [max(1, tokens * (B - b) // B) for b in range(B)]
    return rows, [tokens] * B


# ---------------------------------------------------------------------------
# inputs


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _round_up(n, m):
    return (n + m - 1) // m * m


def _pack(v):
    """Codes [..., 8] of 0 to 15 in int32 words, the first in the lowest bits."""
    shift = torch.arange(0, 32, 4, device=v.device, dtype=torch.int64)
    w = (v.long() << shift).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _make_cache(g, B, kvh, hd, R):
    """A cache of R rows a sequence in one buffer, and its three parts: quantised normal values,
    keys at the size that normalised ones have, values with a size of their own for each row."""
    ng = hd // GROUP
    sizes = [B * kvh * R * hd // 2, B * kvh * R * hd // 2, B * kvh * 4 * ng * R * 2]
    at = [0, _round_up(sizes[0], 256), _round_up(sizes[0], 256) + _round_up(sizes[1], 256)]
    buf = torch.zeros(at[2] + _round_up(sizes[2], 256), dtype=torch.uint8, device=DEV)
    kw = buf[:sizes[0]].view(torch.int32).view(B, kvh, R, hd // 8)
    vw = buf[at[1]:at[1] + sizes[1]].view(torch.int32).view(B, kvh, R // 8, hd)
    par = buf[at[2]:at[2] + sizes[2]].view(torch.float16).view(B, kvh, 4, ng, R)
    for b in range(B):
        for which in (0, 1):
            x = torch.randn((kvh, R, ng, GROUP), generator=g, device=DEV)
            if which:
                x *= 0.25 + torch.rand((kvh, R, 1, 1), generator=g, device=DEV)
            lo, hi = x.amin(-1), x.amax(-1)
            s, z = ((hi - lo) / 15).half(), lo.half()
            c = ((x - z.float()[..., None]) / s.float()[..., None]).round().clamp(0, 15).to(torch.int32).view(kvh, R, hd)
            par[b, :, 2 * which] = s.transpose(1, 2)
            par[b, :, 2 * which + 1] = z.transpose(1, 2)
            if which:
                vw[b] = _pack(c.view(kvh, R // 8, 8, hd).transpose(2, 3))
            else:
                kw[b] = _pack(c.view(kvh, R, hd // 8, 8))
    return buf, kw, vw, par


def _rope_table(n, rot):
    """cos and sin [n, rot / 2, 2] of the f32 angles position * theta^(-2 j / rot)."""
    j = torch.arange(rot // 2, dtype=torch.float64)
    freq = (THETA ** (-(2 * j).float() / max(rot, 1)).double()).float()
    ang = (torch.arange(n).float()[:, None] * freq[None, :]).double()
    return torch.stack([ang.cos(), ang.sin()], -1).float().to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    H, kvh, hd, rot = HEADS[case["heads"]]
    B = case["sequences"]
    rows, new = _lengths(case)
    top = max(r + t for r, t in zip(rows, new))
    R = _round_up(top, 32)
    s = {"case": case, "top": top, "R": R}
    s["buf"], s["kw"], s["vw"], s["par"] = _make_cache(g, B, kvh, hd, R)
    s["rows"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    kind = case["kind"]
    if kind != "evict":
        dt = _type(case["dtype"])
        N = sum(new)
        starts = [sum(new[:b]) for b in range(B + 1)]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["q_norm"] = 1 + 0.1 * torch.randn(hd, generator=g, device=DEV)
        s["k_norm"] = 1 + 0.1 * torch.randn(hd, generator=g, device=DEV)
        s["rope"] = _rope_table(top, rot)
        s["k"] = torch.randn((N, kvh * hd), generator=g, device=DEV).to(dt)
        s["v"] = torch.randn((N, kvh * hd), generator=g, device=DEV).to(dt)
        s["q"] = torch.randn((N, H * 2 * hd), generator=g, device=DEV).to(dt) if kind != "append" else None
        s["out"] = torch.empty((N, H * hd), dtype=dt, device=DEV)
        s["weights"] = torch.rand((B, kvh, R), generator=g, device=DEV) if case.get("weights") else None
        s["tokens"], s["most"] = N, max(new)
    else:
        # gathered weights have a long tail; rows that nothing has looked at are equal
        w = torch.exp(2 * torch.randn((B, kvh, R), generator=g, device=DEV) - 6)
        s["weights"] = torch.where(torch.rand((B, kvh, R), generator=g, device=DEV) < 0.05, 0.0, w)
    if own:
        from swiftlet_amd.attention_q4 import AttentionQ4GPU, Q4Cache
        ones = torch.ones(hd, device=DEV)
        blk = AttentionQ4GPU(H, kvh, hd, rot, THETA, EPS, R, s.get("q_norm", ones), s.get("k_norm", ones), rope_table=s.get("rope"))
        s["block"] = blk
        s["cache"] = Q4Cache(B, kvh, hd, R, data=s["buf"])
        if kind == "evict":
            s["small"] = blk.new_cache(B, case["budget"])
            s["small_weights"] = torch.empty((B, kvh, case["budget"]), device=DEV)
        elif kind != "append":
            s["ws"] = blk.new_workspace(s["cache"], tokens=s["tokens"], max_tokens=s["most"], weights=s["weights"] is not None)
    return s


# ---------------------------------------------------------------------------
# the plain form


def _values(words, scale, bias, which):
    """The values of one kind of a cache: f32 [B, KVH, R, hd]."""
    c = (words[..., None] >> torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)) & 15
    if which == "v":
        c = c.transpose(-1, -2)  # [B, KVH, R / 8, 8, hd]
    B, kvh, ng, R = scale.shape
    c = c.reshape(B, kvh, R, ng, GROUP).float()
    return (c * scale.float().transpose(2, 3)[..., None] + bias.float().transpose(2, 3)[..., None]).view(B, kvh, R, ng * GROUP)


def _norm_rope(x, w, table):
    """x [N, heads, hd] normalised, times w, its first dims turned by table [N, rot / 2, 2]."""
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    h = table.shape[1]
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def _held(x):
    """x [N, KVH, hd] in 64 bits as the cache holds it: f32 values of 4-bit codes."""
    y = x.clamp(-65504, 65504).view(*x.shape[:-1], -1, GROUP)
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    s, z = ((hi - lo) / 15).float().half().double(), lo.float().half().double()
    c = torch.where(s > 0, ((y - z) / s).round().clamp(0, 15), 0.0)
    return (c.float() * s.float() + z.float()).view(x.shape)


def _where(s):
    """Of each token: its sequence, its place among that one's new tokens, its row."""
    n = torch.arange(s["tokens"], device=DEV)
    seq = torch.bucketize(n, s["starts"][1:].long(), right=True)
    i = n - s["starts"].long()[seq]
    return seq, i, s["rows"].long()[seq] + i


def _new_rows(s, row):
    N, hd = s["tokens"], s["k_norm"].numel()
    k = _norm_rope(s["k"].view(N, -1, hd).double(), s["k_norm"].double(), s["rope"][row].double())
    return _held(k), _held(s["v"].view(N, -1, hd).double())


def _plain_attention(s):
    H, kvh, hd, rot = HEADS[s["case"]["heads"]]
    B, N, T, G = s["case"]["sequences"], s["tokens"], s["most"], H // kvh
    seq, i, row = _where(s)
    nk, nv = _new_rows(s, row)
    K = _values(s["kw"], s["par"][:, :, 0], s["par"][:, :, 1], "k")
    V = _values(s["vw"], s["par"][:, :, 2], s["par"][:, :, 3], "v")
    K[seq, :, row], V[seq, :, row] = nk, nv
    q, gate = s["q"].float().view(N, H, 2, hd).unbind(2)
    qp = torch.zeros((B, T, H, hd), device=DEV)
    qp[seq, i] = _norm_rope(q, s["q_norm"], s["rope"][row])
    qp = qp.view(B, T, kvh, G, hd).transpose(1, 2).reshape(B, kvh, T * G, hd)
    sc = torch.matmul(qp, K.transpose(2, 3)).mul_(1 / math.sqrt(hd)).view(B, kvh, T, G, -1)
    last = s["rows"].long()[:, None] + torch.arange(T, device=DEV)  # [B, T]
    see = torch.arange(s["R"], device=DEV) <= last[..., None]
    sc.masked_fill_(~see[:, None, :, None], -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, kvh, T * G, -1), V).view(B, kvh, T, G, hd).transpose(1, 2).reshape(B, T, H, hd)[seq, i]
    got = {"out": (o * torch.sigmoid(gate)).reshape(N, H * hd).to(s["out"].dtype), "k_rows": nk, "v_rows": nv}
    if s["weights"] is not None:
        count = s["starts"].long().diff()
        there = torch.arange(T, device=DEV) < count[:, None]
        add = (p * there[:, None, :, None, None]).sum((2, 3))
        at = torch.arange(s["R"], device=DEV)
        before, after = at < s["rows"].long()[:, None], at < (s["rows"].long() + count)[:, None]
        w = s["weights"]
        w.copy_(torch.where(before[:, None], w + add, torch.where(after[:, None], add, w)))
        got["weights"] = w
    return got


def _plain_evict(s):
    case = s["case"]
    budget, sink, recent = case["budget"], case["sink"], case["recent"]
    w, n, R = s["weights"], s["rows"].long()[:, None, None], s["R"]
    at = torch.arange(R, device=DEV)
    always = (at < sink) | (at >= n - recent)
    key = torch.where(at < n, torch.where(always, math.inf, w), -1.0)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.sort(torch.where(order < n, order, R), dim=-1).values
    kept = torch.where(order < R, order, -1)
    count = torch.clamp(s["rows"], max=budget)
    at = order.clamp(max=R - 1)
    there = (kept >= 0)[..., None]
    K = _values(s["kw"], s["par"][:, :, 0], s["par"][:, :, 1], "k")
    V = _values(s["vw"], s["par"][:, :, 2], s["par"][:, :, 3], "v")
    K, V = (torch.take_along_dim(x, at[..., None], 2).where(there, 0.0).transpose(1, 2).to(torch.bfloat16) for x in (K, V))
    return {"kept": kept.int(), "rows": count, "weights": torch.where(kept >= 0, torch.take_along_dim(w, at, -1), 0.0), "k": K, "v": V}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "evict":
            return _plain_evict(s)
        if kind == "append":
            B, N = case["sequences"], s["tokens"]
            k, v = _new_rows(s, _where(s)[2])
            return {"k": k.view(B, N // B, *k.shape[1:]), "v": v.view(B, N // B, *v.shape[1:])}
        return _plain_attention(s)
    blk, cache = s["block"], s["cache"]
    if kind == "evict":
        kept, rows = blk.evict(cache, s["weights"], s["rows"], s["small"], case["budget"], sink=case["sink"], recent=case["recent"],
                               new_weights=s["small_weights"])
        k, v = s["small"].read(None, case["budget"], dtype=torch.bfloat16, rows=rows)
        return {"kept": kept, "rows": rows, "weights": s["small_weights"], "k": k, "v": v}
    if kind == "append":
        blk.append(s["k"], s["v"], cache, s["rows"], starts=s["starts"], max_tokens=s["most"])
        k, v = cache.read(s["rows"], s["most"])
        return {"k": k, "v": v}
    if kind == "step":
        blk.step(s["q"], s["k"], s["v"], cache, s["rows"], s["ws"], out=s["out"], weights=s["weights"])
        k, v = cache.read(s["rows"], 1)
    else:
        blk.prefill(s["q"], s["k"], s["v"], cache, s["rows"], s["ws"], starts=s["starts"], max_tokens=s["most"], out=s["out"],
                    weights=s["weights"])
        k, v = cache.read(s["rows"], s["most"], starts=s["starts"], tokens=s["tokens"])
    got = {"out": s["out"], "k_rows": k.view(s["tokens"], *k.shape[-2:]), "v_rows": v.view(s["tokens"], *v.shape[-2:])}
    if s["weights"] is not None:
        got["weights"] = s["weights"]
    return got


# ---------------------------------------------------------------------------
# the least that a pass has to read, write and compute


def work(case):
    H, kvh, hd, rot = HEADS[case["heads"]]
    rows, new = _lengths(case)
    row = kvh * (hd + 8 * hd // GROUP)  # bytes of one cached row, k and v
    if case["kind"] == "evict":
        kept = sum(min(r, case["budget"]) for r in rows)
        values = 2 * len(rows) * case["budget"] * kvh * hd * 2
        return {"bytes": sum(rows) * kvh * 4 + kept * (2 * row + 8 * kvh) + values, "flops": sum(rows) * kvh}
    size = 4 if case["dtype"] == "f32" else 2
    N = sum(new)
    given = N * 2 * kvh * hd * size + N * rot * 4
    shown = N * 2 * kvh * hd * 4
    if case["kind"] == "append":
        return {"bytes": given + N * row + shown, "flops": 20 * N * kvh * hd}
    pairs = sum(t * r + t * (t + 1) // 2 for r, t in zip(rows, new))
    total = {"bytes": sum(rows) * row + given + N * row + shown + N * H * hd * 3 * size, "flops": 4 * hd * H * pairs}
    if case["weights"]:
        total["bytes"] += (2 * sum(rows) + N) * kvh * 4
    return total


# ---------------------------------------------------------------------------
# the definition in 64 bits, a head at a time


def _nibbles(words, count):
    return torch.stack([torch.bitwise_and(torch.bitwise_right_shift(words, 4 * i), 15) for i in range(count)], -1)


def _head_values(s, b, h, n):
    """k and v, f64 [n, hd], of one sequence's kv head."""
    par = s["par"][b, h].double().repeat_interleave(GROUP, dim=1)  # [4, hd, R]
    kc = _nibbles(s["kw"][b, h], 8).flatten(1)[:n].double()
    vc = _nibbles(s["vw"][b, h], 8).permute(0, 2, 1).flatten(0, 1)[:n].double()
    return kc * par[0].T[:n] + par[1].T[:n], vc * par[2].T[:n] + par[3].T[:n]


def _turned(x, w, table):
    """One head's rows [T, hd] in 64 bits."""
    y = w.double() * x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPS)
    half = table.shape[1]
    z = torch.view_as_complex(torch.stack([y[:, :half], y[:, half:2 * half]], -1).contiguous()) * torch.view_as_complex(table.double().contiguous())
    return torch.cat([z.real, z.imag, y[:, 2 * half:]], 1)


def _stored(x):
    """Rows [T, hd] as the cache holds them."""
    parts = []
    for p in x.clamp(-65504.0, 65504.0).split(GROUP, 1):
        low = p.min(1, keepdim=True).values
        step = ((p.max(1, keepdim=True).values - low) / 15).float().half().double()
        low = low.float().half().double()
        code = torch.nan_to_num((p - low) / step, nan=0.0).round().clamp(0, 15) * (step > 0)
        parts.append(low + step * code)
    return torch.cat(parts, 1)


def exact(case, seed):
    s = prepare(case, seed)
    H, kvh, hd, _ = HEADS[case["heads"]]
    rows, new = _lengths(case)
    B = len(rows)
    if case["kind"] == "evict":
        budget, sink, recent, R = case["budget"], case["sink"], case["recent"], s["R"]
        kept = torch.full((B, kvh, budget), -1, dtype=torch.int32, device=DEV)
        w = torch.zeros((B, kvh, budget), dtype=torch.float64, device=DEV)
        K, V = (torch.zeros((B, budget, kvh, hd), dtype=torch.float64, device=DEV) for _ in range(2))
        for b, n in enumerate(rows):
            for h in range(kvh):
                keep = torch.ones(n, dtype=torch.bool, device=DEV)
                if n > budget:
                    mid = s["weights"][b, h, sink:n - recent].double()
                    drop = torch.argsort(-mid, stable=True)[budget - sink - recent:] + sink
                    keep[drop] = False
                at = keep.nonzero().flatten()
                k, v = _head_values(s, b, h, n)
                kept[b, h, :at.numel()] = at.int()
                w[b, h, :at.numel()] = s["weights"][b, h, at].double()
                K[b, :at.numel(), h], V[b, :at.numel(), h] = k[at], v[at]
        return {"kept": kept, "rows": torch.tensor([min(n, budget) for n in rows], dtype=torch.int32, device=DEV), "weights": w, "k": K, "v": V}
    N = s["tokens"]
    k_in, v_in = (s[x].double().view(N, kvh, hd) for x in ("k", "v"))
    nk, nv = torch.empty_like(k_in), torch.empty_like(v_in)
    out = torch.empty((N, H, hd), dtype=torch.float64, device=DEV)
    w = s["weights"].double() if s["weights"] is not None else None
    t0 = 0
    for b, (n, t) in enumerate(zip(rows, new)):
        table = s["rope"][n:n + t]
        mask = torch.ones((t, n + t), dtype=torch.bool, device=DEV).tril(n)
        for h in range(kvh):
            nk[t0:t0 + t, h] = _stored(_turned(k_in[t0:t0 + t, h], s["k_norm"], table))
            nv[t0:t0 + t, h] = _stored(v_in[t0:t0 + t, h])
            if case["kind"] == "append":
                continue
            k, v = _head_values(s, b, h, n + t)
            k[n:], v[n:] = nk[t0:t0 + t, h], nv[t0:t0 + t, h]
            gathered = torch.zeros(n + t, dtype=torch.float64, device=DEV)
            for j in range(h * H // kvh, (h + 1) * H // kvh):
                q = s["q"][t0:t0 + t].double().view(t, H, 2, hd)[:, j]
                score = (_turned(q[:, 0], s["q_norm"], table) @ k.T) / hd ** 0.5
                p = torch.softmax(torch.where(mask, score, -math.inf), 1)
                out[t0:t0 + t, j] = (p @ v) / (1 + torch.exp(-q[:, 1]))
                gathered += p.sum(0)
            if w is not None:
                w[b, h, :n] += gathered[:n]
                w[b, h, n:n + t] = gathered[n:]
        t0 += t
    if case["kind"] == "append":
        return {"k": nk.view(B, N // B, kvh, hd), "v": nv.view(B, N // B, kvh, hd)}
    got = {"out": out.view(N, H * hd), "k_rows": nk, "v_rows": nv}
    if w is not None:
        got["weights"] = w
    return got
