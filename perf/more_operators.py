"""What a program that serves a hybrid Qwen3-Next / Qwen3.6 model calls for the tokens of many
sequences between the projections of its blocks: the gated DeltaNet block over prompts and over one
token of each conversation, and the rotary positions of the attention blocks' queries and keys.

Kinds of case (``case["kind"]``):

  delta   tokens of `sequences` sequences through a DeltaNet block between its input projections and
          out_proj: causal convolution and SiLU, query and key norms, gates, the gated delta rule and
          the gated norm, from each sequence's state and into it.  ``lengths``: "even" (`tokens` each),
          "ragged" (from `tokens` down to a fraction of it), "mixed" (one token each, and one
          sequence that brings `tokens`)
  rope    queries and keys turned by their positions, normalised before where the block does so
  table   cos and sin of positions, scaled for long contexts

A sequence's state lies in a slot of a buffer: the last K mixed rows as a ring [K, 2 nk dk + nv dv]
(the row of position p in place p % K), at the next 256-byte boundary the matrices [nv, dv, dk], f32.
Sequences take slots in any order; slots that no sequence takes stay as they are.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
KERNEL = 4
CHUNK = 64

# DeltaNet blocks: key heads, value heads, key and value head size
BLOCKS = {"35b": (16, 32, 128, 128), "quarter": (4, 8, 128, 128), "small": (4, 8, 64, 64), "wide": (2, 8, 128, 64)}
# attention blocks: query heads, kv heads, head size, rotated dims, whether queries lie beside output gates and are normalised
HEADS = {"35b": (16, 2, 256, 64, True), "gqa128": (32, 8, 128, 128, False), "mha64": (8, 8, 64, 32, False)}
THETA = 1e7
SCALINGS = {"none": None, "linear4": ("linear", 4.0, 32768), "ntk8": ("ntk", 8.0, 32768), "yarn4": ("yarn", 4.0, 262144)}


def listed():
    return [
        # one conversation, its next token: latency
        {"name": "delta-b1-step", "kind": "delta", "block": "35b", "sequences": 1, "tokens": 1, "lengths": "even", "layout": "interleaved", "dtype": "f32"},
        # a wide batch of conversations, one token each: the states are what it reads and writes
        {"name": "delta-b64-step", "kind": "delta", "block": "35b", "sequences": 64, "tokens": 1, "lengths": "even", "layout": "interleaved", "dtype": "bf16"},
        # a short turn, its length as it comes, f32 activations
        {"name": "delta-77", "kind": "delta", "block": "35b", "sequences": 1, "tokens": 77, "lengths": "even", "layout": "interleaved", "dtype": "f32"},
        # several prompts in one call, lengths as they come
        {"name": "delta-b4-ragged", "kind": "delta", "block": "35b", "sequences": 4, "tokens": 1000, "lengths": "ragged", "layout": "split", "dtype": "bf16"},
        # conversations that go on while a prompt comes in
        {"name": "delta-b32-mixed", "kind": "delta", "block": "35b", "sequences": 32, "tokens": 600, "lengths": "mixed", "layout": "interleaved", "dtype": "bf16"},
        # a long prompt in one call
        {"name": "delta-4096", "kind": "delta", "block": "35b", "sequences": 1, "tokens": 4096, "lengths": "even", "layout": "interleaved", "dtype": "bf16"},
        # a long document
        {"name": "delta-16384", "kind": "delta", "block": "35b", "sequences": 1, "tokens": 16384, "lengths": "even", "layout": "split", "dtype": "bf16"},
        # queries and keys of one token, f32 activations: latency
        {"name": "rope-1", "kind": "rope", "heads": "35b", "tokens": 1, "layout": "half", "dtype": "f32", "rows": True, "inverse": False},
        # a batch of short turns, whole heads turned in pairs of neighbours
        {"name": "rope-333-pairs", "kind": "rope", "heads": "gqa128", "tokens": 333, "layout": "interleaved", "dtype": "bf16", "rows": True, "inverse": False},
        # a long document's queries and keys
        {"name": "rope-16384", "kind": "rope", "heads": "35b", "tokens": 16384, "layout": "half", "dtype": "bf16", "rows": False, "inverse": False},
        # the positions of a decode batch, anywhere in a long context
        {"name": "table-64", "kind": "table", "heads": "35b", "positions": 64, "scaling": "yarn4", "given": True},
        # every position of a context, once per model
        {"name": "table-262144", "kind": "table", "heads": "35b", "positions": 262144, "scaling": "yarn4", "given": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "delta", "rope", "rope", "table"])
    if kind == "table":
        return {"kind": kind, "heads": rng.choice(sorted(HEADS)), "positions": _log(rng, 1, 200000), "scaling": rng.choice(sorted(SCALINGS)),
                "given": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "rope":
        heads = rng.choice(sorted(HEADS))
        return {"kind": kind, "heads": heads, "tokens": _log(rng, 1, 12000), "layout": rng.choice(["half", "interleaved"]), "dtype": dtype,
                "rows": rng.random() < 0.5, "inverse": not HEADS[heads][4] and rng.random() < 0.3}
    case = {"kind": kind, "block": rng.choice(sorted(BLOCKS) + ["35b"]), "sequences": _log(rng, 1, 64), "tokens": 1,
            "lengths": rng.choice(["even", "ragged", "mixed"]), "layout": rng.choice(["interleaved", "split"]), "dtype": dtype}
    case["tokens"] = rng.choice([1, _log(rng, 1, 16), _log(rng, 8, 12000), _log(rng, 64, 12000)])
    case["tokens"] = max(1, min(case["tokens"], 12000 // case["sequences"]))
    return case


def _lengths(case):
    """Tokens that each sequence brings."""
    B, T = case["sequences"], case["tokens"]
    if case["lengths"] == "even":
        return [T] * B
    if case["lengths"] == "mixed":
        return [1] * (B - 1) + [T]
    return [max(1, T * (B - b) // B) for b in range(B)]


# ---------------------------------------------------------------------------
# inputs


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _ramped(rot, scaling):
    """The angle per position of each turned pair, f64, and what cos and sin are multiplied by."""
    two_j = torch.arange(0, rot, 2, dtype=torch.float64)
    if scaling is None:
        return THETA ** (-two_j / rot), 1.0
    how, factor, original = scaling
    if how == "linear":
        return THETA ** (-two_j / rot) / factor, 1.0
    if how == "ntk":
        return (THETA * factor ** (rot / (rot - 2))) ** (-two_j / rot), 1.0
    place = [rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(THETA)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), rot - 1)
    ramp = ((two_j / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    freq = THETA ** (-two_j / rot)
    return (1 - ramp) * freq + ramp * freq / factor, 1.0 + 0.1 * math.log(factor)


def _cos_sin(position, scaling, rot):
    """[n, rot / 2, 2] f32 of 64-bit angles."""
    freq, size = _ramped(rot, scaling)
    angle = position.double()[:, None] * freq.to(position.device)
    return torch.stack([angle.cos() * size, angle.sin() * size], -1).float()


def _slot_sizes(block):
    nk, nv, dk, dv = BLOCKS[block]
    conv = 2 * nk * dk + nv * dv
    at = (KERNEL * conv * 4 + 255) // 256 * 256
    return conv, at, (at + nv * dv * dk * 4 + 255) // 256 * 256


def _prepare_delta(case, g, s):
    nk, nv, dk, dv = BLOCKS[case["block"]]
    conv, at, size = _slot_sizes(case["block"])
    B, new, dt = case["sequences"], _lengths(case), _type(case["dtype"])
    N, slots = sum(new), case["sequences"] + 1

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s["states"] = torch.zeros(slots * size, dtype=torch.uint8, device=DEV)
    whole = s["states"].view(slots, size)
    s["ring"] = whole[:, :KERNEL * conv * 4].view(torch.float32).view(slots, KERNEL, conv)
    s["rec"] = whole[:, at:at + nv * dv * dk * 4].view(torch.float32).view(slots, nv, dv, dk)
    s["ring"].copy_(normal(slots, KERNEL, conv))
    s["rec"].copy_(normal(slots, nv, dv, dk) * 0.2)
    s["slots"] = torch.randperm(slots, generator=g, device=DEV)[:B].int()
    s["positions"] = torch.randint(0, 100000, (B,), generator=g, device=DEV, dtype=torch.int32)
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    s["tokens"], s["most"] = N, max(new)
    s["qkvz"] = normal(N, conv + nv * dv).to(dt)
    s["ba"] = normal(N, 2 * nv).to(dt)
    s["conv_w"] = normal(conv, KERNEL) * 0.4
    # decays as such models start out with them: rates of 1 to 16, steps of 0.001 to 0.1
    s["a_log"] = (1 + 15 * torch.rand(nv, generator=g, device=DEV)).log()
    step = torch.exp(torch.rand(nv, generator=g, device=DEV) * math.log(100) + math.log(0.001))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["norm_w"] = 1 + 0.1 * normal(dv)
    s["out"] = torch.empty((N, nv * dv), dtype=dt, device=DEV)
    if own:
        from swiftlet_amd._lib import SWQ_DELTA_INTERLEAVED, SWQ_DELTA_SPLIT
        from swiftlet_amd.deltanet import DeltaNetGPU
        s["own"] = DeltaNetGPU(nk, nv, dk, dv, KERNEL, SWQ_DELTA_SPLIT if case["layout"] == "split" else SWQ_DELTA_INTERLEAVED, EPS,
                               s["conv_w"], s["a_log"], s["dt_bias"], s["norm_w"])
        s["ws"] = s["own"].new_batch_workspace(B, N, s["most"])


def _prepare_rope(case, g, s):
    H, kvh, hd, rot, gated = HEADS[case["heads"]]
    N, dt = case["tokens"], _type(case["dtype"])
    s["q_proj"] = torch.randn((N, H, 2 * hd if gated else hd), generator=g, device=DEV).to(dt)
    s["q"] = s["q_proj"][..., :hd]
    s["k"] = torch.randn((N, kvh, hd), generator=g, device=DEV).to(dt)
    s["norms"] = [1 + 0.1 * torch.randn(hd, generator=g, device=DEV) for _ in range(2)] if gated else None
    s["rows"] = torch.randint(0, 40000, (N,), generator=g, device=DEV, dtype=torch.int32) if case["rows"] else None
    place = torch.arange(40000 if case["rows"] else N, device=DEV) + (0 if case["rows"] else 5000)
    s["table"] = _cos_sin(place, SCALINGS["yarn4"], rot)
    s["outs"] = [torch.empty((N, h, hd), dtype=dt, device=DEV) for h in (H, kvh)]
    if own:
        from swiftlet_amd.rope import RopeGPU
        s["own"] = RopeGPU(rot, THETA, layout=case["layout"])


def _prepare_table(case, g, s):
    rot, n = HEADS[case["heads"]][3], case["positions"]
    s["given"] = torch.randint(0, 1000000, (n,), generator=g, device=DEV, dtype=torch.int32) if case["given"] else None
    s["first"] = 0 if case["given"] else int(torch.randint(0, 700000, (1,), generator=g, device=DEV))
    s["table"] = torch.empty((n, rot // 2, 2), device=DEV)
    if own:
        from swiftlet_amd.rope import RopeGPU, RopeScaling
        sc = SCALINGS[case["scaling"]]
        s["own"] = RopeGPU(rot, THETA, scaling=None if sc is None else RopeScaling(sc[0], sc[1], sc[2]))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    {"delta": _prepare_delta, "rope": _prepare_rope, "table": _prepare_table}[case["kind"]](case, g, s)
    return s


# ---------------------------------------------------------------------------
# the plain form


def _parts(s):
    """mixed [N, conv], z [N, nv, dv], b and a [N, nv] of the projections, f32."""
    case = s["case"]
    nk, nv, dk, dv = BLOCKS[case["block"]]
    x, ba = s["qkvz"].float(), s["ba"].float()
    N, rep = x.shape[0], nv // nk
    if case["layout"] == "split":
        conv = 2 * nk * dk + nv * dv
        return x[:, :conv], x[:, conv:].view(N, nv, dv), ba[:, :nv], ba[:, nv:]
    q, k, v, z = x.view(N, nk, -1).split([dk, dk, rep * dv, rep * dv], -1)
    b, a = ba.view(N, nk, 2, rep).unbind(2)
    return torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1), z.reshape(N, nv, dv), b.reshape(N, nv), a.reshape(N, nv)


def _plain_chunks(q, k, v, log_g, beta, S):
    """The delta rule a chunk of C tokens at a time: q, k, v [B, h, chunks, C, d] and gates [.., 1], S [B, h, dk, dv]."""
    C = q.shape[3]
    c = log_g.double().cumsum(3)
    fade = torch.where(torch.ones(C, C, device=q.device).tril().bool(), (c - c.transpose(3, 4)).exp(), 0.0).float()
    grown = c.exp().float()
    # what a chunk's rows take from each other: (1 + A)^-1, row by row
    A = (torch.matmul(k, k.transpose(3, 4).contiguous()) * fade * beta).tril(-1)
    W = torch.eye(C, device=q.device).expand_as(A).clone()
    for r in range(1, C):
        W[..., r, :r] = -(A[..., r, :r, None] * W[..., :r, :r]).sum(-2)
    U, W = torch.matmul(W, beta * v), torch.matmul(W, beta * grown * k)
    inner = torch.matmul(q, k.transpose(3, 4).contiguous()) * fade
    late = (c[:, :, :, -1:] - c).exp().float()
    o = torch.empty_like(v)
    for m in range(q.shape[2]):
        d = U[:, :, m] - torch.matmul(W[:, :, m], S)
        o[:, :, m] = torch.matmul(grown[:, :, m] * q[:, :, m], S) + torch.matmul(inner[:, :, m], d)
        S = grown[:, :, m, -1:] * S + torch.matmul(k[:, :, m].transpose(2, 3).contiguous(), late[:, :, m] * d)
    return o, S


def _plain_delta(s):
    case = s["case"]
    nk, nv, dk, dv = BLOCKS[case["block"]]
    B, N, T = case["sequences"], s["tokens"], s["most"]
    mixed, z, b, a = _parts(s)
    n = torch.arange(N, device=DEV)
    seq = torch.bucketize(n, s["starts"][1:].long(), right=True)
    i = n - s["starts"].long()[seq]
    slot, pos, count = s["slots"].long(), s["positions"].long(), s["starts"].long().diff()

    # the convolution over the kept rows and the new ones
    back = torch.arange(1 - KERNEL, 0, device=DEV)
    ring = s["ring"]
    row = torch.zeros((B, KERNEL - 1 + T, mixed.shape[1]), device=DEV)
    row[:, :KERNEL - 1] = ring[slot[:, None], (pos[:, None] + back) % KERNEL]
    row[seq, KERNEL - 1 + i] = mixed
    x = sum(s["conv_w"][:, j] * row[:, j:j + T] for j in range(KERNEL))
    x = x * torch.sigmoid(x)
    last = i >= count[seq] - KERNEL
    ring[slot[seq[last]], (pos[seq] + i)[last] % KERNEL] = mixed[last]

    # queries, keys, values, gates; nothing where a sequence has no token
    C = min(CHUNK, T)
    P = (T + C - 1) // C * C
    there = (torch.arange(T, device=DEV) < count[:, None])[..., None]
    q, k, v = x.split([nk * dk, nk * dk, nv * dv], -1)
    unit = lambda y: y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(dk)  # noqa: E731
    gates = torch.zeros((2, B, T, nv), device=DEV)
    gates[0, seq, i] = -torch.exp(s["a_log"]) * torch.nn.functional.softplus(a + s["dt_bias"])
    gates[1, seq, i] = torch.sigmoid(b)

    def heads(y, d):  # [B, T, h * d] -> [B, nv, P / C, C, d]
        y = torch.nn.functional.pad(y * there, (0, 0, 0, P - T)).view(B, P // C, C, -1, d)
        return y.repeat_interleave(nv // y.shape[3], 3).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v = heads(unit(q.unflatten(-1, (nk, dk))).flatten(2), dk) / math.sqrt(dk), heads(unit(k.unflatten(-1, (nk, dk))).flatten(2), dk), heads(v, dv)
    log_g, beta = heads(gates[0], 1), heads(gates[1], 1)
    S = s["rec"][slot].transpose(2, 3).contiguous()
    if T == 1:
        turn = lambda y: y[:, :, 0].transpose(2, 3)  # noqa: E731  [B, nv, d, 1]
        S = S * turn(log_g).exp()
        S = S + turn(k) * (turn(beta) * (v[:, :, 0] - (S * turn(k)).sum(2, keepdim=True)))
        o = (S * turn(q)).sum(2)[:, :, None, None]
    else:
        o, S = _plain_chunks(q, k, v, log_g, beta, S)
    s["rec"][slot] = S.transpose(2, 3)
    o = o.flatten(2, 3).transpose(1, 2)[seq, i]
    o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"] * (z * torch.sigmoid(z))
    return {"out": o.flatten(1).to(s["out"].dtype), "ring": ring, "states": s["rec"]}


def _plain_rope(s):
    case = s["case"]
    rot = HEADS[case["heads"]][3]
    table = s["table"] if s["rows"] is None else s["table"][s["rows"].long()]
    c, sn = table[:, None, :, 0], table[:, None, :, 1]
    if case["inverse"]:
        sn = -sn
    outs = []
    for n, x in enumerate((s["q"], s["k"])):
        y = x.float()
        if s["norms"] is not None:
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norms"][n]
        y, rest = y[..., :rot], y[..., rot:]
        if case["layout"] == "half":
            a, b = y.chunk(2, -1)
            y = torch.cat([a * c - b * sn, b * c + a * sn], -1)
        else:
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
        outs.append(torch.cat([y, rest], -1).to(x.dtype))
    return {"q": outs[0], "k": outs[1]}


def run(s):
    case = s["case"]
    if case["kind"] == "table":
        if own:
            return s["own"].table(s["given"], first=s["first"], count=case["positions"], out=s["table"])
        place = s["given"] if s["given"] is not None else s["first"] + torch.arange(case["positions"], device=DEV)
        return _cos_sin(place, SCALINGS[case["scaling"]], HEADS[case["heads"]][3])
    if case["kind"] == "rope":
        if not own:
            return _plain_rope(s)
        q, k = s["own"].apply([s["q"], s["k"]], s["table"], rows=s["rows"], norm_weights=s["norms"], eps=EPS, inverse=case["inverse"], out=s["outs"])
        return {"q": q, "k": k}
    if not own:
        return _plain_delta(s)
    if s["most"] == 1:
        s["own"].step_batch(s["qkvz"], s["ba"], s["states"], s["positions"], s["ws"], slots=s["slots"], out=s["out"])
    else:
        s["own"].prefill(s["qkvz"], s["ba"], s["states"], s["positions"], s["ws"], starts=s["starts"], slots=s["slots"], max_tokens=s["most"], out=s["out"])
    return {"out": s["out"], "ring": s["ring"], "states": s["rec"]}


# ---------------------------------------------------------------------------
# the least that a pass has to read, write and compute


def work(case):
    if case["kind"] == "table":
        rot, n = HEADS[case["heads"]][3], case["positions"]
        return {"bytes": 4 * n * (rot + case["given"]), "flops": 20 * n * rot}
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rope":
        H, kvh, hd, rot, gated = HEADS[case["heads"]]
        N = case["tokens"]
        return {"bytes": N * (2 * (H + kvh) * hd * size + 4 * rot + 4 * case["rows"]), "flops": N * (H + kvh) * (3 * rot + (4 * hd if gated else 0))}
    nk, nv, dk, dv = BLOCKS[case["block"]]
    new = _lengths(case)
    conv, N, B = 2 * nk * dk + nv * dv, sum(new), case["sequences"]
    kept = sum(KERNEL - 1 + min(t, KERNEL) for t in new)
    return {"bytes": N * (conv + 2 * nv * dv + 2 * nv) * size + 4 * kept * conv + 8 * B * nv * dv * dk + 4 * KERNEL * conv,
            "flops": N * (7 * nv * dv * dk + (2 * KERNEL + 6) * conv + 10 * nv * dv)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, token by token


def _exact_delta(s):
    case = s["case"]
    nk, nv, dk, dv = BLOCKS[case["block"]]
    new, rep = _lengths(case), nv // nk
    B, T = len(new), max(new)
    x, ba = s["qkvz"].double(), s["ba"].double()
    slot = s["slots"].tolist()
    pos = s["positions"].tolist()
    ring, rec = s["ring"].double(), s["rec"].double()
    # where each channel of q, k, v, z and each gate lies in a token's row
    key, val = nk * dk, nv * dv
    if case["layout"] == "split":
        at = torch.arange(2 * key + 2 * val, device=DEV)
        gate = torch.arange(2 * nv, device=DEV).view(2, nv)
    else:
        lie = torch.arange(2 * key + 2 * val, device=DEV).view(nk, -1)
        at = torch.cat([p.flatten() for p in (lie[:, :dk], lie[:, dk:2 * dk], lie[:, 2 * dk:2 * dk + rep * dv], lie[:, 2 * dk + rep * dv:])])
        gate = torch.arange(2 * nv, device=DEV).view(nk, 2, rep).transpose(0, 1).reshape(2, nv)
    conv = 2 * key + val
    decay = torch.ones((B, T, nv), dtype=torch.float64, device=DEV)
    beta = torch.zeros((B, T, nv), dtype=torch.float64, device=DEV)
    mixed = torch.zeros((B, T, conv), dtype=torch.float64, device=DEV)
    t0 = 0
    for b, t in enumerate(new):
        u = x[t0:t0 + t][:, at[:conv]]
        past = torch.stack([ring[slot[b], (pos[b] - j) % KERNEL] for j in range(KERNEL - 1, 0, -1)])
        line = torch.cat([past, u]).T[None]  # [1, conv, K - 1 + t]
        y = (line.unfold(2, KERNEL, 1)[0] * s["conv_w"].double()[:, None]).sum(-1).T
        mixed[b, :t] = y / (1 + torch.exp(-y))
        w = ba[t0:t0 + t]
        decay[b, :t] = torch.exp(-torch.exp(s["a_log"].double()) * torch.logaddexp(w[:, gate[1]] + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device=DEV)))
        beta[b, :t] = 1 / (1 + torch.exp(-w[:, gate[0]]))
        for m in range(max(0, t - KERNEL), t):
            ring[slot[b], (pos[b] + m) % KERNEL] = u[m]
        t0 += t
    S = torch.stack([rec[j] for j in slot])  # [B, nv, dv, dk]
    seen = torch.zeros((B, T, nv, dv), dtype=torch.float64, device=DEV)
    del line, y
    for t in range(T):
        q, k = mixed[:, t, :2 * key].view(B, 2, nk, dk).unbind(1)
        q, k = (torch.repeat_interleave(y * (y.pow(2).sum(-1, keepdim=True) / dk + 1e-6).rsqrt(), rep, 1) for y in (q, k))
        v = mixed[:, t, 2 * key:].view(B, nv, dv)
        S *= decay[:, t, :, None, None]
        miss = beta[:, t, :, None] * (v - torch.einsum("bhvk,bhk->bhv", S, k / dk ** 0.5))
        S += miss[..., None] * (k / dk ** 0.5)[:, :, None]
        seen[:, t] = torch.einsum("bhvk,bhk->bhv", S, q / dk)
    for b, j in enumerate(slot):
        rec[j] = S[b]
    o = torch.cat([seen[b, :t] for b, t in enumerate(new)])
    o = o * (o.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * s["norm_w"].double()
    z = x[:, at[conv:]].view(-1, nv, dv)
    return {"out": (o * z / (1 + torch.exp(-z))).flatten(1), "ring": ring, "states": rec}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "delta":
        return _exact_delta(s)
    rot = HEADS[case["heads"]][3]
    if case["kind"] == "table":
        n = s["given"].double() if s["given"] is not None else torch.arange(s["first"], s["first"] + case["positions"], device=DEV).double()
        how, factor, original = SCALINGS[case["scaling"]] or ("none", 1.0, 0)
        size = 1 + 0.1 * math.log(factor) if how == "yarn" else 1.0
        freq = []
        for j in range(rot // 2):
            f = math.exp(-2 * j / rot * math.log(THETA * factor ** (rot / (rot - 2)) if how == "ntk" else THETA))
            if how == "yarn":
                # dims that turn over 32 times in the original context keep their angle, those that turn less than once are stretched
                edge = [rot / 2 * math.log(original / 2 / math.pi / turns, THETA) for turns in (32, 1)]
                edge = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
                share = min(max((j - edge[0]) / max(edge[1] - edge[0], 0.001), 0), 1)
                f *= 1 - share + share / factor
            freq.append(f / factor if how == "linear" else f)
        turn = torch.polar(torch.full((n.numel(), rot // 2), size, dtype=torch.float64, device=DEV), torch.outer(n, torch.tensor(freq, dtype=torch.float64, device=DEV)))
        return torch.view_as_real(turn)
    table = s["table"].double() if s["rows"] is None else s["table"].double()[s["rows"].long()]
    turn = torch.view_as_complex(table.contiguous())[:, None]
    if case["inverse"]:
        turn = turn.conj()
    outs = {}
    for n, name in enumerate("qk"):
        y = s[name].double()
        if s["norms"] is not None:
            y = s["norms"][n].double() * y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS)
        front = y[..., :rot]
        pairs = front.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["layout"] == "half" else front.unflatten(-1, (rot // 2, 2))
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = turned.transpose(-1, -2) if case["layout"] == "half" else turned
        outs[name] = torch.cat([turned.flatten(-2), y[..., rot:]], -1)
    return outs
