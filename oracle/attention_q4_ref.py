"""Oracle of attention over a KV cache held in 4 bits, in 64 bits on the CPU:
the block of QwenCPUModel.attentionForward (QwenCPUModel.swift:285-367) for
many tokens of many sequences, over rows whose values went through the cache's
format (include/swq.h, swq_q4_cache); which rows an eviction keeps.  A sequence
is a dict of codes [KVH, n, hd], scales and biases [KVH, n, hd / 64] of k and v."""

from __future__ import annotations

import math

import numpy as np

GROUP = 64
f64 = np.float64


def rope_table(n: int, rot: int, theta: float) -> np.ndarray:
    """cos, sin f32 [n, rot / 2, 2] with applyRope's float operands (QwenCPUModel.swift:356-358)."""
    out = np.empty((n, rot // 2, 2), np.float32)
    for j in range(rot // 2):
        freq = np.float32(math.pow(f64(np.float32(theta)), f64(-np.float32(2 * j) / np.float32(rot))))
        for p in range(n):
            ang = f64(np.float32(p) * freq)
            out[p, j] = math.cos(ang), math.sin(ang)
    return out


def norm_rope(x, w, eps, turn):
    """x [heads, hd] in 64 bits; turn [rot / 2, 2]."""
    x = x.astype(f64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + f64(np.float32(eps))) * w.astype(f64)
    h = len(turn)
    c, s = turn[:, 0].astype(f64), turn[:, 1].astype(f64)
    a, b = x[:, :h].copy(), x[:, h:2 * h].copy()
    x[:, :h], x[:, h:2 * h] = a * c - b * s, b * c + a * s
    return x


def quantise(x):
    """x [..., hd] -> codes [..., hd], scale and bias f16 [..., hd / 64]."""
    y = np.where(np.isnan(x), 0.0, np.clip(x, -65504.0, 65504.0)).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo, hi = y.min(-1), y.max(-1)
    bias, scale = lo.astype(np.float32).astype(np.float16), ((hi - lo) / 15.0).astype(np.float32).astype(np.float16)
    # the largest scale with which no value passes 65504, where the rounded one is larger
    passes = lambda s: bias.astype(f64) + 15 * s.astype(f64) > 65504  # noqa: E731
    most = ((65504 - bias.astype(f64)) / 15).astype(np.float16)
    scale = np.where(passes(scale), np.where(passes(most), np.nextafter(most, np.float16(0)), most), scale)
    s, b = scale.astype(f64)[..., None], bias.astype(f64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.where(s > 0, np.clip(np.rint((y - b) / s), 0, 15), 0).astype(np.uint8)
    return codes.reshape(x.shape), scale, bias


def values(part):
    codes, scale, bias = part
    return codes.astype(f64) * np.repeat(scale.astype(f64), GROUP, -1) + np.repeat(bias.astype(f64), GROUP, -1)


def empty_sequence(kvh, hd):
    return {x: (np.zeros((kvh, 0, hd), np.uint8), np.zeros((kvh, 0, hd // GROUP), np.float16),
                np.zeros((kvh, 0, hd // GROUP), np.float16)) for x in "kv"}


def random_sequence(rng, kvh, n, hd):
    """n rows of normal values, keys of the size that normalised ones have."""
    return {x: quantise(rng.standard_normal((kvh, n, hd)) * (1.0 if x == "k" else 0.7)) for x in "kv"}


def append(seq, k, v, w, eps, turns):
    """k, v [T, KVH, hd]; turns [T, rot / 2, 2]."""
    rows = np.stack([norm_rope(k[i], w, eps, turns[i]) for i in range(len(k))], 1) if len(k) else None
    if rows is None:
        return seq
    new = {"k": quantise(rows), "v": quantise(v.astype(f64).transpose(1, 0, 2))}
    return {x: tuple(np.concatenate([o, n], 1) for o, n in zip(seq[x], new[x])) for x in "kv"}


def attend(seq, before, q, w, eps, turns):
    """q [T, H, 2, hd] of the tokens whose rows are before .. in `seq`: (out [T, H, hd], the attention
    that each row gathers [KVH, rows])."""
    K, V = values(seq["k"]), values(seq["v"])
    T, H, _, hd = q.shape
    kvh, n = K.shape[:2]
    G = H // kvh
    out, got = np.zeros((T, H, hd)), np.zeros((kvh, n))
    for i in range(T):
        x = norm_rope(q[i, :, 0], w, eps, turns[i])
        m = before + i + 1
        for h in range(H):
            g = h // G
            s = K[g, :m] @ x[h] / math.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            got[g, :m] += p
            out[i, h] = p @ V[g, :m] / (1 + np.exp(-q[i, h, 1].astype(f64)))
    return out, got


def keep(weights, n, budget, sink, recent):
    """Rows of one head that an eviction keeps, in order."""
    if n <= budget:
        return np.arange(n)
    mid = np.where(np.isnan(weights[sink:n - recent]), -np.inf, weights[sink:n - recent].astype(f64))
    best = np.argsort(-mid, kind="stable")[:budget - sink - recent] + sink
    return np.sort(np.concatenate([np.arange(sink), best, np.arange(n - recent, n)])).astype(np.int64)


def words(seq, R):
    """A sequence as the cache lays it out, R rows: k words [KVH, R, hd / 8], v words [KVH, R / 8, hd],
    params [KVH, 4, hd / 64, R]; zeros past its rows."""
    kvh, n, hd = seq["k"][0].shape
    c = {x: np.zeros((kvh, R, hd), np.uint32) for x in "kv"}
    par = np.zeros((kvh, 4, hd // GROUP, R), np.float16)
    for i, x in enumerate("kv"):
        c[x][:, :n] = seq[x][0]
        par[:, 2 * i, :, :n] = seq[x][1].transpose(0, 2, 1)
        par[:, 2 * i + 1, :, :n] = seq[x][2].transpose(0, 2, 1)
    shift = 4 * np.arange(8, dtype=np.uint32)
    k = (c["k"].reshape(kvh, R, hd // 8, 8) << shift).sum(-1, dtype=np.uint32)
    v = (c["v"].reshape(kvh, R // 8, 8, hd) << shift[:, None]).sum(2, dtype=np.uint32)
    return k, v, par
