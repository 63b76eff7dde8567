"""The gated DeltaNet block over the tokens of many sequences, in 64 bits — TEST INFRASTRUCTURE ONLY, what is held against
swq_deltanet_tokens: QwenCPUModel.deltaNetForward's formulas (QwenCPUModel.swift:371-496) token after token, as
deltanet_ref.deltanet_core has them in 32 bits.  torch, on any device."""

from __future__ import annotations

import torch


def split_rows(qkvz, ba, nk, nv, dk, dv, split):
    """The parts of projection rows in either layout, f64: mixed [N, q|k|v], z [N, nv, dv], b and a [N, nv]."""
    x, ba = qkvz.double(), ba.double()
    N, rep = x.shape[0], nv // nk
    if split:
        conv = 2 * nk * dk + nv * dv
        return x[:, :conv], x[:, conv:conv + nv * dv].reshape(N, nv, dv), ba[:, :nv], ba[:, nv:2 * nv]
    per = x[:, :2 * nk * dk + 2 * nv * dv].reshape(N, nk, -1)
    q, k, v, z = per.split([dk, dk, rep * dv, rep * dv], -1)
    gates = ba[:, :2 * nv].reshape(N, nk, 2, rep)
    mixed = torch.cat([t.reshape(N, -1) for t in (q, k, v)], 1)
    return mixed, z.reshape(N, nv, dv), gates[:, :, 0].reshape(N, nv), gates[:, :, 1].reshape(N, nv)


def tokens(qkvz, ba, ring, state, position, conv_w, a_log, dt_bias, norm_w, nk, nv, dk, dv, eps, split):
    """T tokens of one sequence whose conv ring [K, convD] and matrices [nv, dv, dk] hold `position` tokens already.
    Returns (y [T, nv * dv], ring, state), f64, and terms [T, nv * dv]: the size of what an output is the sum of where
    tokens are taken 64 at a time, so with what multiplies the sum.  That is q S over dk for the state before the 64 (as it
    has faded), and (q.k_j) d_j over the tokens since, each q.k_j itself a sum over dk; roots of the sums of squares."""
    mixed, z, b, a = split_rows(qkvz, ba, nk, nv, dk, dv, split)
    T, conv, rep = mixed.shape[0], mixed.shape[1], nv // nk
    w = conv_w.double().reshape(conv, -1)
    K = w.shape[1]
    ring, S = ring.double().clone(), state.double().clone()
    back = [ring[(position - K + 1 + j) % K] for j in range(K - 1)]
    rows = torch.cat([torch.stack(back), mixed]) if back else mixed
    x = sum(w[:, j] * rows[j:j + T] for j in range(K))
    x = x / (1 + torch.exp(-x))
    for i in range(max(0, T - K), T):
        ring[(position + i) % K] = mixed[i]
    q, k = (t.reshape(T, nk, dk) for t in x[:, :2 * nk * dk].chunk(2, 1))
    q, k = (t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (q / dk).repeat_interleave(rep, 1), (k / dk ** 0.5).repeat_interleave(rep, 1)
    v = x[:, 2 * nk * dk:].reshape(T, nv, dv)
    g = torch.exp(-torch.exp(a_log.double()) * torch.nn.functional.softplus(a + dt_bias.double(), threshold=40.0))
    beta = 1 / (1 + torch.exp(-b))
    out, terms = torch.empty((2, T, nv, dv), dtype=torch.float64, device=S.device)
    for t in range(T):
        if t % 64 == 0:
            start, ks, ds = S, [], []
        S, start, ks = S * g[t][:, None, None], start * g[t][:, None, None], [x * g[t][:, None] for x in ks]
        d = beta[t][:, None] * (v[t] - (S * k[t][:, None]).sum(-1))
        S = S + d[:, :, None] * k[t][:, None]
        out[t] = (S * q[t][:, None]).sum(-1)
        ks, ds = ks + [k[t]], ds + [d]
        p = torch.stack(ks) * q[t]  # [tokens since, nv, dk]
        size = (p.sum(-1).square() + p.square().sum(-1))[..., None] * torch.stack(ds).square()
        terms[t] = ((start * q[t][:, None]).square().sum(-1) + size.sum(0)).sqrt()
    lift = norm_w.double() * z / (1 + torch.exp(-z)) / torch.sqrt((out * out).mean(-1, keepdim=True) + eps)
    return (out * lift).reshape(T, nv * dv), ring, S, (terms * lift.abs()).reshape(T, nv * dv)
