"""Blocks and batches for the tests of swq_deltanet_tokens, and what the 64-bit oracle makes of them."""

from __future__ import annotations

import torch

from oracle import deltanet_tokens_ref as R
from swiftlet_amd._lib import SWQ_DELTA_INTERLEAVED, SWQ_DELTA_SPLIT
from swiftlet_amd.deltanet import DeltaNetGPU


class Batch:
    """A block of the given heads, and sequences that bring `lengths` tokens each, with states in `slots` slots in a
    shuffled order.  spread: how far the projections' rows lie apart beyond their width."""

    def __init__(self, heads, lengths, dtype="f32", split=False, K=4, seed=0, spare=2, spread=0, decay=None, size=1.0, eps=1e-6):
        nk, nv, dk, dv = self.heads = heads
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.conv, self.val = 2 * nk * dk + nv * dv, nv * dv
        self.lengths, self.split, self.eps, self.K = lengths, split, eps, K
        self.dtype = torch.float32 if dtype == "f32" else torch.bfloat16
        B, N = len(lengths), sum(lengths)
        self.params = dict(conv_w=n(self.conv, K) * 0.5, a_log=n(nv) * 0.5 if decay is None else torch.full((nv,), float(decay), device="cuda"),
                           dt_bias=n(nv) * 0.5 - 2, norm_w=1 + 0.2 * n(dv))
        self.block = DeltaNetGPU(nk, nv, dk, dv, K, SWQ_DELTA_SPLIT if split else SWQ_DELTA_INTERLEAVED, eps, self.params["conv_w"],
                                 self.params["a_log"], self.params["dt_bias"], self.params["norm_w"])
        self.qkvz = (n(N, self.conv + self.val + spread) * size).to(self.dtype)[:, :self.conv + self.val]
        self.ba = n(N, 2 * nv + spread).to(self.dtype)[:, :2 * nv]
        self.states = self.block.new_states(B + spare)
        ring, rec = self.block.states_views(self.states)
        ring.copy_(n(*ring.shape))
        rec.copy_(n(*rec.shape) * 0.2 * size)
        self.before = self.states.clone()
        self.slots = torch.randperm(B + spare, generator=g, device="cuda")[:B].int()
        self.positions = torch.randint(0, 9, (B,), generator=g, device="cuda", dtype=torch.int32)
        self.starts = torch.tensor([sum(lengths[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
        self.ws = self.block.new_batch_workspace(B, N)

    def run(self, **kw):
        args = dict(starts=self.starts, slots=self.slots, max_tokens=max(max(self.lengths), 1))
        return self.block.prefill(self.qkvz, self.ba, self.states, self.positions, self.ws, **{**args, **kw})

    def oracle(self, lengths=None, left_out=()):
        """(out, rings, matrices) in 64 bits from the states before the call; rows of nothing are 0.  self.terms: the size
        of what each output is the sum of."""
        nk, nv, dk, dv = self.heads
        ring, rec = (t.double() for t in self.block.states_views(self.before))
        out, self.terms = torch.zeros((2, sum(self.lengths), self.val), dtype=torch.float64, device="cuda")
        for b, t in enumerate(lengths or self.lengths):
            if not t or b in left_out:
                continue
            j, n0 = int(self.slots[b]), int(self.starts[b])
            out[n0:n0 + t], ring[j], rec[j], self.terms[n0:n0 + t] = R.tokens(
                self.qkvz[n0:n0 + t], self.ba[n0:n0 + t], ring[j], rec[j], int(self.positions[b]), nk=nk, nv=nv, dk=dk, dv=dv, eps=self.eps,
                split=self.split, **self.params)
        return out, ring, rec

    def views(self):
        return self.block.states_views(self.states)


def off(got, want):
    """Largest error over the largest value."""
    return float((got.double() - want).abs().max() / want.abs().max().clamp_min(1e-300))


def bf16_off(c, got, want, rows=slice(None)):
    """Largest error beyond bf16's rounding (2^-8 of the value), over the size of what an output is the sum of."""
    err = ((got.double() - want).abs() - want.abs() * 2.0 ** -8).clamp_min(0) / c.terms.clamp_min(1e-300)
    return float(err[rows].max())
