"""The 4-bit cache on the device against its oracle in 64 bits (oracle/attention_q4_ref.py).

Bars.  Codes, scales and biases: equal, bit for bit (both sides compute them in 64 bits up to the
same two roundings), and every other byte of the cache as it was.  f32 attention: a score is a sum
of up to 256 products rounded to 24 bits, so it is off by a few 2^-24 of |q||k| / sqrt(hd), at most
16 * w_q * w_k here, say 20 * 4 * 2^-24 = 5e-6, and so is p by that factor; the sum of p v adds the
like of its own: 1e-5 of the largest output.  bf16: half a unit in the last place, 2^-8 of the value,
+ 2^-9 of the largest for queries, keys, values and p held in 11 bits (2^-12 each: 5e-4 in the scores).
Gathered weights are f32 in any case: 1e-5 of the largest, + that of the sum for long ones."""

import math

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from swiftlet_amd import _lib
from swiftlet_amd.attention_q4 import AttentionQ4GPU, Q4Cache

pytestmark = pytest.mark.gpu

f32 = np.float32
EPS, THETA = 1e-6, 1e6


def _torch():
    import torch
    return torch


class Setup:
    """A block, a cache whose unused bytes are all ones (NaN as parameters), the oracle's sequences."""

    def __init__(self, seed, H, KVH, hd, rot, before, max_positions, table=None, positions=0):
        torch = _torch()
        self.rng = rng = np.random.default_rng(seed)
        self.H, self.KVH, self.hd, self.rot, self.max = H, KVH, hd, rot, max_positions
        self.qw, self.kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(f32) for _ in range(2))
        self.table = R.rope_table(positions or max_positions, rot, THETA)
        rope = torch.from_numpy(self.table).cuda() if positions else None
        self.blk = AttentionQ4GPU(H, KVH, hd, rot, THETA, EPS, max_positions, self.qw, self.kw, rope_table=rope)
        self.cache = self.blk.new_cache(len(before))
        self.cache.data.fill_(255)
        self.R = (max_positions + 31) // 32 * 32
        self.seqs = [R.random_sequence(rng, KVH, n, hd) for n in before]
        for b, s in enumerate(self.seqs):
            self.put(b, s)
        self.before = list(before)

    def put(self, b, s):
        torch = _torch()
        n = s["k"][0].shape[1]
        k, v, par = R.words(s, self.R)
        ck, cv, cp = self.cache.views()
        ck[b, :, :n] = torch.from_numpy(k[:, :n].view(np.int32)).cuda()
        full, part = n // 8, n % 8
        cv[b, :, :full] = torch.from_numpy(v[:, :full].view(np.int32)).cuda()
        if part:  # the rest of the last block's words keep their ones
            keep = np.uint32(0xFFFFFFFF) << np.uint32(4 * part)
            cv[b, :, full] = torch.from_numpy((v[:, full] | keep).view(np.int32)).cuda()
        cp[b, :, :, :, :n] = torch.from_numpy(par[..., :n]).cuda()

    def tokens(self, counts, dtype):
        torch = _torch()
        N = sum(counts)
        q, k, v = (self.rng.standard_normal((N, n)).astype(f32) for n in (self.H * 2 * self.hd, self.KVH * self.hd, self.KVH * self.hd))
        t = [torch.from_numpy(x).to(dtype).cuda() for x in (q, k, v)]
        self.q, self.k, self.v = (x.float().cpu().numpy() for x in t)
        return t

    def rows(self):
        return _torch().tensor(self.before, dtype=_torch().int32, device="cuda")

    def starts(self, counts):
        return _torch().tensor(np.cumsum([0, *counts]), dtype=_torch().int32, device="cuda")

    def expect(self, counts, positions=None, attend=True, appended=True):
        """The oracle's sequences advanced, its outputs [N, H*hd] and gathered [B][KVH, rows]."""
        out, got, n0 = [], [], 0
        for b, t in enumerate(counts):
            p0 = self.before[b] if positions is None else positions[b]
            turns = self.table[np.minimum(np.arange(p0, p0 + t), len(self.table) - 1)]
            if appended:
                self.seqs[b] = R.append(self.seqs[b], self.k[n0:n0 + t].reshape(t, self.KVH, self.hd), self.v[n0:n0 + t].reshape(t, self.KVH, self.hd),
                                        self.kw, EPS, turns)
            if attend:
                o, g = R.attend(self.seqs[b], self.before[b], self.q[n0:n0 + t].reshape(t, self.H, 2, self.hd), self.qw, EPS, turns)
                out.append(o.reshape(t, self.H * self.hd))
                got.append(g)
            n0 += t
        return (np.concatenate(out) if out else None), got

    def check_cache(self):
        """Every row of the oracle's in the cache, and ones behind them."""
        ck, cv, cp = (x.cpu().numpy() for x in self.cache.views())
        for b, s in enumerate(self.seqs):
            n = s["k"][0].shape[1]
            k, v, par = R.words(s, self.R)
            assert np.array_equal(ck[b, :, :n].view(np.uint32), k[:, :n]), f"k codes of {b}"
            assert (ck[b, :, n:] == -1).all(), f"k behind {b}"
            gv = cv[b].view(np.uint32)
            codes = np.stack([(gv >> np.uint32(4 * u)) & 15 for u in range(8)], 2).reshape(self.KVH, self.R, self.hd)
            assert np.array_equal(codes[:, :n], s["v"][0]), f"v codes of {b}"
            assert (codes[:, n:] == 15).all(), f"v behind {b}"
            assert np.array_equal(cp[b][..., :n].view(np.uint16), par[..., :n].view(np.uint16)), f"params of {b}"
            assert (cp[b][..., n:].view(np.uint16) == 0xFFFF).all(), f"params behind {b}"


def _types():
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16}


def _close(got, want, dtype):
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    top = np.abs(want).max()
    off = np.abs(got - want)
    bar = 1e-5 * top if dtype == "f32" else np.abs(want) * 2.0 ** -8 + top * 2.0 ** -9
    print(f"  off by {(off / top).max():.2e} of the largest", flush=True)
    assert (off <= bar).all(), (off / top).max()


APPENDS = [  # H, KVH, hd, rot, before, counts
    (16, 2, 256, 64, [0], [1]), (16, 2, 256, 64, [7, 8, 30], [1, 1, 1]), (8, 8, 64, 0, [5, 0, 61], [3, 0, 19]), (4, 1, 128, 128, [31], [33]),
    (6, 3, 128, 34, [1, 2, 3, 60], [1, 9, 30, 5]), (2, 2, 256, 256, [3], [70])]


@pytest.mark.parametrize("H,KVH,hd,rot,before,counts", APPENDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_appended_rows_are_the_oracles(H, KVH, hd, rot, before, counts, dtype):
    s = Setup(hd + len(before), H, KVH, hd, rot, before, 97)
    _, k, v = s.tokens(counts, _types()[dtype])
    print(f"append {before} + {counts}, hd {hd}", flush=True)
    same = len(set(counts)) == 1
    s.blk.append(k, v, s.cache, s.rows(), starts=None if same else s.starts(counts), max_tokens=max(counts))
    s.expect(counts, attend=False)
    s.check_cache()


def test_append_saturates_and_clips():
    """NaN is stored as 0, infinities as the largest finite value; rows past the cache are not written."""
    torch = _torch()
    s = Setup(3, 2, 2, 128, 0, [38], 40)
    _, k, v = s.tokens([6], torch.float32)
    bad = [np.nan, np.inf, -np.inf, 1e30, 3e-8, 0.0]
    s.v[0, :6] = s.v[1, 128:134] = bad
    s.v[1, :64] = 2.5  # equal values
    s.k[1, 3] = np.nan  # spreads over its head by the norm
    k, v = torch.from_numpy(s.k).cuda(), torch.from_numpy(s.v).cuda()
    s.blk.append(k, v, s.cache, s.rows())
    s.k, s.v = s.k[:2], s.v[:2]
    with np.errstate(all="ignore"):
        s.expect([2], attend=False)
    s.check_cache()
    kv, vv = s.cache.read(s.rows(), 4)
    assert torch.isfinite(kv).all() and torch.isfinite(vv).all() and (vv[0, 1, 0, :64] == 2.5).all()
    assert (kv[0, 2:] == 0).all() and (vv[0, 2:] == 0).all()
    assert (kv[0, 1, 0] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_read_gives_the_values(hd, dtype):
    torch = _torch()
    s = Setup(hd, 2, 2, hd, 0, [70, 0, 33], 70)
    t = _types()[dtype]
    first = torch.tensor([3, 0, 30], dtype=torch.int32, device="cuda")
    want = np.zeros((2, 3, 40, 2, hd))
    for i, x in enumerate("kv"):
        for b, (f, n) in enumerate(zip((3, 0, 30), (70, 0, 33))):
            v = R.values(s.seqs[b][x]).transpose(1, 0, 2)[f:f + 40]
            want[i, b, :len(v)] = v
    got = s.cache.read(first, 40, dtype=t, rows=s.rows())
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), torch.from_numpy(w.astype(f32)).to(t))
    starts = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    got = s.cache.read(first, 0, dtype=t, starts=starts, tokens=5, rows=s.rows())
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), torch.from_numpy(np.concatenate([w[0, :2], w[2, :3]]).astype(f32)).to(t))


STEPS = [  # H, KVH, hd, rot, before, max_positions
    (1, 1, 64, 0, [0], 1), (16, 2, 256, 64, [0], 64), (16, 2, 256, 64, [31, 0, 32, 33, 127], 200), (32, 8, 128, 128, [128, 257, 5], 300),
    (8, 8, 64, 16, [511, 1000, 64, 63], 1001), (16, 1, 128, 32, [640], 4096), (3, 1, 256, 2, [1300, 77], 1301), (16, 2, 256, 2, [5000], 5001),
    (20, 4, 64, 2, [2047, 2048, 2049], 2300)]


@pytest.mark.parametrize("H,KVH,hd,rot,before,most", STEPS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("weights", [False, True])
def test_step(H, KVH, hd, rot, before, most, dtype, weights):
    torch = _torch()
    s = Setup(most + H, H, KVH, hd, rot, before, most)
    B = len(before)
    counts = [1] * B
    q, k, v = s.tokens(counts, _types()[dtype])
    ws = s.blk.new_workspace(s.cache, weights=weights)
    ws.fill_(255)
    w = torch.full((B, KVH, most), 0.25, device="cuda") if weights else None
    print(f"step H {H} KVH {KVH} hd {hd} rows {before}", flush=True)
    out = s.blk.step(q, k, v, s.cache, s.rows(), ws, weights=w)
    want, got = s.expect(counts)
    _close(out, want, dtype)
    s.check_cache()
    if weights:
        w = w.cpu().numpy()
        for b, n in enumerate(before):
            assert (w[b, :, n + 1:] == 0.25).all()
            g = got[b].copy()
            g[:, :n] += 0.25
            assert np.abs(w[b, :, :n + 1] - g).max() <= 1e-5 * max(1.0, g.max())


PREFILLS = [  # H, KVH, hd, rot, before, counts, max_positions
    (16, 2, 256, 64, [0], [2], 64), (16, 2, 256, 64, [0], [77], 77), (8, 8, 64, 0, [0, 130], [65, 64], 200), (32, 8, 128, 128, [5, 0, 200], [40, 0, 33], 240),
    (3, 1, 128, 2, [31], [129], 160), (16, 1, 256, 2, [100, 3], [17, 1], 128), (16, 2, 256, 2, [700], [20], 1024), (6, 3, 64, 32, [0, 9, 300], [1, 130, 7], 307),
    (1, 1, 128, 16, [1], [200], 256), (16, 2, 256, 2, [2100], [3], 2103)]


@pytest.mark.parametrize("H,KVH,hd,rot,before,counts,most", PREFILLS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("weights", [False, True])
def test_prefill(H, KVH, hd, rot, before, counts, most, dtype, weights):
    torch = _torch()
    s = Setup(most + H + hd, H, KVH, hd, rot, before, most)
    B, N = len(before), sum(counts)
    q, k, v = s.tokens(counts, _types()[dtype])
    ws = s.blk.new_workspace(s.cache, tokens=N, max_tokens=max(counts), weights=weights)
    ws.fill_(255)
    w = torch.full((B, KVH, most), 0.25, device="cuda") if weights else None
    print(f"prefill H {H} KVH {KVH} hd {hd} rows {before} + {counts}", flush=True)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, starts=s.starts(counts), max_tokens=max(counts), weights=w)
    want, got = s.expect(counts)
    _close(out, want, dtype)
    s.check_cache()
    if weights:
        w = w.cpu().numpy()
        for b, (n, t) in enumerate(zip(before, counts)):
            if t == 0:
                assert (w[b] == 0.25).all()
                continue
            assert (w[b, :, n + t:] == 0.25).all()
            g = got[b].copy()
            g[:, :n] += 0.25
            assert np.abs(w[b, :, :n + t] - g).max() <= 1e-5 * max(1.0, g.max())


@pytest.mark.parametrize("counts", [[1, 1], [5, 9]])
def test_positions_apart_from_rows(counts):
    """After an eviction a token's rotary position is larger than its row; past the table: its last entry."""
    torch = _torch()
    s = Setup(9, 4, 2, 128, 64, [40, 20], 96, positions=500)
    pos = [333, 497]
    q, k, v = s.tokens(counts, torch.float32)
    ws = s.blk.new_workspace(s.cache, tokens=sum(counts), max_tokens=max(counts))
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, starts=s.starts(counts), max_tokens=max(counts),
                        positions=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    want, _ = s.expect(counts, pos)
    _close(out, want, "f32")
    s.check_cache()


@pytest.mark.parametrize("counts", [[1, 1, 1], [4, 30, 2]])
def test_a_shared_cache_is_only_read(counts):
    """k and v None: the rows are there; nothing is written, and the result is that of the call that appends."""
    torch = _torch()
    s = Setup(11, 8, 2, 64, 16, [40, 0, 90], 130)
    q, k, v = s.tokens(counts, torch.float32)
    ws = s.blk.new_workspace(s.cache, tokens=sum(counts), max_tokens=max(counts))
    kw = dict(starts=s.starts(counts), max_tokens=max(counts))
    both = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, **kw)
    held = s.cache.data.clone()
    alone = s.blk.prefill(q, None, None, s.cache, s.rows(), ws, **kw)
    assert torch.equal(both, alone) and torch.equal(held, s.cache.data)
    want, _ = s.expect(counts)
    _close(alone, want, "f32")


@pytest.mark.parametrize("counts,hint", [([1, 1], 1), ([1, 1], 7), ([60, 33], 2), ([3, 2], 1)])
def test_hints_of_rows_only_split_the_work(counts, hint):
    """max_rows too small or too large: the same rows are read, up to the order of sums."""
    torch = _torch()
    s = Setup(12, 16, 2, 128, 32, [700, 431], 800)
    q, k, v = s.tokens(counts, torch.float32)
    ws = s.blk.new_workspace(s.cache, tokens=sum(counts), max_tokens=max(counts), weights=True)
    want, got = s.expect(counts)
    for h in (hint, 0, 760, 10 ** 6):
        w = s.blk.new_weights(s.cache)
        out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, starts=s.starts(counts), max_tokens=max(counts), max_rows=h, weights=w)
        _close(out, want, "f32")
        for b in range(2):
            n = got[b].shape[1]
            assert np.abs(w[b, :, :n].cpu().numpy() - got[b]).max() < 1e-5 * max(1.0, got[b].max())


@pytest.mark.parametrize("size", [1e-4, 300.0, 2e4])
@pytest.mark.parametrize("T", [1, 20])
def test_values_of_any_size(size, T):
    """Values far from 1 and queries of large norm weights: sums keep their relative precision."""
    torch = _torch()
    s = Setup(13, 4, 1, 128, 0, [300], 400)
    for x in ("v",):
        s.seqs[0][x] = R.quantise(s.rng.standard_normal((1, 300, 128)) * size)
    s.put(0, s.seqs[0])
    q, k, v = s.tokens([T], torch.float32)
    v *= size
    s.v = v.cpu().numpy()
    ws = s.blk.new_workspace(s.cache, tokens=T, max_tokens=T)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws)
    want, _ = s.expect([T])
    _close(out, want, "f32")


@pytest.mark.parametrize("T", [1, 40])
def test_one_row_takes_all_the_attention(T):
    """Scores tens of times larger than usual: most weights underflow, none of the sums does."""
    torch = _torch()
    s = Setup(14, 4, 1, 64, 0, [200], 256)
    s.blk.q_norm.mul_(40.0)
    s.qw = s.qw * f32(40)
    s.blk.q_norm.copy_(torch.from_numpy(s.qw))
    q, k, v = s.tokens([T], torch.float32)
    ws = s.blk.new_workspace(s.cache, tokens=T, max_tokens=T)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws)
    want, _ = s.expect([T])
    # scores of up to 40 * 8 * 4 are off by 2^-24 of that each: 40 times the usual bar
    off = np.abs(out.cpu().numpy() - want).max() / np.abs(want).max()
    print(f"  off by {off:.2e}", flush=True)
    assert off < 4e-4


@pytest.mark.parametrize("n,budget,sink,recent,hd", [(1, 1, 0, 0, 64), (100, 100, 4, 4, 64), (100, 99, 4, 4, 128), (1000, 37, 4, 16, 256),
                                                    (1000, 20, 4, 16, 64), (5000, 2500, 0, 0, 64), (1030, 1029, 0, 1, 128), (3000, 1, 0, 0, 64)])
def test_evicted_rows(n, budget, sink, recent, hd):
    torch = _torch()
    rng = np.random.default_rng(n + budget)
    KVH, B = 2, 3
    before = [n, max(1, n // 2), 0]
    s = Setup(n, KVH, KVH, hd, 0, before, n + 3)
    w = np.exp(2 * rng.standard_normal((B, KVH, n + 3))).astype(f32)
    w[rng.random(w.shape) < 0.3] = 0.0
    w[rng.random(w.shape) < 0.1] = f32(0.125)
    w[0, 0, n // 3] = np.nan
    w[0, 1, n // 3:] = 1.0  # ties
    most = budget + 5
    into = s.blk.new_cache(B, most)
    into.data.fill_(255)
    nw = torch.full((B, KVH, most), -1.0, device="cuda")
    print(f"evict {n} to {budget}", flush=True)
    kept, rows = s.blk.evict(s.cache, torch.from_numpy(w).cuda(), s.rows(), into, budget, sink, recent, new_weights=nw)
    kept, nw = kept.cpu().numpy(), nw.cpu().numpy()
    assert rows.tolist() == [min(budget, m) for m in before]
    k, v = (x.cpu().numpy() for x in into.read(None, budget, rows=rows))
    for b in range(B):
        for h in range(KVH):
            want = R.keep(w[b, h], before[b], budget, sink, recent)
            m = len(want)
            assert kept[b, h, :m].tolist() == want.tolist() and (kept[b, h, m:] == -1).all()
            assert np.array_equal(nw[b, h, :m], w[b, h, want], equal_nan=True) and (nw[b, h, m:] == 0).all()
            for x, got in (("k", k), ("v", v)):
                vals = R.values(tuple(p[h] for p in s.seqs[b][x]))[want].astype(f32)
                assert np.array_equal(got[b, :m, h], vals), (b, h, x)
                assert (got[b, m:, h] == 0).all()
    s.check_cache()  # the source is as it was


def test_prompt_eviction_and_tokens_together():
    torch = _torch()
    H, KVH, hd, rot, budget = 8, 2, 64, 16, 40
    s = Setup(21, H, KVH, hd, rot, [0, 0], 128, positions=300)
    small = s.blk.new_cache(2, 64)
    w, small_w = s.blk.new_weights(s.cache), s.blk.new_weights(small)
    ws = s.blk.new_workspace(s.cache, tokens=128, max_tokens=64, weights=True)
    gathered = [np.zeros((KVH, 0)), np.zeros((KVH, 0))]
    rows, pos = s.rows(), s.rows()
    for counts in ([33, 60], [30, 2]):
        q, k, v = s.tokens(counts, torch.float32)
        out = s.blk.prefill(q, k, v, s.cache, rows, ws, starts=s.starts(counts), max_tokens=max(counts), weights=w)
        want, got = s.expect(counts)
        _close(out, want, "f32")
        for b in range(2):
            s.before[b] += counts[b]
            n = gathered[b].shape[1]
            got[b][:, :n] += gathered[b]
            gathered[b] = got[b]
        rows = s.rows()
    pos = rows.clone()
    kept, rows = s.blk.evict(s.cache, w, rows, small, budget, 2, 8, new_weights=small_w)
    kept = kept.cpu().numpy()
    seqs = []
    for b in range(2):
        seq = {}
        for x in "kv":
            parts = []
            for p in s.seqs[b][x]:
                parts.append(np.stack([p[h][kept[b, h]] for h in range(KVH)]))
            seq[x] = tuple(parts)
        for h in range(KVH):
            # the oracle's choice, but for rows whose weights are closer than the device's sums are exact
            best = R.keep(gathered[b][h].astype(f32), s.before[b], budget, 2, 8)
            odd = set(best) ^ set(kept[b, h].tolist())
            border = np.sort(gathered[b][h][2:-8])[::-1][budget - 10 - 1]
            assert all(abs(gathered[b][h][t] - border) < 1e-4 for t in odd)
        seqs.append(seq)
    s.seqs, s.before, s.cache, s.R = seqs, [budget, budget], small, 64
    at = pos.tolist()
    for i in range(20):  # token by token
        q, k, v = s.tokens([1, 1], torch.float32)
        out = s.blk.step(q, k, v, small, rows, ws, weights=small_w, positions=pos)
        want, _ = s.expect([1, 1], [p + i for p in at])
        _close(out, want, "f32")
        s.before = [n + 1 for n in s.before]
        rows, pos = rows + 1, pos + 1


@pytest.mark.parametrize("T,weights", [(1, False), (1, True), (37, True)])
def test_replays_of_a_captured_call_follow_the_rows(T, weights):
    """One captured call, its rows advancing on the device, against eager calls on a cache of its own."""
    torch = _torch()
    s = Setup(31, 16, 2, 128, 32, [300, 41], 500)
    e = Setup(31, 16, 2, 128, 32, [300, 41], 500)
    N = 2 * T
    q, k, v = (torch.empty((N, n), device="cuda") for n in (16 * 256, 256, 256))
    ws, we = (x.blk.new_workspace(x.cache, tokens=N, max_tokens=T, weights=weights) for x in (s, e))
    w, u = ((x.blk.new_weights(x.cache) if weights else None) for x in (s, e))
    rows, mine, out = s.rows(), e.rows(), torch.empty((N, 16 * 128), device="cuda")

    def fill(i):
        for j, x in enumerate((q, k, v)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(10 * i + j), device="cuda"))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held, kept = s.cache.data.clone(), (w.clone() if weights else None)
    with torch.cuda.stream(side):
        s.blk.prefill(q, k, v, s.cache, rows, ws, out=out, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.blk.prefill(q, k, v, s.cache, rows, ws, out=out, weights=w)
        rows.add_(T)
    s.cache.data.copy_(held)
    if weights:
        w.copy_(kept)
    for i in range(4):
        fill(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        want = e.blk.prefill(q, k, v, e.cache, mine, we, weights=u)
        mine = mine + T
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(s.cache.data, e.cache.data) and (not weights or torch.equal(w, u)), i


def test_two_streams_with_workspaces_of_their_own():
    """Calls on two streams at once give what they give one after the other."""
    torch = _torch()
    both, want = [], []
    for seed in (41, 42):
        s = Setup(seed, 16, 2, 256, 64, [1200], 1300)
        s.args = s.tokens([9], torch.bfloat16)
        s.ws = s.blk.new_workspace(s.cache, tokens=9, max_tokens=9, weights=True)
        s.w = s.blk.new_weights(s.cache)
        want.append((s.blk.prefill(*s.args, s.cache, s.rows(), s.ws, weights=s.w), s.w.clone(), s.cache.data.clone()))
        both.append(s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    for s in both:
        s.w.zero_()
        s.r = s.rows()
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(both, streams)):
            with torch.cuda.stream(st):
                s.w.zero_()
            got[i] = s.blk.prefill(*s.args, s.cache, s.r, s.ws, weights=s.w, stream=st)
    torch.cuda.synchronize()
    for s, g, (o, w, c) in zip(both, got, want):
        assert torch.equal(g, o) and torch.equal(s.w, w) and torch.equal(s.cache.data, c)


def test_same_bits_again_and_in_any_batch():
    """A call repeated gives the same bits; a single-token call of one sequence those that it has in a
    batch with the same hint of rows."""
    torch = _torch()
    s = Setup(51, 16, 2, 256, 64, [900, 3, 400], 1000)
    q, k, v = s.tokens([1, 1, 1], torch.float32)
    ws = s.blk.new_workspace(s.cache, weights=True)
    first = None
    for _ in range(3):
        w = s.blk.new_weights(s.cache)
        out = s.blk.step(q, k, v, s.cache, s.rows(), ws, weights=w)
        if first is not None:
            assert torch.equal(out, first[0]) and torch.equal(w, first[1])
        first = (out, w)


def test_bad_rows_and_starts_stay_in_bounds():
    """Device arrays are clamped: the call returns, and writes rows of the cache only.  rows past the
    cache: nothing is appended, every row is seen; negative ones count as none."""
    torch = _torch()
    for rows, counts in (([64, -5], [1, 1]), ([1000, -2 ** 31], [1, 1]), ([2 ** 31 - 1, 60], [3, 9]), ([-7, 63], [20, 4])):
        s = Setup(61, 4, 2, 64, 16, [64, 64], 64)
        q, k, v = s.tokens(counts, torch.float32)
        N = sum(counts)
        ws = s.blk.new_workspace(s.cache, tokens=N, max_tokens=max(counts), weights=True)
        r = torch.tensor(rows, dtype=torch.int32, device="cuda")
        w = s.blk.new_weights(s.cache)
        held = s.cache.data.clone()
        out = s.blk.prefill(q, k, v, s.cache, r, ws, starts=s.starts(counts), max_tokens=max(counts), weights=w)
        assert torch.isfinite(out).all() and torch.isfinite(w).all(), rows
        if min(rows) >= 64:
            assert torch.equal(held, s.cache.data)
    starts = torch.tensor([-3, 900, 2], dtype=torch.int32, device="cuda")
    out = s.blk.prefill(q, k, v, s.cache, r, ws, starts=starts, max_tokens=max(counts))
    torch.cuda.synchronize()
    assert out.shape[0] == N


def test_no_tokens_and_refusals_in_python():
    torch = _torch()
    s = Setup(71, 4, 2, 64, 16, [3, 3], 64)
    q, k, v = s.tokens([1, 1], torch.float32)
    ws = s.blk.new_workspace(s.cache)
    held = s.cache.data.clone()
    none = q[:0]
    assert s.blk.prefill(none, k[:0], v[:0], s.cache, s.rows(), ws, max_tokens=1).shape == (0, 4 * 64)
    s.blk.append(k[:0], v[:0], s.cache, s.rows(), max_tokens=1)
    for call, code in ((lambda: s.blk.step(q.half(), k.half(), v.half(), s.cache, s.rows(), ws), _lib.SWQ_ERR_UNSUPPORTED_DTYPE),
                       (lambda: s.blk.step(q, k.bfloat16(), v, s.cache, s.rows(), ws), _lib.SWQ_ERR_UNSUPPORTED_DTYPE),
                       (lambda: s.blk.step(q, None, v, s.cache, s.rows(), ws), _lib.SWQ_ERR_INVALID_ARGUMENT),
                       (lambda: s.blk.step(q[:1], k, v, s.cache, s.rows(), ws), _lib.SWQ_ERR_BAD_SHAPE),
                       (lambda: s.blk.step(q, k[:1], v, s.cache, s.rows(), ws), _lib.SWQ_ERR_BAD_SHAPE),
                       (lambda: s.blk.step(q, k, v, s.cache, s.rows().long(), ws), _lib.SWQ_ERR_BAD_SHAPE),
                       (lambda: s.blk.step(q, k, v, s.cache, s.rows(), ws[:256]), _lib.SWQ_ERR_WORKSPACE),
                       (lambda: s.blk.step(q, k, v, s.cache, s.rows(), ws, weights=torch.zeros(2, 2, 63, device="cuda")), _lib.SWQ_ERR_BAD_SHAPE),
                       (lambda: s.blk.step(q.T.contiguous().T, k, v, s.cache, s.rows(), ws), _lib.SWQ_ERR_BAD_SHAPE),
                       (lambda: s.cache.read(None, 0, starts=s.starts([1, 1])), _lib.SWQ_ERR_INVALID_ARGUMENT),
                       (lambda: Q4Cache(1, 2, 96, 10), _lib.SWQ_ERR_LIMIT),
                       (lambda: Q4Cache(2, 2, 64, 64, data=held[:1024]), _lib.SWQ_ERR_WORKSPACE),
                       (lambda: s.blk.evict(s.cache, s.blk.new_weights(s.cache), s.rows(), s.blk.new_cache(2, 8), 9), _lib.SWQ_ERR_LIMIT),
                       (lambda: s.blk.evict(s.cache, s.blk.new_weights(s.cache), s.rows(), s.cache, 9), _lib.SWQ_ERR_INVALID_ARGUMENT)):
        with pytest.raises(_lib.SwqError) as e:
            call()
        assert e.value.code == code
    torch.cuda.synchronize()
    assert torch.equal(held, s.cache.data)


def test_a_block_of_the_checkpoint_over_a_4_bit_cache():
    """forward_token: projections, step and o_proj, against the oracle's block on the same projections."""
    torch = _torch()
    from swiftlet_amd.attention import AttentionGPU
    from swiftlet_amd.engine import HipEngine
    from swiftlet_amd.moe import synth_linear
    eng = HipEngine()
    H, KVH, hd, rot, width = 4, 2, 64, 16, 256
    lin = lambda i, rows, cols: synth_linear(i, 0, "router", None, rows, cols, 4, 64)  # noqa: E731
    s = Setup(81, H, KVH, hd, rot, [0], 40)
    at = AttentionGPU(H, KVH, hd, rot, THETA, EPS, 40, s.qw, s.kw, projections=[lin(i, n, width) for i, n in
                      enumerate((2 * H * hd, KVH * hd, KVH * hd))], o_proj=lin(9, width, H * hd))
    s.blk = AttentionQ4GPU.of(at)
    ws = s.blk.new_workspace(s.cache)
    for i in range(5):
        x = torch.from_numpy(s.rng.standard_normal(width).astype(f32)).cuda()
        r = s.blk.forward_token(eng, x, s.cache, s.rows(), ws, norm_weight=torch.ones(width, device="cuda"), eps=EPS)
        q, k, v = (torch.empty(p.out_dim, device="cuda") for p in at.projections)
        eng.encode_gemv_multi(list(at.projections), x, [q, k, v], norm_weight=torch.ones(width, device="cuda"), eps=EPS)
        s.q, s.k, s.v = (t.cpu().numpy()[None] for t in (q, k, v))
        want, _ = s.expect([1])
        y = torch.empty(width, device="cuda")
        eng.encode_gemv(at.o_proj, torch.from_numpy(want[0].astype(f32)).cuda(), y)
        assert float((r - y).abs().max() / y.abs().max()) < 2e-5
        s.before[0] += 1
    s.check_cache()
