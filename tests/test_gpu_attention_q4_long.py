"""The 4-bit cache on the device where sizes get large, calls mixed and arguments misplaced: caches
whose bytes pass 32 bits, tens of thousands of rows against attention in 64 bits over the values read
back, evictions of more rows than are held in registers at once, two captured calls that share a
workspace, calls on another stream, f32 and bf16 on either side of one call, tensors of the host.

Bars.  As for short ones, in f32 1e-5 of the largest: a score is off by 5e-6 at most, and so is each p,
whatever their number; l and the sums of p v are made of lanes' f32 sums of a few hundred to a thousand
terms, whose roundings, to the nearest and of either sign, add up to some 32 * 2^-24 = 2e-6.  bf16: half a
unit in the last place, 2^-8 of the value, + 2^-9 of the largest for what is held in 11 bits."""

import math

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from swiftlet_amd import _lib
from swiftlet_amd.attention_q4 import AttentionQ4GPU, Q4Cache

pytestmark = pytest.mark.gpu

f32 = np.float32


def _torch():
    import torch
    return torch


def _block(H, KVH, hd, rot, max_positions, seed, table=None):
    rng = np.random.default_rng(seed)
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(f32) for _ in range(2))
    return AttentionQ4GPU(H, KVH, hd, rot, 1e6, 1e-6, max_positions, qw, kw, rope_table=table), qw, kw


def _random(seed, *shapes, dtype=None):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(dtype or torch.float32) for s in shapes]


def _queries(q, H, hd, qw, turns):
    """Normalised and turned queries [T, H, hd] and sigmoids of the gates, in 64 bits."""
    q = q.double().cpu().numpy().reshape(len(q), H, 2, hd)
    x = np.stack([R.norm_rope(q[i, :, 0], qw, 1e-6, turns[i]) for i in range(len(q))])
    return x, 1 / (1 + np.exp(-q[:, :, 1]))


def _attend(x, gate, k, v, before, chunk=64):
    """Attention of x [T, H, hd] over k, v [n, KVH, hd] (device, f64), and what each row gathers [KVH, n]."""
    torch = _torch()
    T, H, hd = x.shape
    n, KVH = k.shape[:2]
    G = H // KVH
    out, got = torch.empty((T, H, hd), dtype=torch.float64, device="cuda"), torch.zeros((KVH, n), dtype=torch.float64, device="cuda")
    xq = torch.from_numpy(x).cuda()
    for t in range(0, T, chunk):
        m = min(chunk, T - t)
        hidden = torch.arange(n, device="cuda")[None, :] > before + t + torch.arange(m, device="cuda")[:, None]
        for h in range(H):
            s = xq[t:t + m, h] @ k[:, h // G].T.contiguous() / math.sqrt(hd)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            got[h // G] += p.sum(0)
            out[t:t + m, h] = p @ v[:, h // G].contiguous()
    return (out * torch.from_numpy(gate).cuda()).reshape(T, H * hd), got


def _close(got, want, bf16, what):
    off, top = (got.double() - want).abs(), want.abs().max()
    print(f"  {what} off by {(off / top).max().item():.2e} of the largest", flush=True)
    assert bool(_torch().isfinite(got).all())
    bar = want.abs() * 2.0 ** -8 + top * 2.0 ** -9 if bf16 else 1e-5 * top
    assert bool((off <= bar).all()), what


@pytest.mark.parametrize("H,KVH,hd,rot,n,T", [(16, 2, 256, 64, 33000, 1), (8, 8, 64, 0, 20011, 1), (8, 2, 128, 128, 33000, 1), (8, 2, 256, 64, 33000, 75),
                                               (16, 8, 64, 32, 9001, 130), (8, 2, 128, 128, 20011, 200)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_caches(H, KVH, hd, rot, n, T, dtype):
    torch = _torch()
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    blk, qw, _ = _block(H, KVH, hd, rot, n + T + 7, n + T)
    cache = blk.new_cache(1)
    k0, v0, k, v, q = _random(n, (n, KVH * hd), (n, KVH * hd), (T, KVH * hd), (T, KVH * hd), (T, 2 * H * hd), dtype=dt)
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k0, v0, cache, rows)
    rows += n
    w, ws = blk.new_weights(cache), blk.new_workspace(cache, tokens=T, max_tokens=T, weights=True)
    print(f"{n} rows, {T} tokens, {dtype}", flush=True)
    plain = blk.prefill(q, k, v, cache, rows, ws, max_rows=n + T)
    out = blk.prefill(q, None, None, cache, rows, ws, weights=w)  # and with as many splits as the cache allows
    kk, vv = cache.read(None, n + T)
    turns = (blk.rope_table.cpu().numpy() if rot else np.zeros((n + T, 0, 2), f32))[n:n + T]
    want, got = _attend(*_queries(q, H, hd, qw, turns), kk[0].double(), vv[0].double(), n)
    _close(plain, want, dtype == "bf16", "out")
    _close(out, want, dtype == "bf16", "out beside weights")
    _close(w[0, :, :n + T], got, False, "weights")
    assert not w[0, :, n + T:].any()


def test_a_cache_of_more_bytes_than_32_bits_count():
    """Two sequences of 4,300,000 rows of 4 heads of 256 (4.4 GB of key words alone): rows of zeros but
    the last ones, so that attention has a closed form."""
    torch = _torch()
    H = KVH = 4
    hd, rot, maxp = 256, 32, 4_300_000
    table = R.rope_table(64, rot, 1e6)
    blk, qw, kw = _block(H, KVH, hd, rot, maxp, 5, torch.from_numpy(table).cuda())
    cache = blk.new_cache(2)
    assert cache.views()[0].numel() * 4 > 2 ** 32
    n = maxp - 40
    rows = torch.tensor([9, n], dtype=torch.int32, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    seq, before = R.empty_sequence(KVH, hd), 0
    w = blk.new_weights(cache)
    for counts in ([1, 1], [7, 13]):
        N, T = sum(counts), counts[1]
        k, v, q = _random(N, (N, KVH * hd), (N, KVH * hd), (N, 2 * H * hd))
        starts = torch.tensor(np.cumsum([0, *counts]), dtype=torch.int32, device="cuda")
        ws = blk.new_workspace(cache, tokens=N, max_tokens=max(counts), weights=True)
        held = w[1].clone()
        print(f"{counts} tokens at {n + before}", flush=True)
        out = blk.prefill(q, k, v, cache, rows, ws, starts=starts, max_tokens=max(counts), weights=w, positions=pos)
        turns = table[np.minimum(np.arange(before, before + T), 63)]
        mine = slice(counts[0], N)
        seq = R.append(seq, *(x[mine].cpu().numpy().reshape(T, KVH, hd) for x in (k, v)), kw, 1e-6, turns)
        x, gate = _queries(q[mine], H, hd, qw, turns)
        K, V = R.values(seq["k"]), R.values(seq["v"])
        want, got, empty = np.zeros((T, H, hd)), np.zeros((KVH, before + T)), np.zeros(KVH)
        for i in range(T):
            for h in range(H):
                m = before + i + 1
                p = np.exp(K[h, :m] @ x[i, h] / math.sqrt(hd))
                total = n + p.sum()
                want[i, h] = p @ V[h, :m] / total * gate[i, h]
                got[h, :m] += p / total
                empty[h] += 1 / total
        _close(out[mine].cpu(), torch.from_numpy(want.reshape(T, H * hd)), False, "out")
        added = w[1].double() - held.double()
        added[:, n + before:] = w[1, :, n + before:].double()
        for at in (0, 123_457, n - 1):
            assert np.allclose(added[:, at].cpu().numpy(), empty, rtol=1e-5), at
        _close((added[:, n:n + before + T]).cpu(), torch.from_numpy(got), False, "weights")
        rows += torch.tensor(counts, dtype=torch.int32, device="cuda")
        pos += torch.tensor(counts, dtype=torch.int32, device="cuda")
        before += T
    kk, vv = cache.read(rows - before, before, rows=rows)
    for x, y in (("k", kk), ("v", vv)):
        assert np.array_equal(y[1].cpu().numpy(), R.values(seq[x]).astype(f32).transpose(1, 0, 2))
    into = blk.new_cache(2, 3000)
    w = torch.rand(w.shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    kept, new_rows = blk.evict(cache, w, rows, into, 2500, 2, before)
    assert new_rows.tolist() == [9 + 8, 2500]
    for h in (0, KVH - 1):
        assert kept[1, h].tolist() == R.keep(w[1, h].cpu().numpy(), n + before, 2500, 2, before).tolist()
    a, b = into.read(torch.tensor([0, 2500 - before], dtype=torch.int32, device="cuda"), before, rows=new_rows)
    assert torch.equal(a[1], kk[1]) and torch.equal(b[1], vv[1])


@pytest.mark.parametrize("n,budget,sink,recent", [(49153, 20000, 3, 100), (120000, 119999, 0, 0), (120000, 50000, 1, 1), (60000, 5, 2, 3), (150000, 4096, 4, 512)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evictions_of_many_rows(n, budget, sink, recent, kind):
    torch = _torch()
    rng = np.random.default_rng(n + budget)
    KVH = 2
    w = np.exp(3 * rng.standard_normal((1, KVH, n))).astype(f32)
    if kind == "ties":  # most of the middle is one value, the rest above and below it
        w = np.where(rng.random(w.shape) < 0.8, f32(0.5), w).astype(f32)
    if kind == "odd":
        w *= np.where(rng.random(w.shape) < 0.5, f32(1), f32(-1))
        for value, share in ((0.0, 0.2), (-0.0, 0.2), (np.nan, 0.05), (np.inf, 0.01), (-np.inf, 0.01), (1e-42, 0.1)):
            w[rng.random(w.shape) < share] = value
    blk, _, _ = _block(KVH, KVH, 64, 0, n, 1)
    cache, into = blk.new_cache(1), blk.new_cache(1, budget)
    cache.data.random_(0, 59, generator=torch.Generator(device="cuda").manual_seed(n))  # finite as parameters
    rows = torch.tensor([n], dtype=torch.int32, device="cuda")
    nw = torch.empty((1, KVH, budget), device="cuda")
    print(f"evict {n} to {budget}, {kind}", flush=True)
    kept, new_rows = blk.evict(cache, torch.from_numpy(w).cuda(), rows, into, budget, sink, recent, new_weights=nw)
    assert new_rows.tolist() == [budget]
    k, v = cache.read(None, n)
    k2, v2 = into.read(None, budget)
    for h in range(KVH):
        # a NaN is below every number, also below -inf, which the oracle takes it for
        mine = np.where(np.isnan(w[0, h]), np.nan, np.maximum(w[0, h], np.finfo(f32).min))
        want = R.keep(mine, n, budget, sink, recent)
        assert np.array_equal(kept[0, h].cpu().numpy(), want), h
        at = torch.from_numpy(want).cuda()
        assert np.array_equal(nw[0, h].cpu().numpy(), w[0, h, want], equal_nan=True)
        assert torch.equal(k2[0, :, h], k[0, at, h]) and torch.equal(v2[0, :, h], v[0, at, h])


def test_two_captured_calls_share_a_workspace():
    """A prompt's call and a token's, each in a graph of its own, replayed in turn with eager calls between."""
    torch = _torch()
    H, KVH, hd = 16, 2, 256
    blk, _, _ = _block(H, KVH, hd, 64, 2000, 2)
    caches, weights = zip(*((c, blk.new_weights(c)) for c in (blk.new_cache(2) for _ in range(2))))
    k0, v0 = _random(1, (1400, KVH * hd), (1400, KVH * hd))
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    for c in caches:
        blk.append(k0, v0, c, start)
    ws = blk.new_workspace(caches[0], tokens=22, max_tokens=11, weights=True)
    calls, outs = [], []
    rows = [torch.full((2,), 700, dtype=torch.int32, device="cuda") for _ in range(2)]
    held = caches[0].data.clone()
    for T in (11, 1):
        q, k, v = _random(T, (2 * T, 2 * H * hd), (2 * T, KVH * hd), (2 * T, KVH * hd))
        calls.append((T, q, k, v))
        outs.append(torch.empty((2 * T, H * hd), device="cuda"))

    def run(i, which, out=None):
        T, q, k, v = calls[i]
        r = blk.prefill(q, k, v, caches[which], rows[which], ws, out=out, weights=weights[which])
        rows[which].add_(T)
        return r

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            run(i, 0, outs[i])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(i, 0, outs[i])
        graphs.append(g)
    caches[0].data.copy_(held)
    weights[0].zero_()
    rows[0].fill_(700)
    for turn in range(4):
        for i in (0, 1, 1):
            graphs[i].replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            want = run(i, 1)
            torch.cuda.synchronize()
            assert torch.equal(got, want), (turn, i)
    assert torch.equal(caches[0].data, caches[1].data) and torch.equal(*weights) and torch.equal(*rows)


def test_calls_on_another_stream():
    """Every call of the block and the cache with stream=, what it returns held by that stream."""
    torch = _torch()
    H, KVH, hd = 8, 2, 128
    blk, _, _ = _block(H, KVH, hd, 64, 900, 3)
    k0, v0, q, k, v = _random(4, (600, KVH * hd), (600, KVH * hd), (20, 2 * H * hd), (20, KVH * hd), (20, KVH * hd))
    side = torch.cuda.Stream()
    results = []
    for stream in (None, side):
        cache, into = blk.new_cache(2), blk.new_cache(2, 128)
        ws, w = blk.new_workspace(cache, tokens=20, max_tokens=10, weights=True), blk.new_weights(cache)
        rows = torch.zeros(2, dtype=torch.int32, device="cuda")
        after = rows + 300
        torch.cuda.synchronize()
        blk.append(k0, v0, cache, rows, stream=stream)
        out = blk.prefill(q, k, v, cache, after, ws, weights=w, stream=stream)
        one = blk.step(q[:2], k[:2], v[:2], cache, after, ws, weights=w, stream=stream)
        kept, new_rows = blk.evict(cache, w, after, into, 100, 3, 20, stream=stream)
        values = into.read(None, 100, rows=new_rows, stream=stream)
        torch.cuda.synchronize()
        results.append((out, one, kept, new_rows, *values, cache.data, into.data, w))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 33])
@pytest.mark.parametrize("given", ["f32", "bf16"])
def test_inputs_and_outputs_of_two_types(T, given):
    """f32 in and bf16 out, and the other way: the f32 call's result, rounded or not."""
    torch = _torch()
    a, b = (torch.float32, torch.bfloat16) if given == "f32" else (torch.bfloat16, torch.float32)
    H, KVH, hd = 8, 2, 256
    blk, _, _ = _block(H, KVH, hd, 64, 900, 4)
    cache = blk.new_cache(1)
    k0, v0, q, k, v = _random(T, (500, KVH * hd), (500, KVH * hd), (T, 2 * H * hd), (T, KVH * hd), (T, KVH * hd), dtype=a)
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k0, v0, cache, rows)
    rows += 500
    ws = blk.new_workspace(cache, tokens=T, max_tokens=T)
    out = blk.prefill(q, k, v, cache, rows, ws, out=torch.empty((T, H * hd), dtype=b, device="cuda"))
    held = cache.data.clone()
    want = blk.prefill(q.float(), k.float(), v.float(), cache, rows, ws)
    assert torch.equal(held, cache.data)  # bf16 values are f32 ones too
    if given == "bf16":
        assert torch.equal(out, want)
    else:
        assert torch.equal(out, want.bfloat16())


def test_tensors_of_the_host_are_refused():
    torch = _torch()
    H, KVH, hd = 4, 2, 64
    blk, _, _ = _block(H, KVH, hd, 16, 64, 5)
    cache, into = blk.new_cache(2), blk.new_cache(2, 32)
    q, k, v = _random(1, (2, 2 * H * hd), (2, KVH * hd), (2, KVH * hd))
    rows, w, ws = torch.zeros(2, dtype=torch.int32, device="cuda"), blk.new_weights(cache), blk.new_workspace(cache, weights=True)
    step = lambda q=q, k=k, v=v, cache=cache, rows=rows, ws=ws, **kw: blk.step(q, k, v, cache, rows, ws, **kw)  # noqa: E731
    host = Q4Cache(2, KVH, hd, 64, device="cpu")
    for call in (lambda: step(q=q.cpu()), lambda: step(k=k.cpu()), lambda: step(v=v.cpu()), lambda: step(rows=rows.cpu()),
                 lambda: step(ws=ws.cpu()), lambda: step(weights=w.cpu()), lambda: step(positions=rows.cpu()),
                 lambda: step(out=torch.empty((2, H * hd))), lambda: step(cache=host), lambda: host.read(None, 3),
                 lambda: blk.append(k, v, cache, rows.cpu()), lambda: blk.append(k.cpu(), v, cache, rows),
                 lambda: blk.append(k, v, cache, rows, starts=torch.tensor([0, 1, 2], dtype=torch.int32), max_tokens=1),
                 lambda: blk.evict(cache, w.cpu(), rows, into, 9), lambda: blk.evict(cache, w, rows.cpu(), into, 9),
                 lambda: blk.evict(cache, w, rows, host, 9), lambda: cache.read(rows.cpu(), 3), lambda: cache.read(None, 3, rows=rows.cpu()),
                 lambda: _block(H, KVH, hd, 16, 64, 5, torch.zeros(64, 8, 2))):
        with pytest.raises(_lib.SwqError) as e:
            call()
        assert e.value.code == _lib.SWQ_ERR_INVALID_ARGUMENT
    assert cache.read(None, 0)[0].shape == (2, 0, KVH, hd)  # no rows: nothing to do


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_stays_with_its_head(T, dtype, bad):
    """A query that is not finite makes its head's output NaN and no other's, nor the weights of another
    kv head; such a gate its dim's (a sigmoid of infinity is 0 or 1); rows behind the last token stay."""
    torch = _torch()
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    H, KVH, hd = 8, 2, 128
    blk, _, _ = _block(H, KVH, hd, 64, 400, 6)
    cache = blk.new_cache(1)
    k0, v0, q, k, v = _random(7, (300, KVH * hd), (300, KVH * hd), (T, 2 * H * hd), (T, KVH * hd), (T, KVH * hd), dtype=dt)
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k0, v0, cache, rows)
    rows += 300
    ws = blk.new_workspace(cache, tokens=T, max_tokens=T, weights=True)
    r = q.clone().view(T, H, 2, hd)
    r[T - 1, 2, 0, 77] = bad
    r[0, 5, 1, 3] = bad
    for weights in (False, True):
        outs, gathered = [], []
        for x in (q, r.view(T, -1)):
            w = blk.new_weights(cache) if weights else None
            out = torch.full((T + 1, H * hd), 7.0, dtype=dt, device="cuda")
            blk.prefill(x, k, v, cache, rows, ws, out=out[:T], weights=w)
            assert bool((out[T] == 7).all())
            outs.append(out[:T].float().view(T, H, hd))
            gathered.append(w)
        good, got = outs
        assert bool(got[T - 1, 2].isnan().all())
        at = got[0, 5, 3].item()
        assert math.isnan(at) if math.isnan(bad) else bool((at == 0) if bad < 0 else abs(at) >= abs(good[0, 5, 3].item()))
        got[T - 1, 2], got[0, 5, 3] = good[T - 1, 2], good[0, 5, 3]
        assert torch.equal(good, got)
        if weights:
            assert torch.equal(gathered[0][:, 1], gathered[1][:, 1])


@pytest.mark.parametrize("T", [1, 2, 9])
def test_a_padded_batch(T):
    """Room for many more tokens than the sequences bring: the queried workspace does, the rows behind
    the last sequence's stay as they are, in and out, and the results are those of the tight call."""
    torch = _torch()
    H, KVH, hd, room = 16, 2, 128, 3000
    blk, _, _ = _block(H, KVH, hd, 64, 20000, 8)
    results = []
    for N in (2 * T, room):
        cache = blk.new_cache(2)
        q, k, v = _random(9, (room, 2 * H * hd), (room, KVH * hd), (room, KVH * hd))
        rows = torch.zeros(2, dtype=torch.int32, device="cuda")
        k0, v0 = _random(10, (4000, KVH * hd), (4000, KVH * hd))
        blk.append(k0, v0, cache, rows)
        rows += 2000
        starts = torch.tensor([0, T, 2 * T], dtype=torch.int32, device="cuda")
        ws, w = blk.new_workspace(cache, tokens=N, max_tokens=T, weights=True), blk.new_weights(cache)
        out = torch.full((N, H * hd), 7.0, device="cuda")
        blk.prefill(q[:N], k[:N], v[:N], cache, rows, ws, starts=starts, max_tokens=T, out=out, weights=w)
        assert bool((out[2 * T:] == 7).all())
        results.append((out[:2 * T], w, cache.data))
    for i, (a, b) in enumerate(zip(*results)):
        if i == 2:
            assert torch.equal(a, b)
        else:  # the padded call may be split in another way
            assert bool(((a - b).abs() <= 2e-5 * a.abs().max()).all())


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 62), (128, 64), (128, 32), (256, 128), (256, 256), (256, 254)])
@pytest.mark.parametrize("n,T", [(0, 150), (900, 33)])
def test_every_kind_of_rotation_in_bf16(hd, rot, n, T):
    """bf16 prompts prepare their queries where they are used if the dims that turn together allow it."""
    torch = _torch()
    H, KVH = 6, 2
    blk, qw, _ = _block(H, KVH, hd, rot, n + T, rot + n)
    cache = blk.new_cache(1)
    k0, v0, k, v, q = _random(n + T, (n, KVH * hd), (n, KVH * hd), (T, KVH * hd), (T, KVH * hd), (T, 2 * H * hd), dtype=torch.bfloat16)
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    if n:
        blk.append(k0, v0, cache, rows)
    rows += n
    out = blk.prefill(q, k, v, cache, rows, blk.new_workspace(cache, tokens=T, max_tokens=T))
    kk, vv = cache.read(None, n + T)
    want, _ = _attend(*_queries(q, H, hd, qw, blk.rope_table.cpu().numpy()[n:n + T]), kk[0].double(), vv[0].double(), n)
    _close(out, want, True, f"{hd} {rot}")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_largest_values(hd, T, dtype):
    """Values at both ends of what the cache takes: 15 steps of a rounded scale do not pass f16's
    largest number, and attention over them is finite."""
    torch = _torch()
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    H, KVH, n = 4, 2, 70
    blk, qw, _ = _block(H, KVH, hd, 0, n + T, hd + T)
    cache = blk.new_cache(1)
    k, q, v = _random(hd, (n + T, KVH * hd), (T, 2 * H * hd), (n + T, KVH * hd))
    k, q, v = k.to(dt), q.to(dt), (v.sign() * 7e4).to(dt)
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k[:n], v[:n], cache, rows)
    rows += n
    ws, w = blk.new_workspace(cache, tokens=T, max_tokens=T, weights=True), blk.new_weights(cache)
    out = blk.prefill(q, k[n:], v[n:], cache, rows, ws)
    beside = blk.prefill(q, None, None, cache, rows, ws, weights=w)
    kk, vv = cache.read(None, n + T)
    assert 65300 < vv.max().item() <= 65504 and vv.min().item() == -65504
    want, _ = _attend(*_queries(q, H, hd, qw, np.zeros((T, 0, 2), f32)), kk[0].double(), vv[0].double(), n)
    _close(out, want, dtype == "bf16", "out")
    _close(beside, want, dtype == "bf16", "out beside weights")
