"""The 4-bit cache's calls at the ends of what they accept, against the oracle in 64 bits; bars as in
test_gpu_attention_q4.py where no other is derived beside the test."""

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from swiftlet_amd.attention_q4 import AttentionQ4GPU
from tests.test_gpu_attention_q4 import Setup, _close, _torch, _types
from tests.test_gpu_attention_q4_long import _attend, _block, _queries, _random
from tests.test_oracle_attention_q4_range import near_the_top

pytestmark = pytest.mark.gpu

f32 = np.float32


@pytest.mark.parametrize("hd,KVH", [(64, 8), (128, 2), (256, 2)])
@pytest.mark.parametrize("before,counts", [([0, 5], [20, 0]), ([3, 39, 7], [0, 9, 0]), ([13, 2, 1], [1, 0, 0]), ([5, 40, 33], [0, 0, 2])])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sequences_that_bring_nothing(hd, KVH, before, counts, dtype):
    """First, in the middle and last, their rows filling a block of 8 or not; k and v are the front of larger
    tensors, whose rest is NaN."""
    torch = _torch()
    H, N = 2 * KVH, sum(counts)
    s = Setup(hd + N, H, KVH, hd, 32, before, 70)
    q, k, v = s.tokens(counts, _types()[dtype])
    k, v = (torch.cat([x, torch.full_like(x[:1].expand(9, -1), float("nan"))])[:N] for x in (k, v))
    ws = s.blk.new_workspace(s.cache, tokens=N, max_tokens=max(counts))
    print(f"{before} + {counts}, hd {hd}", flush=True)
    held = s.cache.data.clone()
    s.blk.append(k, v, s.cache, s.rows(), starts=s.starts(counts), max_tokens=max(counts))
    want, _ = s.expect(counts)
    s.check_cache()
    s.cache.data.copy_(held)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, starts=s.starts(counts), max_tokens=max(counts))
    _close(out, want, dtype)
    s.check_cache()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("before,T,most", [(0, 2, 1), (0, 2, 2), (1, 2, 2), (0, 2, 3), (2, 5, 3), (1, 2, 3), (0, 4, 4), (3, 20, 4), (5, 3, 7)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("weights", [False, True])
def test_prompts_over_the_smallest_caches(hd, before, T, most, dtype, weights):
    """Caches of a few rows, with room for the tokens or not: those past the last row see all of them."""
    torch = _torch()
    H, KVH = 4, 2
    s = Setup(hd + most + T, H, KVH, hd, 16, [before], most)
    q, k, v = s.tokens([T], _types()[dtype])
    ws = s.blk.new_workspace(s.cache, tokens=T, max_tokens=T, weights=weights)
    ws.fill_(255)
    w = torch.full((1, KVH, most), 0.25, device="cuda") if weights else None
    print(f"{before} + {T} of {most} rows, hd {hd}", flush=True)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, weights=w)
    new = min(T, most - before)
    turns = s.table[np.minimum(np.arange(before, before + new), most - 1)]
    s.seqs[0] = R.append(s.seqs[0], *(x[:new].reshape(new, KVH, hd) for x in (s.k, s.v)), s.kw, 1e-6, turns)
    want, got = s.expect([T], appended=False)
    _close(out, want, dtype)
    s.check_cache()
    if weights:
        got[0][:, :before] += 0.25
        w, n = w[0].cpu().numpy(), before + new
        assert np.abs(w[:, :n] - got[0]).max() <= 1e-5 * max(1.0, got[0].max()) and (w[:, n:] == 0.25).all()


@pytest.mark.parametrize("dtype,weights", [("bf16", False), ("bf16", True), ("f32", False)])
def test_many_sequences_without_their_longest(dtype, weights):
    """max_tokens left out is that of all tokens, as much as 8 M workgroups for a tile each; lengths mixed or alike,
    the same bits as with the longest given."""
    torch = _torch()
    H, KVH, hd, B, most = 32, 8, 64, 1024, 64
    blk = AttentionQ4GPU(H, KVH, hd, 64, 1e6, 1e-6, 2 * most, np.ones(hd, f32), np.ones(hd, f32))
    g = torch.Generator(device="cuda").manual_seed(3)
    for counts in ([32] * B, [most if b % 3 == 0 else b % 7 for b in range(B)]):
        N = sum(counts)
        q, k, v = (torch.randn((N, n), generator=g, device="cuda").to(_types()[dtype]) for n in (2 * H * hd, KVH * hd, KVH * hd))
        rows = torch.arange(B, dtype=torch.int32, device="cuda") % most
        starts = torch.tensor(np.cumsum([0, *counts]), dtype=torch.int32, device="cuda")
        got = []
        for longest in (max(counts), None):
            print(f"{N} tokens, longest {longest}", flush=True)
            cache = blk.new_cache(B, 2 * most)
            w = blk.new_weights(cache) if weights else None
            ws = blk.new_workspace(cache, tokens=N, max_tokens=longest or N, weights=weights)
            out = blk.prefill(q, k, v, cache, rows, ws, starts=starts, max_tokens=longest, weights=w)
            got.append((out, cache.data, w))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and (not weights or torch.equal(got[0][2], got[1][2]))
        assert bool(got[1][0].isfinite().all()) and bool(got[1][0].any())


# Single tokens in f32 whose splits are long.  A sum over a split adds 32 rows at a time, twice (p * scale is two
# numbers), on two or four accumulators: 33,000 rows are 2 * 33,000 / 32 / 2 = 1,031 additions, each off by half a unit
# in the last place at most, 2^-25 of the running sum, of either sign: 32 * 2^-25 = 1e-6 of it for all, as one standard
# deviation at most; the largest of a few hundred outputs is off by three times that at most.  A running sum of signed terms
# is about the size of the outputs.  Scores, off by some 3e-7 of either sign each, add a part of that: 64 * 2^-24 = 3.8e-6.
LONG = 64 * 2.0 ** -24


@pytest.mark.parametrize("H,KVH,hd,n", [(8, 2, 64, 33000), (4, 2, 128, 20011), (16, 2, 256, 33000)])
@pytest.mark.parametrize("weights", [False, True])
def test_long_splits_keep_their_precision(H, KVH, hd, n, weights):
    """A hint of few rows leaves a long sequence to one split."""
    torch = _torch()
    blk, qw, _ = _block(H, KVH, hd, 0, n + 1, n)
    cache = blk.new_cache(1)
    k0, v0, k, v, q = _random(n, (n, KVH * hd), (n, KVH * hd), (1, KVH * hd), (1, KVH * hd), (1, 2 * H * hd))
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k0, v0, cache, rows)
    rows += n
    w = blk.new_weights(cache) if weights else None
    out = blk.step(q, k, v, cache, rows, blk.new_workspace(cache, weights=weights), weights=w, max_rows=64)
    kk, vv = cache.read(None, n + 1)
    want, got = _attend(*_queries(q, H, hd, qw, np.zeros((1, 0, 2), f32)), kk[0].double(), vv[0].double(), n)
    off = ((out.double() - want).abs().max() / want.abs().max()).item()
    print(f"{n} rows of {hd}: off by {off:.1e}", flush=True)
    assert off <= LONG
    if weights:
        assert (w[0].double() - got).abs().max() <= 1e-5 * got.max()


@pytest.mark.parametrize("H,KVH,hd", [(8, 2, 64), (16, 2, 256)])
@pytest.mark.parametrize("T", [3, 130])
@pytest.mark.parametrize("sharp", [1, 6])
def test_prompts_of_one_long_split(H, KVH, hd, T, sharp):
    """As above for several tokens: three products a tile of 32 rows are 3,093 additions to one accumulator, each off by
    2^-24 of it at most, evenly spread: one standard deviation is sqrt(3093 / 3) * 2^-24 = 1.9e-6, the largest of
    some thousand outputs four of them, 7.7e-6, and 2e-6 of sums of weights and scores make 1e-5."""
    torch = _torch()
    n = 33000
    blk, qw, _ = _block(H, KVH, hd, 0, n + T, n)
    blk.q_norm.mul_(sharp)
    cache = blk.new_cache(1)
    k0, v0, k, v, q = _random(n + T, (n, KVH * hd), (n, KVH * hd), (T, KVH * hd), (T, KVH * hd), (T, 2 * H * hd))
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    blk.append(k0, v0, cache, rows)
    rows += n
    out = blk.prefill(q, k, v, cache, rows, blk.new_workspace(cache, tokens=T, max_tokens=T), max_rows=64)
    kk, vv = cache.read(None, n + T)
    want, _ = _attend(*_queries(q, H, hd, qw * f32(sharp), np.zeros((T, 0, 2), f32)), kk[0].double(), vv[0].double(), n)
    off = ((out.double() - want).abs().max() / want.abs().max()).item()
    print(f"{T} tokens of {hd}: off by {off:.1e}", flush=True)
    assert off <= 1e-5


def test_a_wide_batch_in_f32_keeps_its_precision():
    """32 sequences of up to 16,383 rows of 8 heads: splits of 2,048 rows."""
    torch = _torch()
    B, H, KVH, hd, n = 32, 16, 8, 64, 16383
    blk, qw, _ = _block(H, KVH, hd, 0, n + 1, 7)
    cache = blk.new_cache(B)
    k0, v0 = _random(8, (B * n, KVH * hd), (B * n, KVH * hd))
    blk.append(k0, v0, cache, torch.zeros(B, dtype=torch.int32, device="cuda"))
    del k0, v0
    k, v, q = _random(9, (B, KVH * hd), (B, KVH * hd), (B, 2 * H * hd))
    rows = torch.tensor([n - 400 * b for b in range(B)], dtype=torch.int32, device="cuda")
    out = blk.step(q, k, v, cache, rows, blk.new_workspace(cache))
    for b in (0, 1, 17, B - 1):
        m = n - 400 * b
        first = torch.zeros(B, dtype=torch.int32, device="cuda")
        kk, vv = (x[b, :m + 1].double() for x in cache.read(first, m + 1))
        want, _ = _attend(*_queries(q[b:b + 1], H, hd, qw, np.zeros((1, 0, 2), f32)), kk, vv, m)
        off = ((out[b:b + 1].double() - want).abs().max() / want.abs().max()).item()
        print(f"sequence {b}, {m} rows: off by {off:.1e}", flush=True)
        assert off <= LONG, b


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 40])
def test_values_up_to_the_largest_number(hd, T):
    """Groups whose bias rounds up next to f16's largest number: rows as the oracle's, bit for bit, none of their values
    past it, and finite attention; by the call for rows alone and by that of a single token."""
    torch = _torch()
    H, KVH, n = 2, 1, 41
    s = Setup(hd + T, H, KVH, hd, 0, [0, 0], n)
    x = near_the_top(2 * n * (hd // 64), hd).reshape(2, n, hd).astype(f32)
    x[1] = -x[1]  # the bias is -65504 there
    x[0, 3, :64] = np.linspace(65462.25, 65504, 64)
    rows = s.rows()
    ws = s.blk.new_workspace(s.cache, tokens=2 * T, max_tokens=T)
    for t in range(0, n - T + 1, T):
        q, k, _ = s.tokens([T, T], torch.float32)
        s.v = x[:, t:t + T].reshape(2 * T, hd)
        v = torch.from_numpy(s.v).cuda()
        out = s.blk.prefill(q, k, v, s.cache, rows, ws)
        assert bool(out.isfinite().all()) and out.abs().max() <= 65504
        assert bool(s.blk.prefill(q.bfloat16(), None, None, s.cache, rows, ws).isfinite().all())
        s.expect([T, T], attend=False)
        s.before = [b + T for b in s.before]
        rows = s.rows()
    s.check_cache()
    _, vv = s.cache.read(None, n, rows=rows)
    assert vv.max() <= 65504 and vv.min() >= -65504
