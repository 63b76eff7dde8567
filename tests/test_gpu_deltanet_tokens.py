"""The gated DeltaNet block over the tokens of many sequences (swq_deltanet_tokens) against the 64-bit oracle
(oracle/deltanet_tokens_ref.py).

Bars.  f32 outputs and states: 1e-5 of the largest, as for swq_deltanet_step.  Rings: the inputs bit for bit.  bf16
outputs: their rounding, 2^-8 of the value, and 2^-9 of the size of what an output is the sum of beside it (the oracle's
`terms`).  Products of a prompt may take queries, keys, states, P and d rounded to f16: a product's two factors are off
by at most 2^-12 each, 2e-4 rms of it together; five times that, 2^-10, covers the largest of some 10^6 sums of independent
errors, and twice as much sums whose terms are few."""

import pytest
import torch

from tests.deltanet_cases import Batch, bf16_off, off

pytestmark = pytest.mark.gpu

BIG, SMALL, WIDE = (16, 32, 128, 128), (4, 8, 64, 64), (2, 8, 128, 64)


def check(c, out, **kw):
    want, ring, rec = c.oracle(**kw)
    got_ring, got_rec = c.views()
    assert torch.equal(got_ring.double(), ring)
    print(f"state {off(got_rec, rec):.2e}", flush=True)
    assert off(got_rec, rec) < 1e-5
    if not len(want):
        return
    err = off(out, want) if out.dtype == torch.float32 else bf16_off(c, out, want)
    print(f"out {err:.2e}", flush=True)
    assert err < (1e-5 if out.dtype == torch.float32 else 2.0 ** -9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("split", [False, True], ids=["interleaved", "split"])
@pytest.mark.parametrize("heads,lengths", [(BIG, [1]), (BIG, [5, 1, 0, 2]), (BIG, [77]), (BIG, [64, 65, 1, 129, 0, 63]), (SMALL, [200, 3, 16, 17]),
                                           (WIDE, [31, 1, 130]), ((3, 3, 64, 128), [100, 1]), ((1, 1, 128, 16), [1, 70])], ids=str)
def test_tokens(heads, lengths, split, dtype):
    c = Batch(heads, lengths, dtype, split, seed=len(lengths))
    check(c, c.run())


@pytest.mark.parametrize("K", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("heads", [(2, 4, 8, 5), (1, 3, 16, 16), (2, 2, 32, 24), (1, 2, 256, 1000), (2, 4, 64, 64), (1, 2, 128, 144)], ids=str)
def test_other_heads_and_kernels(heads, K):
    c = Batch(heads, [1, 0, 2, 40, 7, 90], "f32", K % 2 == 0, K=K, seed=K)
    check(c, c.run())


@pytest.mark.parametrize("heads", [BIG, SMALL, (2, 4, 8, 5)], ids=str)
@pytest.mark.parametrize("B", [1, 5])
def test_single_tokens_are_the_steps(heads, B):
    """One token of each sequence: swq_deltanet_step's outputs and states, within 1e-5 of the largest.  Both sum the
    same products in the same order, but which product of a sum enters an fma unrounded is the compiler's choice: a
    lane's dk / 4 terms and two exchanges are off by (dk / 4 + 2) 2^-24 of the sum of absolute terms, 2e-6 at dk 128,
    and that sum is about sqrt(dk) / 6 times the largest of the outputs: 4e-6."""
    c = Batch(heads, [1] * B, seed=3)
    states = c.states.clone()
    out = c.block.step_batch(c.qkvz, c.ba, c.states, c.positions, c.ws, slots=c.slots)
    n = c.block.slot_bytes
    for b in range(B):
        j = int(c.slots[b])
        y = c.block.step(c.qkvz[b].contiguous(), c.ba[b].contiguous(), states[j * n:(j + 1) * n], int(c.positions[b]))
        assert off(y, out[b].double()) < 1e-5, b
    for a, b in zip(c.block.states_views(states), c.views()):
        assert off(a, b.double()) < 1e-5
    assert torch.equal(c.block.states_views(states)[0], c.views()[0])


@pytest.mark.parametrize("heads", [BIG, (2, 4, 8, 5)], ids=str)
def test_a_prompt_in_pieces(heads):
    """A sequence in one call, and the same in pieces with the position going on."""
    c = Batch(heads, [210], seed=9)
    whole = c.run()
    rec = c.views()[1].clone()
    c.states.copy_(c.before)
    parts, at = [], 0
    for n in (64, 1, 100, 3, 42):
        pos = c.positions + at
        parts.append(c.block.prefill(c.qkvz[at:at + n], c.ba[at:at + n], c.states, pos, c.ws, slots=c.slots))
        at += n
    assert off(torch.cat(parts), whole.double()) < 1e-5
    assert off(c.views()[1], rec.double()) < 1e-5
    check(c, torch.cat(parts))


def test_what_is_left_out_stays():
    """Sequences without tokens or without a slot, slots of nobody and rows behind the last sequence."""
    c = Batch(BIG, [70, 0, 3, 66, 1], "bf16", seed=4, spare=3)
    used = c.slots.clone()
    for dead, value in ((3, -1), (2, c.slots.numel() + 3)):
        c.slots[dead] = value
    rows = torch.cat([c.qkvz, c.qkvz[:5]]), torch.cat([c.ba, c.ba[:5]])
    out = torch.full((len(rows[0]), c.val), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = c.block.new_batch_workspace(5, len(rows[0]))
    c.block.prefill(*rows, c.states, c.positions, ws, starts=c.starts, slots=c.slots, max_tokens=70, out=out)
    assert bool((out[70:139] == 7).all()) and bool((out[140:] == 7).all())
    want, ring, rec = c.oracle(left_out=(2, 3))
    got_ring, got_rec = c.views()
    n = c.block.slot_bytes
    for j in range(8):
        if j not in (int(used[0]), int(used[4])):
            assert torch.equal(c.states[j * n:(j + 1) * n], c.before[j * n:(j + 1) * n]), j
    assert torch.equal(got_ring.double(), ring) and off(got_rec, rec) < 1e-5
    live = list(range(70)) + [139]
    assert bf16_off(c, out[:140], want, live) < 2.0 ** -9


@pytest.mark.parametrize("lengths,most", [([90, 3, 70], 64), ([5, 2], 3), ([4, 1, 9], 1)])
def test_no_more_than_max_tokens(lengths, most):
    c = Batch(SMALL, lengths, seed=5)
    out = torch.zeros((sum(lengths), c.val), device="cuda")
    c.run(max_tokens=most, out=out)
    check(c, out, lengths=[min(n, most) for n in lengths])


@pytest.mark.parametrize("heads", [BIG, (2, 4, 8, 5)], ids=str)
@pytest.mark.parametrize("spread", [1, 8, 24])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_apart(heads, spread, dtype):
    c = Batch(heads, [80, 2], dtype, seed=6, spread=spread)
    check(c, c.run())


def test_equal_lengths_without_starts():
    c = Batch(SMALL, [70, 70, 70], seed=7)
    check(c, c.run(starts=None, max_tokens=None))


@pytest.mark.parametrize("dtype,out_dtype", [("f32", torch.bfloat16), ("bf16", torch.float32)])
def test_types_mixed(dtype, out_dtype):
    c = Batch(WIDE, [100, 1], dtype, seed=8)
    out = torch.empty((101, c.val), dtype=out_dtype, device="cuda")
    check(c, c.run(out=out))


@pytest.mark.parametrize("heads", [BIG, SMALL], ids=str)
@pytest.mark.parametrize("lengths,dtype", [([77], "f32"), ([64], "f32"), ([1000], "bf16"), ([300, 5], "bf16")], ids=str)
def test_states_and_f32_outputs_keep_22_bits(heads, lengths, dtype):
    """In the 2-norm.  Factors of products are off by 2^-23, their low parts' product of 2^-24 is left out: 2.5 * 2^-23
    a product; a state comes through four in a row (k.k to T, T k to W, W S to d, k d): 10 * 2^-23 = 1.2e-6 at most, and an
    output through one more at its side."""
    c = Batch(heads, lengths, dtype, seed=27)
    out = c.run()
    want, _, rec = c.oracle()
    norm = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    for j in c.slots.tolist():
        print(f"state {norm(c.views()[1][j], rec[j]):.2e}", flush=True)
        assert norm(c.views()[1][j], rec[j]) < 1.2e-6
    if dtype == "f32":
        assert norm(out, want) < 1.5e-6


@pytest.mark.parametrize("decay", [-12.0, 3.0, 6.0, 100.0])
def test_decays(decay):
    """From heads that forget next to nothing to heads that forget everything at once."""
    c = Batch(SMALL, [150, 3], seed=10, decay=decay)
    check(c, c.run())


@pytest.mark.parametrize("size", [1e-4, 300.0, 1e7])
def test_sizes_of_values(size):
    """Values and states far from 1, also beyond what 16 bits hold."""
    c = Batch(SMALL, [150, 3], seed=11, size=size)
    check(c, c.run())


@pytest.mark.parametrize("lengths", [[64, 4, 5, 0, 3, 12, 1, 2, 11, 13], [4, 4, 12], [11, 11, 3], [19, 1, 5, 4, 2, 0, 18, 12, 13], [20, 1, 5, 4, 2, 0, 18, 12, 13]], ids=str)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_short_ones_beside_long_ones(lengths, dtype):
    c = Batch(BIG, lengths, dtype, seed=18, K=3)
    check(c, c.run())


@pytest.mark.parametrize("heads,tokens,most", [(SMALL, 2048, None), (SMALL, 2049, None), (SMALL, 4160, None), (SMALL, 6200, 4100), ((1, 2, 128, 16), 5000, None)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_long_prompt(heads, tokens, most, dtype):
    """A prompt alone passes through the workspace 2,048 tokens at a time."""
    c = Batch(heads, [tokens], dtype, seed=tokens)
    out = torch.full((tokens, c.val), 7.0, dtype=c.dtype, device="cuda")
    c.run(max_tokens=most or tokens, out=out)
    assert bool((out[most or tokens:] == 7).all())
    if most:
        out[most:] = 0
    check(c, out, lengths=[most or tokens])


def test_one_long_prompt_captured():
    c = Batch(SMALL, [4500], "bf16", True, seed=19)
    out = torch.empty((4500, c.val), dtype=torch.bfloat16, device="cuda")
    c.run(out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out)
    for n in (4500, 2100, 30, 4500):  # of the captured call's tokens
        c.starts[1] = n
        c.states.copy_(c.before)
        want = c.run(out=torch.empty_like(out))[:n].clone()
        states = c.states.clone()
        c.states.copy_(c.before)
        c.ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:n], want) and torch.equal(c.states, states), n
    check(c, out)


def test_long():
    c = Batch(SMALL, [2500, 1, 700], "bf16", True, seed=12)
    check(c, c.run())


def test_the_same_call_gives_the_same_bits():
    c = Batch(BIG, [130, 1, 64], "bf16", seed=13)
    first = c.run()
    states = c.states.clone()
    for _ in range(3):
        c.states.copy_(c.before)
        c.ws.fill_(255)
        assert torch.equal(c.run(), first) and torch.equal(c.states, states)


@pytest.mark.parametrize("lengths", [[1, 1, 1], [70, 1, 5]])
def test_captured_and_replayed(lengths):
    """A captured call follows what its device arrays hold, with eager calls between the replays."""
    c = Batch(SMALL, lengths, seed=14)
    out = torch.empty((sum(lengths), c.val), device="cuda")
    c.run(out=out)
    c.states.copy_(c.before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out)
    for step in range(3):
        c.states.copy_(c.before)
        c.positions.add_(step)
        c.slots.copy_(c.slots.flip(0))
        c.qkvz.mul_(0.9)
        want = c.run()
        states = c.states.clone()
        c.states.copy_(c.before)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(c.states, states), step
    check(c, out)


def test_on_another_stream():
    c = Batch(SMALL, [70, 1], seed=15)
    want = c.run()
    states = c.states.clone()
    c.states.copy_(c.before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = c.run(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and torch.equal(c.states, states)


def test_a_workspace_for_more_serves_fewer():
    c = Batch(BIG, [70, 200, 1], "bf16", seed=16)
    ws = c.block.new_batch_workspace(9, 5000, 4096)
    want = c.run()
    states = c.states.clone()
    c.states.copy_(c.before)
    assert torch.equal(c.block.prefill(c.qkvz, c.ba, c.states, c.positions, ws, starts=c.starts, slots=c.slots, max_tokens=200), want)
    assert torch.equal(c.states, states)


def test_what_is_not_finite_stays_with_its_head():
    """An infinity and a NaN in one value head's inputs: the other heads and sequences are as without."""
    c = Batch((2, 4, 64, 64), [100, 70], split=True, seed=17)
    want = c.run()
    states = c.states.clone()
    c.states.copy_(c.before)
    c.qkvz[30, 2 * 128 + 64 + 5] = float("inf")   # value head 1, token 30 of sequence 0
    c.qkvz[31, 2 * 128 + 64 + 9] = float("nan")
    got = c.run()
    live = torch.ones_like(want, dtype=torch.bool)
    live[:100, 64:128] = False
    assert torch.equal(got[live], want[live])
    a, b = c.block.states_views(states)[1], c.views()[1]
    a[int(c.slots[0]), 1] = b[int(c.slots[0]), 1] = 0
    assert torch.equal(a, b)


def test_two_captured_calls_share_a_workspace():
    """Two calls in graphs of their own, one after another on a stream, in the same workspace."""
    a, b = Batch(SMALL, [130, 2], seed=20), Batch(SMALL, [2, 70], seed=21)
    wants = []
    for c in (a, b):
        wants.append((c.run(), c.states.clone()))
        c.states.copy_(c.before)
    ws = a.block.new_batch_workspace(2, 132)
    outs, graphs = [torch.empty_like(w[0]) for w in wants], []
    torch.cuda.synchronize()
    for c, out in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.block.prefill(c.qkvz, c.ba, c.states, c.positions, ws, starts=c.starts, slots=c.slots, max_tokens=max(c.lengths), out=out)
        graphs.append(graph)
    for _ in range(3):
        for c, graph in zip((a, b), graphs):
            c.states.copy_(c.before)
            graph.replay()
        torch.cuda.synchronize()
        for c, out, (want, states) in zip((a, b), outs, wants):
            assert torch.equal(out, want) and torch.equal(c.states, states)
            out.zero_()


def test_two_streams_with_workspaces_of_their_own():
    cs = [Batch(SMALL, [300, 5, 1], "bf16", seed=22 + i) for i in range(2)]
    wants = []
    for c in cs:
        wants.append((c.run(), c.states.clone()))
        c.states.copy_(c.before)
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [c.run(stream=s) for c, s in zip(cs, streams)]
        torch.cuda.synchronize()
        for c, out, (want, states) in zip(cs, outs, wants):
            assert torch.equal(out, want) and torch.equal(c.states, states)
            c.states.copy_(c.before)
        torch.cuda.synchronize()


@pytest.mark.parametrize("split", [False, True], ids=["interleaved", "split"])
def test_rows_that_no_wide_load_fits(split):
    """Projections that start off a multiple of 8 bytes and outputs likewise: token after token, the same results."""
    c = Batch(SMALL, [90, 2], "bf16", split, seed=24)
    wide = torch.empty(c.qkvz.numel() + 1, dtype=torch.bfloat16, device="cuda")
    rows = wide[1:].view(c.qkvz.shape)
    rows.copy_(c.qkvz)
    out = torch.empty(92 * c.val + 1, dtype=torch.bfloat16, device="cuda")[1:].view(92, c.val)
    c.qkvz = rows
    check(c, c.run(out=out))


def test_starts_that_do_not_rise():
    """Nor end with the rows; slots of nobody, positions below 0: taken as no tokens or as 0, nothing out of bounds."""
    c = Batch(SMALL, [70, 20, 30], seed=25)
    c.starts.copy_(torch.tensor([-5, 90, 20, 4000], dtype=torch.int32))
    c.positions.copy_(torch.tensor([-7, 3, 2 ** 31 - 1], dtype=torch.int32))
    c.slots[1] = -2 ** 31
    out = c.run(max_tokens=120)
    assert bool(torch.isfinite(out).all())
    n = c.block.slot_bytes
    used = {int(c.slots[0]), int(c.slots[2])}
    for j in range(5):
        if j not in used:
            assert torch.equal(c.states[j * n:(j + 1) * n], c.before[j * n:(j + 1) * n])


def test_refusals_in_python():
    from swiftlet_amd._lib import SwqError
    c = Batch(SMALL, [70, 1], seed=26)
    good = dict(qkvz=c.qkvz, ba=c.ba, states=c.states, positions=c.positions, ws=c.ws, starts=c.starts, slots=c.slots, max_tokens=70)
    y = torch.empty((71, c.val), device="cuda")
    for kw in (dict(qkvz=c.qkvz.half()), dict(qkvz=c.qkvz.bfloat16()), dict(qkvz=c.qkvz[:, :-1]), dict(qkvz=c.qkvz.cpu()), dict(qkvz=c.qkvz[:70]), dict(ba=c.ba[:70]),
               dict(ba=c.ba[:, :-1]), dict(ba=c.ba.cpu()), dict(states=c.states.float()), dict(states=c.states.cpu()),
               dict(states=c.states[:c.block.slot_bytes - 1]), dict(positions=c.positions.long()), dict(positions=c.positions.cpu()), dict(ws=c.ws[:256]), dict(ws=c.ws.cpu()),
               dict(ws=c.ws[1:]), dict(starts=c.starts[:2]), dict(starts=c.starts.long()), dict(slots=c.slots[:1]), dict(slots=c.slots.cpu()),
               dict(starts=None), dict(max_tokens=-1), dict(out=y[:70]), dict(out=y.half()), dict(out=y.cpu())):
        with pytest.raises(SwqError):
            c.block.prefill(**{**good, **kw})
    torch.cuda.synchronize()
    assert torch.equal(c.states, c.before)


def test_offsets_past_32_bits():
    """A prompt of more than 2^31 elements: the bits of the same in two calls, whose second begins with a span of its own;
    states more than 4 GB apart."""
    c = Batch(BIG, [16], "bf16", seed=28)
    T, cut, slots = 180000, 86 * 2048, 2100
    assert T * (c.conv + c.val) > 2 ** 31 and (slots - 1) * c.block.slot_bytes > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(29)
    qkvz = torch.randn((4500, c.conv + c.val), generator=g, device="cuda").bfloat16().repeat(T // 4500, 1)
    ba = torch.randn((T, 64), generator=g, device="cuda").bfloat16()
    states = torch.zeros(slots * c.block.slot_bytes, dtype=torch.uint8, device="cuda")
    last, first = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (slots - 1, 0))
    ws, at = c.block.new_batch_workspace(1, T), torch.zeros(1, dtype=torch.int32, device="cuda")
    whole = c.block.prefill(qkvz, ba, states, at, ws, slots=last)
    parts = [c.block.prefill(qkvz[:cut], ba[:cut], states, at, ws, slots=first), c.block.prefill(qkvz[cut:], ba[cut:], states, at + cut, ws, slots=first)]
    assert torch.equal(whole[:cut], parts[0]) and torch.equal(whole[cut:], parts[1])
    n = c.block.slot_bytes
    assert torch.equal(states[:n], states[-n:]) and bool(states[:n].any())
    assert not bool(states[n:2 * n].any()) and not bool(states[-2 * n:-n].any())
    one = c.block.step_batch(qkvz[-1:], ba[-1:], states, at + T, ws, slots=last)
    assert torch.equal(one, c.block.step_batch(qkvz[-1:], ba[-1:], states, at + T, ws, slots=first))
    rows = qkvz[[0, T - 1]]
    far = qkvz.as_strided(rows.shape, ((T - 1) * rows.shape[1], 1))
    states[-n:].copy_(states[:n])
    assert torch.equal(c.block.prefill(far, ba[:2], states, at, ws, slots=last), c.block.prefill(rows, ba[:2], states, at, ws, slots=first))
    assert torch.equal(states[:n], states[-n:])


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_more_sequences_than_lanes(B):
    c = Batch((1, 2, 64, 32), [(37 * i) % 90 if i % 7 else 0 for i in range(B)], "f32", True, seed=B)
    check(c, c.run())
