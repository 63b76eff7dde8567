"""Infinities and NaN among what the DeltaNet block over many tokens takes (swq_deltanet_tokens): the tokens before them, the
other heads and the other sequences keep their bits; from that token on the head's outputs are not finite where
swq_deltanet_step's are not, and neither is its state.  Lengths on both sides of where a prompt goes in chunks."""

import pytest
import torch

from tests.deltanet_cases import Batch

pytestmark = pytest.mark.gpu

SMALL, BIG = (2, 4, 64, 64), (16, 32, 128, 128)
INF, NAN = float("inf"), float("nan")


def steps(c, b, states):
    """Sequence b by swq_deltanet_step, from and into a copy of its state in `states`."""
    n, j = c.block.slot_bytes, int(c.slots[b])
    state = states[j * n:(j + 1) * n]
    rows = range(int(c.starts[b]), int(c.starts[b + 1]))
    return torch.stack([c.block.step(c.qkvz[t].float().contiguous(), c.ba[t].float().contiguous(), state, int(c.positions[b]) + i) for i, t in enumerate(rows)])


def same(c, spoil, at, head, first):
    """Spoils the call's inputs and holds it against itself without: `head` of sequence 0 changes from token `first` (of
    the sequence) on, and where swq_deltanet_step is finite there and where it is not."""
    nv, dv = c.heads[1], c.heads[3]
    want = c.run()
    states = c.states.clone()
    c.states.copy_(c.before)
    spoil()
    start = c.states.clone()
    got = c.run()
    stepped = start.clone()
    by_step = steps(c, 0, stepped)
    heads = lambda t: t.reshape(len(t), nv, dv)  # noqa: E731
    live = torch.ones_like(heads(want), dtype=torch.bool)
    live[first:c.lengths[0], head] = False
    assert torch.equal(heads(got)[live], heads(want)[live])
    T = c.lengths[0]
    assert torch.equal(heads(got)[first:T, head].isfinite(), heads(by_step)[first:T, head].isfinite())
    j = int(c.slots[0])
    others = torch.ones(c.views()[1].shape[:2], dtype=torch.bool)
    others[j, head] = False
    rec, before = c.views()[1], c.block.states_views(states)[1]
    assert torch.equal(rec[others], before[others])
    by_step_rec = c.block.states_views(stepped)[1][j, head]
    # a row of the state that the steps leave finite may be NaN here: its head gives nothing finite any more
    assert not bool((rec[j, head].isfinite() & ~by_step_rec.isfinite()).any())
    if bool(by_step_rec.isfinite().all()):
        assert bool(rec[j, head].isfinite().all())
    assert torch.equal(c.views()[0][j].nan_to_num(7.0), c.block.states_views(stepped)[0][j].nan_to_num(7.0))


LENGTHS = [[11], [12], [40], [64], [150], [2100], [150, 20, 1]]


@pytest.mark.parametrize("what", ["a", "b", "a_log", "dt_bias"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_a_gate_that_is_no_number_is_not_hidden(lengths, what):
    """From its token on the head's outputs and its state are no numbers either; other heads and sequences keep their bits."""
    c = Batch(SMALL, lengths, split=True, seed=40)
    want = c.run().reshape(-1, 4, 64)
    states = c.views()[1].clone()
    c.states.copy_(c.before)
    T, at, j = lengths[0], min(9, lengths[0] - 1), int(c.slots[0])
    if what in ("a", "b"):
        c.ba[at, (4 if what == "a" else 0) + 2] = NAN
        got = c.run().reshape(-1, 4, 64)
        assert torch.equal(got[T:], want[T:])
    else:
        at = 0
        getattr(c.block, what)[2] = NAN
        got = c.run().reshape(-1, 4, 64)
    assert not bool(got[at:T, 2].isfinite().any())
    assert not bool(c.views()[1][j, 2].isfinite().any())
    others = torch.tensor([True, True, False, True])
    assert torch.equal(got[:, others], want[:, others]) and torch.equal(c.views()[1][:, others], states[:, others])


@pytest.mark.parametrize("what", ["a", "b"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_gates(lengths, what):
    c = Batch(SMALL, lengths, split=True, seed=41)
    at = min(9, lengths[0] - 1)

    def spoil():
        c.ba[at, (4 if what == "a" else 0) + 2] = NAN

    same(c, spoil, at, 2, at)


@pytest.mark.parametrize("at", [0, 63, 64, 100, 149])
@pytest.mark.parametrize("what", ["a", "b"])
def test_gates_anywhere(what, at):
    c = Batch(SMALL, [150, 20], split=True, seed=42)

    def spoil():
        c.ba[at, (4 if what == "a" else 0) + 1] = NAN

    same(c, spoil, at, 1, at)


@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("what", ["a", "b"])
def test_gates_that_saturate(what, value):
    """Infinite gates are decays of 0 or 1 and writes of nothing or everything: all stays finite, as in the steps."""
    c = Batch(SMALL, [150], split=True, seed=43)
    c.ba[40, (4 if what == "a" else 0) + 1] = value
    start = c.states.clone()
    got, want = c.run(), steps(c, 0, start)
    assert bool(got.isfinite().all()) and float((got - want).abs().max() / want.abs().max()) < 1e-5
    j = int(c.slots[0])
    a, b = c.views()[1][j], c.block.states_views(start)[1][j]
    assert float((a - b).abs().max() / b.abs().max()) < 1e-5


@pytest.mark.parametrize("which", ["a_log", "dt_bias"])
def test_parameters(which):
    c = Batch(SMALL, [150], split=True, seed=44)

    def spoil():
        getattr(c.block, which)[3] = NAN

    same(c, spoil, 0, 3, 0)


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("at", [0, 5, 30, 63, 64, 130, 149])
def test_values(at, value):
    """One value of head 1."""
    c = Batch(SMALL, [150, 20], split=True, seed=45)

    def spoil():
        c.qkvz[at, 2 * 128 + 64 + 9] = value

    same(c, spoil, at, 1, at)


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_values_of_prompts_of_any_length(lengths):
    c = Batch(SMALL, lengths, split=True, seed=46)
    at = min(9, lengths[0] - 1)

    def spoil():
        c.qkvz[at, 2 * 128 + 2 * 64 + 33] = INF

    same(c, spoil, at, 2, at)


def of_key_head(c, channel, at, value):
    """An element of key head 1's queries (channel < 64) or keys: both of its value heads, one after the other."""
    for head in (2, 3):
        nv, dv = c.heads[1], c.heads[3]
        c.states.copy_(c.before)
        clean = c.qkvz.clone()
        want = c.run().reshape(-1, nv, dv)
        states = c.views()[1].clone()
        c.states.copy_(c.before)
        c.qkvz[at, 64 + channel if channel < 64 else 128 + channel] = value
        start = c.states.clone()
        got = c.run().reshape(-1, nv, dv)
        by_step = steps(c, 0, start).reshape(-1, nv, dv)
        T = c.lengths[0]
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[T:], want[T:])
        assert torch.equal(got[:, :2], want[:, :2])
        assert torch.equal(got[at:T, head].isfinite(), by_step[at:T, head].isfinite())
        j = int(c.slots[0])
        a, b = c.views()[1][j, head], c.block.states_views(start)[1][j, head]
        assert torch.equal(a.isfinite(), b.isfinite())
        assert torch.equal(c.views()[1][j, :2], states[j, :2])
        c.qkvz.copy_(clean)


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("at", [0, 30, 63, 64, 149])
def test_keys(at, value):
    of_key_head(Batch(SMALL, [150, 20], split=True, seed=47), 64 + 7, at, value)


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("at", [0, 30, 63, 64, 140])
@pytest.mark.parametrize("K", [1, 2, 3, 4, 6])
def test_queries(at, value, K):
    """A query is of its own token and of the K - 1 after it, whose convolution it is in."""
    of_key_head(Batch(SMALL, [150, 20], split=True, seed=48, K=K), 7, at, value)


@pytest.mark.parametrize("K", [1, 2, 3, 6])
def test_queries_token_after_token(K):
    of_key_head(Batch(SMALL, [10, 3], split=True, seed=49, K=K), 7, 4, NAN)


@pytest.mark.parametrize("heads", [SMALL, BIG, (1, 2, 128, 256)], ids=str)
@pytest.mark.parametrize("value", [INF, NAN])
def test_states(heads, value):
    """An element of one head's state: that head's outputs, and of its state that row."""
    c = Batch(heads, [150], split=True, seed=50)
    want = c.run().reshape(150, heads[1], heads[3])
    states = c.views()[1].clone()
    c.states.copy_(c.before)
    j = int(c.slots[0])
    c.views()[1][j, 1, 5, 3] = value
    got = c.run().reshape(150, heads[1], heads[3])
    rec = c.views()[1]
    assert not bool(got[:, 1].isfinite().any())
    others = torch.arange(heads[1]) != 1
    assert torch.equal(got[:, others], want[:, others]) and torch.equal(rec[j, others], states[j, others])
    rows = torch.arange(heads[3]) != 5
    assert not bool(rec[j, 1, 5].isfinite().any())
    assert torch.equal(rec[j, 1, rows], states[j, 1, rows])


@pytest.mark.parametrize("split", [False, True], ids=["interleaved", "split"])
def test_a_ring_that_is_not_finite(split):
    """Rows of tokens before the call: from its first token on."""
    c = Batch(SMALL, [100, 70], split=split, seed=51)
    want = c.run().reshape(170, 4, 64)
    c.states.copy_(c.before)
    j = int(c.slots[0])
    c.views()[0][j, :, 2 * 128 + 64 + 3] = NAN  # value head 1
    got = c.run().reshape(170, 4, 64)
    others = torch.tensor([True, False, True, True])
    assert torch.equal(got[:, others], want[:, others]) and torch.equal(got[100:], want[100:])
    assert not bool(got[:100, 1].isfinite().any())


@pytest.mark.parametrize("heads", [SMALL, BIG], ids=str)
def test_captured(heads):
    """What a replay leaves in the workspace spoils no later one."""
    c = Batch(heads, [150, 40], split=True, seed=52)
    clean = c.qkvz.clone()
    out = torch.empty_like(c.run())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out)
    nk, nv, dk, dv = heads
    for at in (None, 70, None, 3, None):
        c.qkvz.copy_(clean)
        if at is not None:
            c.qkvz[at, 2 * nk * dk + 5] = NAN
            c.qkvz[at + 1, nk * dk + 5] = INF
        c.states.copy_(c.before)
        want, states = c.run(), c.states.clone()
        c.states.copy_(c.before)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), at
        assert torch.equal(c.states, states), at
        assert bool(out.isfinite().all()) == (at is None)
