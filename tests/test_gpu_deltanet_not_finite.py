"""Infinities and NaN among what the DeltaNet block over many tokens takes (swq_deltanet_tokens).  Lengths on both sides of
where a prompt goes in chunks."""

import pytest
import torch

from tests.deltanet_cases import Batch

pytestmark = pytest.mark.gpu

SMALL = (2, 4, 64, 64)
NAN = float("nan")
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
