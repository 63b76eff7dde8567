"""What the DeltaNet block over many tokens keeps of its numbers (swq_deltanet_tokens), whatever their types and sizes.

Bars.  The same prompt with f32 and with bf16 outputs: the same numbers, rounded once, so bit for bit."""

import pytest
import torch

from tests.deltanet_cases import Batch

pytestmark = pytest.mark.gpu

BIG, SMALL, WIDE = (16, 32, 128, 128), (4, 8, 64, 64), (2, 8, 128, 64)


@pytest.mark.parametrize("heads,lengths", [(BIG, [12]), (BIG, [77]), (BIG, [64, 65, 1, 129, 0, 63]), (SMALL, [2100]), (SMALL, [200, 3, 16, 17]), (WIDE, [31, 1, 130]),
                                           ((1, 2, 128, 256), [70, 90]), ((1, 1, 128, 16), [4, 70])], ids=str)
def test_bf16_outputs_are_the_f32_ones_rounded(heads, lengths):
    c = Batch(heads, lengths, "bf16", seed=len(lengths))
    narrow = c.run()
    states = c.states.clone()
    c.states.copy_(c.before)
    wide = c.run(out=torch.empty(narrow.shape, device="cuda"))
    assert torch.equal(narrow, wide.bfloat16())
    assert torch.equal(c.states, states)
