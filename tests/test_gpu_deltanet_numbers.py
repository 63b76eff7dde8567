"""What the DeltaNet block over many tokens keeps of its numbers (swq_deltanet_tokens), whatever their types and sizes.

Bars.  The same prompt with f32 and with bf16 outputs: the same numbers, rounded once, so bit for bit.  Numbers of mixed
size: an output is a sum whose terms' size the oracle has, and a product's two factors are off by 2^-24 each, their
low parts' product of 2^-24 is left out: 3 * 2^-24 a product, five in a row (k.k to T, T k to W, W S to d, P d, each sum's
own rounding): 15 * 2^-24 = 9e-7 of its terms rms.  A row of a head is a sum over 64 columns or more, its error at most ten
times that, 1e-5, also swq_deltanet_step's bar; so is a head's state, over its own size."""

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


@pytest.mark.parametrize("most", [23, 24])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_both_sides_of_where_many_go_in_chunks(most, dtype):
    c = Batch(BIG, [most, 1, 5, 4, 2, 0, 18, 12, 13], dtype, split=True, seed=36)
    close(c, c.run())


def close(c, out):
    """Every row of every head over the size of its terms, every head's state over its own size."""
    want, _, rec = c.oracle()
    got = c.views()[1].double()
    nv, dv = c.heads[1], c.heads[3]
    rows = lambda t: t.reshape(len(out), nv, dv).norm(dim=-1)  # noqa: E731
    err = rows(out.double() - want)
    if out.dtype == torch.bfloat16:
        err = (err - rows(want) * 2.0 ** -8).clamp_min(0)
    err = float((err / rows(c.terms).clamp_min(1e-300)).max())
    state = max(float(((got[j] - rec[j]).flatten(1).norm(dim=1) / rec[j].flatten(1).norm(dim=1)).max()) for j in c.slots.tolist())
    print(f"rows {err:.2e} state {state:.2e}", flush=True)
    assert err < 1e-5 and state < 1e-5


def value_row(c, n, by):
    """Token n's values (of every head) `by` times what they were."""
    nk, nv, dk, dv = c.heads
    assert c.split
    c.qkvz[n, 2 * nk * dk:2 * nk * dk + nv * dv] *= by


@pytest.mark.parametrize("by", [1e3, 1e5, 1e6])
@pytest.mark.parametrize("at", [0, 20, 100, 255])
@pytest.mark.parametrize("decay", [None, 3.0], ids=["slow", "fast"])
@pytest.mark.parametrize("lengths", [[256], [256, 70]], ids=str)
def test_one_large_value_row(lengths, decay, at, by):
    """The first token, one in the middle of a chunk, one of a later chunk, the last: rows before it are as good as without,
    and rows after it once it has faded."""
    c = Batch(SMALL, lengths, split=True, seed=31, decay=decay)
    value_row(c, at, by)
    close(c, c.run())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [BIG, WIDE], ids=str)
def test_one_large_value_row_of_larger_heads(heads, dtype):
    c = Batch(heads, [150, 90], dtype, split=True, seed=32, decay=2.0)
    value_row(c, 70, 1e4)
    value_row(c, 239, 1e5)
    close(c, c.run())


@pytest.mark.parametrize("lengths", [[2048, 3], [2100]], ids=str)
def test_a_large_row_at_the_end_of_a_long_prompt(lengths):
    c = Batch((1, 2, 64, 64), lengths, split=True, seed=35)
    value_row(c, lengths[0] - 1, 1e5)
    close(c, c.run())


@pytest.mark.parametrize("by", [1e3, 1e5])
@pytest.mark.parametrize("lengths", [[200], [130, 70]], ids=str)
def test_a_large_state_that_fades(lengths, by):
    c = Batch(SMALL, lengths, seed=33, decay=3.0)
    c.views()[1].mul_(by)
    c.before.copy_(c.states)
    close(c, c.run())


def test_heads_of_different_sizes():
    """The values and states of each head at a size of its own, from 1e-12 to 1e9."""
    c = Batch(SMALL, [150, 70], split=True, seed=34)
    nk, nv, dk, dv = c.heads
    size = 10.0 ** torch.linspace(-12, 9, nv, device="cuda")
    c.qkvz[:, 2 * nk * dk:2 * nk * dk + nv * dv] *= size.repeat_interleave(dv)
    ring, rec = c.views()
    ring[:, :, 2 * nk * dk:] *= size.repeat_interleave(dv)
    rec *= size[:, None, None]
    c.before.copy_(c.states)
    close(c, c.run())
