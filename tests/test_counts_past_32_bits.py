"""Counts of more than 32 bits at the Python entry points of swq_deltanet_tokens and swq_rope_table: refused or as large as
they are, never cut to their low bits."""

import pytest
import torch

from swiftlet_amd import _lib
from swiftlet_amd._lib import SWQ_DELTA_SPLIT
from swiftlet_amd.deltanet import DeltaNetGPU
from swiftlet_amd.rope import RopeGPU

WRAPS = 2 ** 32 + 5


def block():
    return DeltaNetGPU(1, 2, 64, 64, 4, SWQ_DELTA_SPLIT, 1e-6, torch.zeros(256 * 4), torch.zeros(2), torch.zeros(2), torch.ones(64), device="cpu")


def test_more_tokens_of_a_sequence_than_there_are():
    b = block()
    assert b.new_batch_workspace(2, 100, WRAPS).numel() == b.new_batch_workspace(2, 100, 100).numel() == b.new_batch_workspace(2, 100).numel()
    assert b.new_batch_workspace(2, 100, 2 ** 40).numel() == b.new_batch_workspace(2, 100).numel()
    assert b.new_batch_workspace(2, 100, 1).numel() == 256


@pytest.mark.parametrize("args", [(WRAPS, 100), (2, WRAPS), (WRAPS,)], ids=str)
def test_workspaces(args):
    with pytest.raises(_lib.SwqError) as e:
        block().new_batch_workspace(*args)
    assert e.value.code == _lib.SWQ_ERR_LIMIT


@pytest.mark.parametrize("count", [WRAPS, 2 ** 31])
def test_rows_of_a_table(count):
    out = torch.empty((count, 32, 2), device="meta")
    for kw in ({}, {"out": out}):
        with pytest.raises(_lib.SwqError) as e:
            RopeGPU(64, 1e6, device="meta").table(count=count, **kw)
        assert e.value.code == _lib.SWQ_ERR_LIMIT
