"""Evictions whose outputs lie over their inputs are refused before anything is launched: one head's selection would
write what another's still reads."""

import ctypes

import pytest

from swiftlet_amd import _lib
from tests.test_attention_q4_calls import FAKE, cache, lib  # noqa: F401

FAR = FAKE + (1 << 32)


@pytest.mark.parametrize("output", ["new_weights", "new_rows", "kept"])
def test_outputs_over_inputs(lib, output):  # noqa: F811
    B, KVH, n, most, budget = 3, 2, 100, 60, 50
    src, dst = cache(lib), cache(lib, data=FAR, max_positions=most)
    size = {"new_weights": B * KVH * most * 4, "new_rows": B * 4, "kept": B * KVH * budget * 4}[output]
    weights, rows = FAKE + (1 << 34), FAKE + (1 << 35)
    for start, length in ((weights, B * KVH * n * 4), (rows, B * 4)):
        for at in (start, start + 4, start + length - 4, start - 4, start + 4 - size):
            out = {"new_weights": None, "new_rows": FAKE + (1 << 36), "kept": FAKE + (1 << 37), output: at}
            got = lib.swq_q4_evict(ctypes.byref(src), B, weights, rows, ctypes.byref(dst), budget, 4, 8, out["new_weights"], out["new_rows"],
                                   out["kept"], None)
            assert got == _lib.SWQ_ERR_INVALID_ARGUMENT, (output, at - start)
