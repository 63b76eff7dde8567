"""Which tokens' k and v the rows' kernel loads, from the indexes that it computes (csrc/q4_cache.hpp), compiled for
the host: every one is a token of the call, also where a sequence that brings none is the last one."""

import ctypes
import itertools
import subprocess

import numpy as np
import pytest

from swiftlet_amd.build import CSRC, HIPCC

SOURCE = """
#include "q4_cache.hpp"
using namespace swq;
// Walks the blocks as q4_append does; loads[n]: loads of token n, index N for any other; stores[row]: tokens of row r, -1 else.
extern "C" int walk(int b, int B, int N, int max_tokens, const int32_t *starts, const int32_t *rows, int maxp, int step, int32_t *loads,
                    int32_t *stores) {
    Q4Batch d{};
    d.B = B;
    d.N = N;
    d.max_tokens = max_tokens;
    d.starts = starts;
    d.rows = rows;
    const Q4Rows w = d.written(b, maxp);
    int blocks = 0;
    for (int first = 0; first < step; ++first)
        for (int blk = w.block0() + first; blk < w.block_end(); blk += step, ++blocks)
            for (int row = blk * kQ4Block; row < (blk + 1) * kQ4Block; ++row) {
                const int n = w.token(row);
                ++loads[n >= 0 && n < N ? n : N];
                if (w.has(row)) {
                    if (row < 0 || row >= maxp || stores[row] != -1) return -1;
                    stores[row] = n;
                }
            }
    return blocks;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("q4_rows")
    (d / "rows.hip").write_text(SOURCE)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "rows.hip"), "-o",
                        str(d / "rows.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    fn = ctypes.CDLL(str(d / "rows.so")).walk
    P = ctypes.c_void_p
    fn.argtypes = [ctypes.c_int] * 4 + [P, P, ctypes.c_int, ctypes.c_int, P, P]

    def run(counts, before, maxp, step=1, starts=None):
        B = len(before)
        starts = np.cumsum([0, *counts]) if starts is None else starts
        starts, rows = np.asarray(starts, np.int32), np.asarray(before, np.int32)
        N = sum(counts)
        out = []
        for b in range(B):
            loads, stores = np.zeros(N + 1, np.int32), np.full(maxp, -1, np.int32)
            blocks = fn(b, B, N, max(counts), starts.ctypes.data, rows.ctypes.data, maxp, step, loads.ctypes.data, stores.ctypes.data)
            out.append((blocks, loads, stores))
        return out

    return run


@pytest.mark.parametrize("step", [1, 3])
def test_every_load_is_of_a_token_of_its_sequence(walk, step):
    for r0, r1, c0, c1 in itertools.product((0, 5, 8, 23, 39, 40, 50), (0, 1, 7, 8, 39, 40), (0, 1, 9), (0, 1, 20)):
        if c0 + c1 == 0:
            continue
        n0 = 0
        for (blocks, loads, stores), r, c in zip(walk([c0, c1], [r0, r1], 40, step), (r0, r1), (c0, c1)):
            new = max(0, min(r + c, 40) - min(r, 40))
            assert loads[c0 + c1] == 0, "a load behind the last token"
            assert loads.sum() == loads[n0:n0 + c].sum()
            assert (blocks == 0) == (new == 0)
            want = np.full(40, -1)
            want[min(r, 40):min(r, 40) + new] = n0 + np.arange(new)
            assert np.array_equal(stores, want)
            n0 += c


def test_starts_and_rows_out_of_range(walk):
    for starts in ([-3, 900, 2], [0, 24, 24], [24, 24, 24], [5, 3, 30]):
        for blocks, loads, _ in walk([20, 4], [-7, 63], 64, 1, starts):
            assert blocks >= 0 and loads[24] == 0, starts
