"""How prompts over a 4-bit cache are cut into workgroups (csrc/attention_q4_prefill.hip's plan, called on the host): what
no launch takes is not asked for, whatever a call gives as the most tokens of one sequence."""

import ctypes
import itertools
import subprocess

import pytest

from swiftlet_amd import _lib
from swiftlet_amd.build import CSRC, HIPCC, LIB

SOURCE = """
#include "attention_q4.hpp"
using namespace swq;
extern "C" void plan(int64_t max_tokens, int64_t tokens, int64_t rows, int64_t sequences, int64_t kvh, int group, int hd, int maxp, int f32,
                     int weights, int64_t *out) {
    const Q4PrefillPlan p = plan_q4_prefill(max_tokens, tokens * kvh * group, rows, sequences * kvh, group, hd, 64, maxp, f32, weights);
    out[0] = p.rows_per;
    out[1] = p.tiles;
    out[2] = p.splits;
    out[3] = p.gparts;
}
extern "C" int64_t workgroups(int64_t most, int64_t heads, int64_t work) { return q4_workgroups(most, heads, work); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    _lib.load()  # built if it is not there
    d = tmp_path_factory.mktemp("q4_plans")
    (d / "plans.hip").write_text(SOURCE)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plans.hip"),
                        f"-Wl,{LIB},-rpath,{LIB.parent}", "-o", str(d / "plans.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = ctypes.CDLL(str(d / "plans.so"))
    L = ctypes.c_int64
    lib.plan.argtypes = [L] * 5 + [ctypes.c_int] * 5 + [ctypes.c_void_p]
    lib.workgroups.argtypes, lib.workgroups.restype = [L] * 3, L
    return lib


def _plan(host, *args):
    out = (ctypes.c_int64 * 4)()
    host.plan(*args, out)
    return list(out)


def _up(a, b):
    return -(-a // b)


# sequences, kv heads, query heads of one, head size, tokens of all sequences
BATCHES = [(1, 2, 8, 256, 4096), (4, 8, 4, 128, 2500), (256, 8, 4, 64, 131072), (1024, 8, 4, 64, 32768), (1, 8, 16, 128, 1 << 20), (8191, 8, 1, 64, 1 << 22),
           (65535, 1, 16, 64, 65536 * 4), (5, 8, 8, 128, 70001)]


@pytest.mark.parametrize("B,kvh,group,hd,tokens", BATCHES)
@pytest.mark.parametrize("f32,weights", [(0, 0), (1, 0), (0, 1)])
def test_launches_stay_in_their_limits(host, B, kvh, group, hd, tokens, f32, weights):
    """A launch has fewer than 2^32 work-items a dimension; workgroups have at most 512."""
    for most, rows in itertools.product((_up(tokens, B), tokens), (1, 300, 40000)):
        per, tiles, splits, gparts = _plan(host, most, tokens, rows, B, kvh, group, hd, 40000, f32, weights)
        groups = tiles * splits * B * kvh
        assert tiles >= 1 and splits >= 1 and gparts >= weights
        assert groups * 512 < 2 ** 32, (most, rows)
        # mostly with work: at most 4 times the tiles that all sequences together can have, or few
        if splits == 1:
            assert groups <= max(1 << 16, 4 * (tokens * group * kvh // per + B * kvh))


@pytest.mark.parametrize("B,kvh,group,hd,tokens", BATCHES)
def test_like_lengths_have_a_workgroup_a_tile(host, B, kvh, group, hd, tokens):
    most = _up(tokens, B)
    per, tiles, _, _ = _plan(host, most, tokens, 1000, B, kvh, group, hd, 40000, 0, 0)
    assert tiles == _up(most * group, per)


def test_workgroups_of_launches_that_go_round(host):
    assert host.workgroups(10, 16, 160) == 10
    assert host.workgroups(1, 65535, 0) == 1
    assert host.workgroups(10 ** 6, 1, 5) == 1 << 16
    assert host.workgroups(16385, 2048, 131072 + 4096) == 4 * (131072 + 4096) // 2048
