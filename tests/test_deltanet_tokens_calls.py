"""swq_deltanet_tokens without a GPU: sizes, and what it refuses before it touches a device."""

import ctypes

import pytest

from swiftlet_amd import _lib
from swiftlet_amd._lib import DeltaNetBatch, DeltaNetLayer

FAKE = 0x7F0000000000  # a well-aligned address; a refused call uses none
E = _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def layer(**kw):
    d = dict(num_key_heads=16, num_value_heads=32, key_head_dim=128, value_head_dim=128, conv_kernel=4, layout=0, norm_eps=1e-6, reserved=0,
             conv_weight=FAKE, a_log=FAKE, dt_bias=FAKE, norm_weight=FAKE)
    return DeltaNetLayer(**{**d, **kw})


def batch(**kw):
    d = dict(sequences=3, tokens=300, max_tokens=200, slots=5, starts=FAKE, positions=FAKE, slot=FAKE, qkvz_stride=0, ba_stride=0, reserved=0)
    return DeltaNetBatch(**{**d, **kw})


def call(lib, l, b, qkvz=FAKE, ba=FAKE, dtype=E.SWQ_BF16, states=FAKE, n=1 << 40, out=FAKE, out_dtype=E.SWQ_BF16, ws=FAKE, m=1 << 40):
    return lib.swq_deltanet_tokens(ctypes.byref(l), ctypes.byref(b), qkvz, ba, dtype, states, n, out, out_dtype, ws, m, None)


def test_slot_bytes(lib):
    l = layer()
    n = lib.swq_deltanet_slot_bytes(ctypes.byref(l))
    assert n == 4 * 8192 * 4 + 32 * 128 * 128 * 4 == lib.swq_deltanet_state_bytes(ctypes.byref(l))
    odd = layer(num_key_heads=1, num_value_heads=1, key_head_dim=8, value_head_dim=5)
    assert lib.swq_deltanet_slot_bytes(ctypes.byref(odd)) == 512 + 256 and lib.swq_deltanet_state_bytes(ctypes.byref(odd)) == 512 + 160
    assert lib.swq_deltanet_slot_bytes(ctypes.byref(layer(key_head_dim=12))) == 0


LAYERS = [(dict(num_value_heads=31), E.SWQ_ERR_BAD_SHAPE), (dict(key_head_dim=48), E.SWQ_ERR_LIMIT), (dict(value_head_dim=1025), E.SWQ_ERR_LIMIT),
          (dict(conv_kernel=9), E.SWQ_ERR_LIMIT), (dict(conv_kernel=0), E.SWQ_ERR_BAD_SHAPE), (dict(layout=2), E.SWQ_ERR_INVALID_ARGUMENT),
          (dict(norm_eps=float("nan")), E.SWQ_ERR_INVALID_ARGUMENT), (dict(a_log=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(reserved=1), E.SWQ_ERR_INVALID_ARGUMENT)]
BATCHES = [(dict(sequences=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(tokens=-1), E.SWQ_ERR_INVALID_ARGUMENT), (dict(slots=0), E.SWQ_ERR_INVALID_ARGUMENT),
           (dict(max_tokens=0), E.SWQ_ERR_BAD_SHAPE), (dict(max_tokens=-5), E.SWQ_ERR_BAD_SHAPE), (dict(starts=None, tokens=301), E.SWQ_ERR_BAD_SHAPE),
           (dict(slot=None, slots=2), E.SWQ_ERR_BAD_SHAPE), (dict(qkvz_stride=12287), E.SWQ_ERR_BAD_SHAPE), (dict(qkvz_stride=-1), E.SWQ_ERR_INVALID_ARGUMENT),
           (dict(ba_stride=63), E.SWQ_ERR_BAD_SHAPE), (dict(ba_stride=-64), E.SWQ_ERR_INVALID_ARGUMENT), (dict(reserved=1), E.SWQ_ERR_INVALID_ARGUMENT),
           (dict(sequences=1 << 20, tokens=1 << 20, slots=1 << 20), E.SWQ_ERR_LIMIT)]


@pytest.mark.parametrize("change,want", LAYERS, ids=str)
def test_layers(lib, change, want):
    assert call(lib, layer(**change), batch()) == want
    assert lib.swq_deltanet_tokens_workspace_bytes(ctypes.byref(layer(**change)), ctypes.byref(batch())) == 0


@pytest.mark.parametrize("change,want", BATCHES, ids=str)
def test_batches(lib, change, want):
    assert call(lib, layer(), batch(**change)) == want
    assert lib.swq_deltanet_tokens_workspace_bytes(ctypes.byref(layer()), ctypes.byref(batch(**change))) == 0


@pytest.mark.parametrize("change,want", [
    (dict(qkvz=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(ba=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(states=None), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(out=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(dtype=E.SWQ_F16), E.SWQ_ERR_UNSUPPORTED_DTYPE), (dict(out_dtype=7), E.SWQ_ERR_UNSUPPORTED_DTYPE),
    (dict(qkvz=FAKE + 1), E.SWQ_ERR_MISALIGNED), (dict(ba=FAKE + 2, dtype=E.SWQ_F32), E.SWQ_ERR_MISALIGNED), (dict(out=FAKE + 1), E.SWQ_ERR_MISALIGNED),
    (dict(states=FAKE + 16), E.SWQ_ERR_MISALIGNED), (dict(ws=FAKE + 16), E.SWQ_ERR_MISALIGNED), (dict(ws=None), E.SWQ_ERR_WORKSPACE),
    (dict(m=255), E.SWQ_ERR_WORKSPACE), (dict(n=5 * 2228224 - 1), E.SWQ_ERR_WORKSPACE)], ids=str)
def test_pointers_and_sizes(lib, change, want):
    assert call(lib, layer(), batch(), **change) == want


def test_positions_are_wanted(lib):
    assert call(lib, layer(), batch(positions=None)) == E.SWQ_ERR_INVALID_ARGUMENT


def test_no_tokens_need_nothing(lib):
    assert call(lib, layer(), batch(tokens=0), qkvz=None, ba=None, states=None, out=None, ws=None, n=0, m=0) == E.SWQ_OK


@pytest.mark.parametrize("heads", [(16, 32, 128, 128), (4, 8, 64, 64), (1, 1, 8, 5)], ids=str)
def test_a_workspace_for_more_serves_fewer(lib, heads):
    l = layer(num_key_heads=heads[0], num_value_heads=heads[1], key_head_dim=heads[2], value_head_dim=heads[3])
    size = lambda **kw: lib.swq_deltanet_tokens_workspace_bytes(ctypes.byref(l), ctypes.byref(batch(slots=100, **kw)))  # noqa: E731
    last = {}
    for most in (1, 2, 64, 65, 5000):
        for B in (1, 2, 63, 64, 100):
            for n in (1, 63, 64, 65, 1000, 100000):
                got = size(sequences=B, tokens=n, max_tokens=most)
                assert got >= 256 and got % 256 == 0
                for low in ((m, b, t) for m, b, t in last if m <= most and b <= B and t <= n):
                    assert last[low] <= got, (low, most, B, n)
                last[most, B, n] = got
    # equal lengths without starts need no more than with them
    assert size(sequences=4, tokens=400, max_tokens=1, starts=None) <= size(sequences=4, tokens=400, max_tokens=100)
