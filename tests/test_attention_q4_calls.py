"""The 4-bit cache's entry points without a GPU: sizes, and what they refuse before they touch a device."""

import ctypes

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from swiftlet_amd import _lib
from swiftlet_amd._lib import AttentionLayer, Q4Batch, Q4CacheDesc

FAKE = 0x7F0000000000  # a well-aligned address; a refused call uses none


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def layer(**kw):
    d = dict(num_heads=16, num_kv_heads=2, head_dim=256, rotary_dims=64, rope_theta=1e7, norm_eps=1e-6, max_positions=1,
             reserved=0, q_norm_weight=FAKE, k_norm_weight=FAKE)
    return AttentionLayer(**{**d, **kw})


def cache(lib, **kw):
    d = dict(data=FAKE, sequences=3, num_kv_heads=2, head_dim=256, max_positions=100)
    d.update(kw)
    n = lib.swq_q4_cache_bytes(d["sequences"], d["num_kv_heads"], d["head_dim"], d["max_positions"])
    return Q4CacheDesc(**{"bytes": n, **d})


def batch(**kw):
    d = dict(sequences=3, tokens=3, max_tokens=1, max_rows=0, starts=None, rows=FAKE, positions=None, rope=FAKE,
             rope_positions=200, reserved=0)
    return Q4Batch(**{**d, **kw})


def test_cache_bytes(lib):
    # k and v codes, and 4 x f16 per 64 dims, of rows rounded up to 32; parts padded to 256 bytes
    assert lib.swq_q4_cache_bytes(3, 2, 256, 100) == 3 * 2 * 128 * (256 + 4 * 4 * 2)
    assert lib.swq_q4_cache_bytes(1, 1, 64, 1) == 32 * (64 + 8)
    big = lib.swq_q4_cache_bytes(64, 8, 128, 1 << 20)
    assert big == 64 * 8 * (1 << 20) * 144
    for bad in ((0, 2, 256, 9), (1, 0, 256, 9), (1, 2, 96, 9), (1, 2, 256, 0), (1, 2, 32, 9), (1 << 14, 4, 64, 9), (1, 1, 64, (1 << 30) + 1)):
        assert lib.swq_q4_cache_bytes(*bad) == 0, bad


def test_rope_table_is_the_steps(lib):
    out = np.empty((5, 16, 2), np.float32)
    assert lib.swq_q4_rope_table(32, 1e6, 7, 5, out.ctypes.data) == 0
    assert np.array_equal(out, R.rope_table(12, 32, 1e6)[7:])
    for bad, want in (((3, 1e6, 0, 5), _lib.SWQ_ERR_BAD_SHAPE), ((0, 1e6, 0, 5), _lib.SWQ_ERR_BAD_SHAPE),
                      ((32, 0.0, 0, 5), _lib.SWQ_ERR_INVALID_ARGUMENT), ((32, 1e6, -1, 5), _lib.SWQ_ERR_INVALID_ARGUMENT),
                      ((32, 1e6, 0, 0), _lib.SWQ_ERR_INVALID_ARGUMENT)):
        assert lib.swq_q4_rope_table(*bad, out.ctypes.data) == want, bad
    assert lib.swq_q4_rope_table(32, 1e6, 0, 5, None) == _lib.SWQ_ERR_INVALID_ARGUMENT


E = _lib
LAYERS = [(dict(num_heads=15), E.SWQ_ERR_BAD_SHAPE), (dict(num_heads=34), E.SWQ_ERR_LIMIT), (dict(rotary_dims=3), E.SWQ_ERR_BAD_SHAPE),
          (dict(rotary_dims=258), E.SWQ_ERR_BAD_SHAPE), (dict(reserved=1), E.SWQ_ERR_INVALID_ARGUMENT), (dict(num_kv_heads=0), E.SWQ_ERR_BAD_SHAPE),
          (dict(q_norm_weight=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(k_norm_weight=None), E.SWQ_ERR_INVALID_ARGUMENT),
          (dict(head_dim=32, rotary_dims=0), E.SWQ_ERR_LIMIT), (dict(norm_eps=float("nan")), E.SWQ_ERR_INVALID_ARGUMENT),
          (dict(num_kv_heads=4), E.SWQ_ERR_BAD_SHAPE), (dict(head_dim=128), E.SWQ_ERR_BAD_SHAPE)]
CACHES = [(dict(data=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(data=FAKE + 16), E.SWQ_ERR_MISALIGNED), (dict(bytes=1000), E.SWQ_ERR_WORKSPACE),
          (dict(head_dim=48), E.SWQ_ERR_LIMIT), (dict(sequences=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(max_positions=-1), E.SWQ_ERR_INVALID_ARGUMENT)]
BATCHES = [(dict(sequences=4, tokens=4), E.SWQ_ERR_BAD_SHAPE), (dict(sequences=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(tokens=4), E.SWQ_ERR_BAD_SHAPE),
           (dict(tokens=-3), E.SWQ_ERR_INVALID_ARGUMENT), (dict(starts=FAKE, max_tokens=0), E.SWQ_ERR_BAD_SHAPE), (dict(rows=None), E.SWQ_ERR_INVALID_ARGUMENT),
           (dict(rope=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(rope_positions=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(max_rows=-1), E.SWQ_ERR_INVALID_ARGUMENT),
           (dict(reserved=1), E.SWQ_ERR_INVALID_ARGUMENT), (dict(rope=FAKE + 4), E.SWQ_ERR_MISALIGNED)]


def _append(lib, l, c, b, k=FAKE, v=FAKE, dtype=E.SWQ_F32):
    return lib.swq_q4_append(ctypes.byref(l), ctypes.byref(c), ctypes.byref(b), k, v, dtype, None)


def _attend(lib, l, c, b, q=FAKE, k=FAKE, v=FAKE, dtype=E.SWQ_F32, w=None, out=FAKE, out_dtype=E.SWQ_F32, ws=FAKE, n=1 << 40):
    return lib.swq_attention_q4(ctypes.byref(l), ctypes.byref(c), ctypes.byref(b), q, k, v, dtype, w, out, out_dtype, ws, n, None)


@pytest.mark.parametrize("call", [_append, _attend])
def test_refused_layers_caches_and_batches(lib, call):
    for kw, want in LAYERS:
        assert call(lib, layer(**kw), cache(lib), batch()) == want, kw
    for kw, want in CACHES:
        assert call(lib, layer(), cache(lib, **kw), batch()) == want, kw
    for kw, want in BATCHES:
        assert call(lib, layer(), cache(lib), batch(**kw)) == want, kw
    assert call(lib, layer(), cache(lib), batch(), dtype=E.SWQ_F16) == E.SWQ_ERR_UNSUPPORTED_DTYPE
    assert call(lib, layer(), cache(lib), batch(), k=None) == E.SWQ_ERR_INVALID_ARGUMENT
    assert call(lib, layer(), cache(lib), batch(), v=FAKE + 2) == E.SWQ_ERR_MISALIGNED
    assert call(lib, layer(), cache(lib), batch(tokens=0)) == E.SWQ_OK  # nothing to do


def test_refused_attention_arguments(lib):
    l, c, b = layer(), cache(lib), batch()
    n = lib.swq_attention_q4_workspace_bytes(ctypes.byref(l), ctypes.byref(c), ctypes.byref(b), 0)
    assert n > 0
    for kw, want in ((dict(q=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(out=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(out_dtype=1), E.SWQ_ERR_UNSUPPORTED_DTYPE),
                     (dict(ws=None), E.SWQ_ERR_WORKSPACE), (dict(n=n - 1), E.SWQ_ERR_WORKSPACE), (dict(ws=FAKE + 128), E.SWQ_ERR_MISALIGNED),
                     (dict(q=FAKE + 1), E.SWQ_ERR_MISALIGNED), (dict(out=FAKE + 2), E.SWQ_ERR_MISALIGNED), (dict(w=FAKE + 2), E.SWQ_ERR_MISALIGNED)):
        assert _attend(lib, l, c, b, **kw) == want, kw
    assert lib.swq_attention_q4_workspace_bytes(ctypes.byref(layer(num_heads=15)), ctypes.byref(c), ctypes.byref(b), 0) == 0
    assert lib.swq_attention_q4_workspace_bytes(ctypes.byref(l), ctypes.byref(c), ctypes.byref(batch(tokens=4)), 0) == 0
    with_weights = lib.swq_attention_q4_workspace_bytes(ctypes.byref(l), ctypes.byref(c), ctypes.byref(b), 1)
    assert with_weights >= n


def test_a_workspace_serves_smaller_calls(lib):
    """One sized for the most tokens is enough for fewer, whichever form they take."""
    c = cache(lib, max_positions=5000)
    size = lambda t, m, w: lib.swq_attention_q4_workspace_bytes(  # noqa: E731
        ctypes.byref(layer()), ctypes.byref(c), ctypes.byref(batch(tokens=t, max_tokens=m, starts=FAKE)), w)
    for w in (0, 1):
        most = 0
        for m in (1, 2, 3, 7, 8, 9, 31, 64, 100, 333, 1000, 4096):
            n = size(m * 3, m, w)
            assert n >= most, (m, w)
            assert n >= size(m, m, w)
            most = n


def test_refused_reads(lib):
    c = cache(lib)
    read = lambda c=c, B=3, first=None, starts=None, rows=None, count=5, k=FAKE, v=FAKE, dtype=0: lib.swq_q4_read(  # noqa: E731
        ctypes.byref(c), B, first, starts, rows, count, k, v, dtype, None)
    for kw, want in CACHES:
        assert read(cache(lib, **kw)) == want, kw
    for kw, want in ((dict(B=4), E.SWQ_ERR_BAD_SHAPE), (dict(B=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(count=-1), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(k=None, v=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(dtype=3), E.SWQ_ERR_UNSUPPORTED_DTYPE), (dict(k=FAKE + 2), E.SWQ_ERR_MISALIGNED),
                     (dict(count=0), E.SWQ_OK)):
        assert read(**kw) == want, kw


def test_refused_evictions(lib):
    src = cache(lib)
    far = FAKE + (1 << 32)

    def evict(src=src, B=3, w=FAKE, rows=FAKE, dst=None, budget=50, sink=4, recent=8, nw=None, nr=far, kept=far):
        dst = dst or cache(lib, data=far, max_positions=60)
        return lib.swq_q4_evict(ctypes.byref(src), B, w, rows, ctypes.byref(dst), budget, sink, recent, nw, nr, kept, None)

    for kw, want in CACHES:
        assert evict(cache(lib, **kw)) == want, kw
        assert evict(dst=cache(lib, **{"data": far, **kw})) == want, kw
    for kw, want in ((dict(B=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(B=4), E.SWQ_ERR_BAD_SHAPE), (dict(w=None), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(rows=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(nr=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(kept=None), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(budget=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(budget=61), E.SWQ_ERR_LIMIT), (dict(sink=-1), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(sink=43), E.SWQ_ERR_BAD_SHAPE), (dict(recent=47), E.SWQ_ERR_BAD_SHAPE), (dict(nw=FAKE), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(dst=cache(lib, max_positions=60)), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(dst=cache(lib, data=FAKE + 256, max_positions=60)), E.SWQ_ERR_INVALID_ARGUMENT),
                     (dict(dst=cache(lib, data=far, head_dim=128)), E.SWQ_ERR_BAD_SHAPE),
                     (dict(dst=cache(lib, data=far, sequences=2)), E.SWQ_ERR_BAD_SHAPE)):
        assert evict(**kw) == want, kw


@pytest.mark.parametrize("weights", [0, 1])
@pytest.mark.parametrize("tokens_each", [1, 40])
def test_a_workspace_does_for_calls_of_fewer_sequences(lib, weights, tokens_each):
    l, c = layer(num_heads=4, num_kv_heads=1, head_dim=64), cache(lib, sequences=2100, num_kv_heads=1, head_dim=64, max_positions=200_000)
    before = 0
    for b in range(1, 2101):
        x = batch(sequences=b, tokens=b * tokens_each, max_tokens=tokens_each, starts=FAKE)
        n = lib.swq_attention_q4_workspace_bytes(ctypes.byref(l), ctypes.byref(c), ctypes.byref(x), weights)
        assert n >= before, b
        before = n
