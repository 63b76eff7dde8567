"""The 4-bit cache's oracle against closed forms and the f32 attention oracle."""

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from oracle import attention_ref as A

f32 = np.float32


@pytest.mark.parametrize("scale", [1.0, 1e-4, 3e3])
def test_quantised_values_are_within_half_a_step(scale):
    """|value - x| <= s / 2 from the code, + the roundings of scale and bias to f16: half a unit of
    2^-10 of each, at most 15 steps (2^-24 below the normal numbers), + the values past the last code."""
    x = np.random.default_rng(0).standard_normal((5, 3, 128)) * scale
    part = R.quantise(x)
    s, b = (np.repeat(p.astype(np.float64), 64, -1) for p in part[1:])
    slack = 15 * np.maximum(s * 2.0 ** -11, 2.0 ** -25) + np.maximum(np.abs(b) * 2.0 ** -11, 2.0 ** -25)
    assert (np.abs(R.values(part) - x) <= s / 2 + 2 * slack).all()
    assert part[0].min() == 0 and part[0].max() == 15


def test_equal_values_and_values_out_of_range():
    x = np.full((1, 128), 3.0)
    x[0, 64:] = [np.nan, np.inf, -np.inf, 1e9] * 16
    part = R.quantise(x)
    v = R.values(part)
    assert (v[0, :64] == 3.0).all() and np.isfinite(v).all()
    assert part[2][0, 1] == -65504 and (part[0][0, 64:68] == [7, 15, 0, 15]).all() or (part[0][0, 64:68] == [8, 15, 0, 15]).all()


def test_words_hold_codes_in_order():
    seq = R.random_sequence(np.random.default_rng(1), 2, 21, 64)
    k, v, par = R.words(seq, 32)
    for h, row, d in ((0, 0, 0), (1, 20, 63), (0, 13, 17)):
        assert (k[h, row, d // 8] >> (4 * (d % 8))) & 15 == seq["k"][0][h, row, d]
        assert (v[h, row // 8, d] >> (4 * (row % 8))) & 15 == seq["v"][0][h, row, d]
        assert par[h, 3, 0, row] == seq["v"][2][h, row, 0]
    assert (v[:, 2] >> 20 == 0).all()


def test_attention_is_the_f32_oracles_over_the_held_values():
    """Over rows that are already values of the cache, the two oracles differ by the f32 one's rounding."""
    rng = np.random.default_rng(2)
    H, KVH, hd, rot, S = 4, 2, 64, 16, 5
    prm = dict(q_norm_w=(1 + 0.1 * rng.standard_normal(hd)).astype(f32), k_norm_w=np.ones(hd, f32), H=H, KVH=KVH, hd=hd, rot=rot,
               theta=1e4, eps=1e-6)
    q, k, v = (rng.standard_normal((S, n)).astype(f32) for n in (H * 2 * hd, KVH * hd, KVH * hd))
    table = R.rope_table(S, rot, 1e4)
    seq = R.append(R.empty_sequence(KVH, hd), k.reshape(S, KVH, hd), v.reshape(S, KVH, hd), prm["k_norm_w"], 1e-6, table)
    out, got = R.attend(seq, 0, q.reshape(S, H, 2, hd), prm["q_norm_w"], 1e-6, table)
    K, V = (R.values(seq[x]).transpose(1, 0, 2).astype(f32) for x in "kv")
    for s in range(S):
        # the f32 oracle appends the token's own f32 row, so it is given the rows before, and that one's values
        core, _, _ = A.attention_core(q[s:s + 1], k[s:s + 1], v[s:s + 1], cache_k=K[:s], cache_v=V[:s], **prm)
        x = R.norm_rope(q[s].reshape(H, 2, hd)[:, 0], prm["q_norm_w"], 1e-6, table[s])
        for h in range(H):
            z = K[:s + 1, h // 2].astype(np.float64) @ x[h] / 8
            p = np.exp(z - z.max()) / np.exp(z - z.max()).sum()
            want = p @ V[:s + 1, h // 2] / (1 + np.exp(-q[s].reshape(H, 2, hd)[h, 1].astype(np.float64)))
            np.testing.assert_allclose(out[s, h], want, rtol=1e-5, atol=1e-6)
        # the new row is off by its quantisation alone: half of a step of about a third
        assert np.abs(core.reshape(H, hd) - out[s]).max() < 0.3
    np.testing.assert_allclose(got.sum(-1), S * H / KVH)


def test_keep_ties_and_short_sequences():
    w = np.array([0, 5, 1, 1, 1, 9, 0, 0], f32)
    assert R.keep(w, 8, 4, 1, 1).tolist() == [0, 1, 5, 7]
    assert R.keep(w, 8, 5, 1, 1).tolist() == [0, 1, 2, 5, 7]
    assert R.keep(w, 8, 2, 0, 0).tolist() == [1, 5]
    assert R.keep(w, 3, 4, 1, 1).tolist() == [0, 1, 2]
    w[1] = np.nan
    assert R.keep(w, 8, 3, 1, 1).tolist() == [0, 5, 7]


def test_no_value_passes_the_largest_f16():
    rng = np.random.default_rng(9)
    lo = -65504 + 400 * rng.random((300, 1, 1))
    hi = 65504 - 400 * rng.random((300, 1, 1))
    x = np.concatenate([lo, hi, lo + (hi - lo) * rng.random((300, 1, 62))], -1)
    part = R.quantise(x)
    v = R.values(part)
    assert (v <= 65504).all() and (np.abs(v - x) <= (hi - lo) / 30 + 140).all()  # half a step, the scale's and the bias' rounding
    plain = ((hi - lo) / 15).astype(np.float32).astype(np.float16)
    up = part[2].astype(np.float64) + 15 * plain.astype(np.float64)
    assert (up > 65504).any() and ((up > 65504) == (part[1] < plain)).all()
