"""The 4-bit cache's format at the end of f16's range: no value passes 65504, whatever bias and scale round to."""

import numpy as np

from oracle import attention_q4_ref as R


def near_the_top(count, seed=0):
    """Groups [count, 1, 64] whose minimum lies anywhere below the largest f16 number, mostly close to where a bias
    rounds up (by 16 at most), and whose maximum is that number."""
    rng = np.random.default_rng(seed)
    lo = np.concatenate([65504 - 32 * rng.integers(0, 200, count // 2) - 16 + rng.choice([-2, -0.25, 0, 0.25, 2], count // 2),
                         65504 - 10 ** rng.uniform(-2, 5, count - count // 2)])[:, None, None]
    x = np.concatenate([lo, np.full_like(lo, 65504.0), lo + (65504 - lo) * rng.random((count, 1, 62))], -1)
    return np.clip(x, -65504, 65504)


def test_a_rounded_up_bias_takes_more_than_one_step_of_the_scale():
    x = np.linspace(65462.25, 65504, 64)[None, None]
    codes, scale, bias = R.quantise(x)
    assert bias[0, 0, 0] == 65472  # rounded up: the values are 9.75 above the numbers
    v = R.values((codes, scale, bias))
    assert v.max() <= 65504 and np.abs(v - x).max() <= 10
    # the largest scale that does: the next one would pass
    up = np.nextafter(scale, np.float16(np.inf)).astype(np.float64)
    assert (bias.astype(np.float64) + 15 * up > 65504).all()


def test_no_value_passes_the_largest_number():
    x = near_the_top(4000)
    part = R.quantise(x)
    v = R.values(part)
    assert v.max() <= 65504
    s, b = (p.astype(np.float64) for p in part[1:])
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    plain = ((hi - lo) / 15).astype(np.float32).astype(np.float16)
    over = b + 15 * plain.astype(np.float64) > 65504
    assert over.mean() > 0.2 and np.array_equal(part[1][~over], plain[~over])
    up = np.nextafter(part[1], np.float16(np.inf)).astype(np.float64)
    assert (b + 15 * up > 65504)[over].all()
    # half a step, the bias' rounding (16) at either end, and what f16's step of a scale up to 8,736 leaves (15 * 8 / 2)
    assert (np.abs(v - x) <= (hi - lo) / 30 + 32 + 15 * np.maximum(s * 2.0 ** -10, 2.0 ** -24)).all()
