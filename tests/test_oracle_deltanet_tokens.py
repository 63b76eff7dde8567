"""The 64-bit oracle of swq_deltanet_tokens against oracle/deltanet_ref.py, which mlx's fixtures pin: the same block in 32 bits,
token after token, so 1e-5 of the largest as between that oracle and the device."""

import numpy as np
import pytest
import torch

from oracle import deltanet_ref as D
from oracle import deltanet_tokens_ref as R


def case(K, T, start, seed=0):
    rng = np.random.default_rng(seed)
    nk, nv, dk, dv = 2, 4, 8, 8
    conv, val = 2 * nk * dk + nv * dv, nv * dv
    n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    prm = dict(conv_w=n(conv, K) * 0.5, a_log=n(nv) * 0.5, dt_bias=n(nv) * 0.5, norm_w=1 + 0.2 * n(dv), eps=1e-6, nk=nk, nv=nv, dk=dk, dv=dv)
    return prm, n(T, conv), n(T, val), n(T, nv), n(T, nv), n(K, conv), n(nv, dv, dk) * 0.3


@pytest.mark.parametrize("K,T,start", [(4, 1, 0), (4, 9, 5), (2, 5, 3), (4, 2, 7)])
def test_the_same_block_as_the_step_oracle(K, T, start):
    prm, mixed, z, b, a, ring, state = case(K, T, start, seed=K + T)
    tail = np.stack([ring[(start - (K - 1) + j) % K] for j in range(K - 1)])
    want, _, s_want = D.deltanet_core(mixed, z, b, a, conv_tail=tail, state=state.copy(), **prm)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x))  # noqa: E731
    weights = {k: t(v) for k, v in prm.items() if isinstance(v, np.ndarray)}
    y, ring_after, s, _ = R.tokens(t(np.concatenate([mixed, z], 1)), t(np.concatenate([b, a], 1)), t(ring).double(), t(state).double(), start,
                                   nk=2, nv=4, dk=8, dv=8, eps=1e-6, split=True, **weights)
    assert np.abs(y.numpy() - want).max() < 1e-5 * np.abs(want).max()
    assert np.abs(s.numpy() - s_want).max() < 1e-5 * np.abs(s_want).max()
    for i in range(max(T - K, 0), T):
        assert np.array_equal(ring_after[(start + i) % K].numpy(), mixed[i].astype(np.float64))


def test_a_planted_mistake_shows():
    """Queries and keys exchanged."""
    prm, mixed, z, b, a, ring, state = case(4, 6, 0)
    swapped = np.concatenate([mixed[:, 16:32], mixed[:, :16], mixed[:, 32:]], 1)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x))  # noqa: E731
    weights = {k: t(v) for k, v in prm.items() if isinstance(v, np.ndarray)}
    outs = [R.tokens(t(np.concatenate([m, z], 1)), t(np.concatenate([b, a], 1)), t(ring).double() * 0, t(state).double() * 0, 0, nk=2, nv=4, dk=8, dv=8,
                     eps=1e-6, split=True, **weights)[0] for m in (mixed, swapped)]
    assert float((outs[0] - outs[1]).abs().max()) > 1e-2 * float(outs[0].abs().max())
