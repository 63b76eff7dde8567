"""The 4-bit cache's calls at the ends of what they accept, against the oracle in 64 bits; bars as in
test_gpu_attention_q4.py where no other is derived beside the test."""

import numpy as np
import pytest

from oracle import attention_q4_ref as R
from tests.test_gpu_attention_q4 import Setup, _close, _torch, _types

pytestmark = pytest.mark.gpu

f32 = np.float32


@pytest.mark.parametrize("hd,KVH", [(64, 8), (128, 2), (256, 2)])
@pytest.mark.parametrize("before,counts", [([0, 5], [20, 0]), ([3, 39, 7], [0, 9, 0]), ([13, 2, 1], [1, 0, 0]), ([5, 40, 33], [0, 0, 2])])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sequences_that_bring_nothing(hd, KVH, before, counts, dtype):
    """First, in the middle and last, their rows filling a block of 8 or not; k and v are the front of larger
    tensors, whose rest is NaN."""
    torch = _torch()
    H, N = 2 * KVH, sum(counts)
    s = Setup(hd + N, H, KVH, hd, 32, before, 70)
    q, k, v = s.tokens(counts, _types()[dtype])
    k, v = (torch.cat([x, torch.full_like(x[:1].expand(9, -1), float("nan"))])[:N] for x in (k, v))
    ws = s.blk.new_workspace(s.cache, tokens=N, max_tokens=max(counts))
    print(f"{before} + {counts}, hd {hd}", flush=True)
    held = s.cache.data.clone()
    s.blk.append(k, v, s.cache, s.rows(), starts=s.starts(counts), max_tokens=max(counts))
    want, _ = s.expect(counts)
    s.check_cache()
    s.cache.data.copy_(held)
    out = s.blk.prefill(q, k, v, s.cache, s.rows(), ws, starts=s.starts(counts), max_tokens=max(counts))
    _close(out, want, dtype)
    s.check_cache()
