"""Keys of a q4_0 cache whose turned block has two values of nearly the largest size and of unlike signs: which of them becomes the
step decides every number of the block, so it is the one of the exactly turned values, rounded to f32 (the first of equals)."""
import numpy as np
import pytest
import torch

import paged_ref as R
import share_ref as X
from srhpm_b200 import _lib as L
from test_paged_gpu import cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_two_largest_values_of_unlike_signs(ctx, D, qt):
    rng = np.random.default_rng(D)
    n, P = 512, 16
    pos = rng.integers(1, 100000, n).astype(np.int32)
    target = rng.uniform(-0.9, 0.9, (n, 1, D // 32, 32))
    for t in target.reshape(-1, 32):
        i, j = rng.permutation(32)[:2]
        t[i], t[j] = 1.0, -1.0
    back = R.turn(target.reshape(n, 1, D), -pos.astype(np.int64), 1e6)  # turned back: the store turns it there but for 2^-24
    x = np.zeros((n, 3, D), np.float32)
    x[:, 1:2] = back
    kc, vc = (torch.zeros((n // P, P, 1, D // 32 * 18), dtype=torch.uint8, device="cuda") for _ in range(2))
    ctx.rope_kv_paged(cu(x.reshape(n, -1)), cu(pos), cu(np.arange(n)), kc, vc, L.Q4_0, torch.zeros((n, 1, D), device="cuda", dtype=qt))
    d, num = X.q4_parts(kc.cpu().numpy().reshape(n, 1, -1))
    dw, numw = X.q4_parts(X.q4_pack(R.turn(x[:, 1:2], pos, 1e6).astype(np.float32)))
    # what 64 bits leave open: two libraries' sines differ in their last places, which f32 shows once in 2^28
    assert (num != numw).any(-1).sum() == 0
    assert (np.sign(d) == np.sign(dw)).all()
    ctx.check()
