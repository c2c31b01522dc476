"""As many sequences as a step may have: the plan's sums of all of them stand in shared memory, where the cache's rows land next."""
import numpy as np
import pytest
import torch

from srhpm_b200 import _lib as L
from test_paged_gpu import attn_case, attn_check, cu
from test_q4_cache_gpu import case4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D,H", [(L.Q4_0, 64, 2), (L.Q4_0, 128, 4), (L.Q4_0, 64, 16), (L.Q4_0, 256, 12), (L.F16, 64, 2), (L.Q8_0, 256, 2)])
def test_attention(ctx, qt, kv, D, H):
    rng = np.random.default_rng(D + H)
    n, P = 8192, 16
    past, new = rng.integers(0, 20, n).tolist(), rng.integers(0, 3, n).tolist()
    past[:2], new[:2], past[-1], new[-1] = [3000, 1], [3, 2], 500, 1
    case = case4(rng, past, new, H, 1, D, P, qt) if kv == L.Q4_0 else attn_case(rng, past, new, H, 1, D, P, kv, qt)
    q, caches, vals, table, q_start, kv_len = case
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    runs = [ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=D ** -0.5) for _ in range(3)]
    attn_check(runs[0].cpu().numpy(), q, vals, table, q_start, kv_len, D ** -0.5)
    assert all(torch.equal(r, runs[0]) for r in runs[1:])
    ctx.check()
