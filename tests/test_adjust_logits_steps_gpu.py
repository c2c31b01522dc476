"""Rules on logits (srhpm_adjust_logits), bit by bit: every operation of the rules is rounded to f32 by itself."""
import numpy as np
import pytest
import torch

from test_adjust_logits_gpu import rules
from test_paged_gpu import cu

pytestmark = pytest.mark.gpu


def steps(lg, ids, q_start, history, n_history, repeat, frequency, presence, bias=None):
    """The rules in f32, one operation at a time."""
    out, f = lg.copy(), np.float32
    for s in range(len(q_start) - 1):
        for r in range(q_start[s], q_start[s + 1]):
            l = out[r]
            if bias is not None:
                start, tok, val = bias
                at = np.array(list(dict.fromkeys(tok[start[s]:start[s + 1]].tolist())), np.int64)
                last = dict(zip(tok[start[s]:start[s + 1]].tolist(), val[start[s]:start[s + 1]].tolist()))
                l[at] = l[at] + np.array([last[int(x)] for x in at], f)
            x, c = np.unique(np.concatenate([history[s, :n_history[s]], ids[q_start[s]:r + 1]]), return_counts=True)
            v = np.where(l[x] > 0, l[x] / repeat[s], l[x] * repeat[s]).astype(f)
            l[x] = v - ((c.astype(f) * frequency[s]).astype(f) + presence[s]).astype(f)
    return out


@pytest.mark.parametrize("ks,V", [([5, 3], 3000), ([4] * 64, 40003), ([3, 0, 9] * 30, 40004)])
def test_every_operation_is_rounded(ctx, ks, V):
    rng = np.random.default_rng(V)
    ids, q_start, r = rules(rng, ks, V, cap=3000, bias=200, hot=min(V, 500))
    lg = (rng.standard_normal((len(ids), V)) * 4).astype(np.float32)
    want = steps(lg, ids, q_start, **r)
    got = ctx.adjust_logits(cu(lg), cu(ids), cu(q_start), **{k: tuple(cu(x) for x in v) if k == "bias" else cu(v) for k, v in r.items()})
    assert np.array_equal(got.cpu().numpy().view(np.int32), want.view(np.int32))
    ctx.check()
