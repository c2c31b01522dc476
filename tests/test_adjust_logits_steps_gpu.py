"""Rules on logits (srhpm_adjust_logits), bit by bit: every operation of the rules is rounded to f32 by itself, and a rule
that a token does not have leaves its sign of zero alone."""
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


@pytest.mark.parametrize("S", [1, 70])
@pytest.mark.parametrize("in_place", [False, True])
def test_zeros_keep_their_sign(ctx, S, in_place):
    """-0 that is penalised by nothing stays -0 where only other tokens are biased; +0 and a bias of -0 likewise. Tokens that come
    into the window with a later row too."""
    V, f = 40000, np.float32
    lg = np.zeros((3 * S, V), f)
    lg[:, ::2] = -0.0
    ids = np.tile(np.array([20, 31, 39998], np.int32), S)
    history = np.tile(np.array([0, 1, 2, 3, 39000, 39001], np.int32), (S, 1))
    r = dict(history=history, n_history=np.full(S, 6, np.int32), repeat=np.full(S, 1.5, f), frequency=np.zeros(S, f),
             presence=np.zeros(S, f),
             bias=(np.arange(S + 1, dtype=np.int32) * 4, np.tile(np.array([2, 3, 50, 60], np.int32), S),
                   np.tile(np.array([0.0, -0.0, -0.0, 0.0], f), S)))
    q_start = np.arange(S + 1, dtype=np.int32) * 3
    want = steps(lg, ids, q_start, **r)
    src = cu(lg)
    got = ctx.adjust_logits(src, cu(ids), cu(q_start), out=src if in_place else None,
                            **{k: tuple(cu(x) for x in v) if k == "bias" else cu(v) for k, v in r.items()})
    assert np.array_equal(got.cpu().numpy().view(np.int32), want.view(np.int32))
    ctx.check()
