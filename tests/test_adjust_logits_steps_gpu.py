"""Rules on logits (srhpm_adjust_logits), bit by bit: every operation of the rules is rounded to f32 by itself, and a rule that a
token does not have leaves its sign of zero alone. And the form that takes all rows of a sequence in one CTA, over
vocabularies of several slices: windows that move from row to row, masked rows beside free ones, in place and not."""
import numpy as np
import pytest
import torch

from test_adjust_logits_gpu import check, rules
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


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,V", [(64, 40003), (64, 40004), (17, 151936), (17, 151933), (150, 16384), (200, 12289)])
@pytest.mark.parametrize("hot", [40, 1 << 30])
def test_rows_of_a_sequence_in_one_block(ctx, S, V, hot, in_place):
    """0 to 9 rows each, windows of every kind, biases; each second row masked, so that rows that go through whole and rows of which
    only the listed tokens change follow one another."""
    rng = np.random.default_rng(S + V + hot % 7)
    ks = rng.integers(0, 10, S)
    ks[:3] = [9, 0, 1]
    ids, q_start, r = rules(rng, ks.tolist(), V, cap=5000, last=[1, 3, 4096, -1, 0, 2], bias=60, mask=True, hot=hot)
    r["mask_row"][::2] = -1
    check(ctx, (rng.standard_normal((len(ids), V)) * 4).astype(np.float32), ids, q_start, r, in_place=in_place, pad=3)
    ctx.check()


@pytest.mark.parametrize("in_place", [False, True])
def test_windows_that_move_within_one_block(ctx, in_place):
    """Drafts that say the same tokens again and again, at the borders of slices and of the warps' parts of them, with windows of a few
    tokens: a token enters, counts twice, and leaves from one row to the next."""
    rng = np.random.default_rng(11)
    S, V = 80, 40001
    edge = np.array([0, 511, 512, 4095, 4096, 4097, 8191, 8192, 36863, 36864, 40000], np.int32)
    ks = [9] * S
    ids, q_start, r = rules(rng, ks, V, cap=6, last=[1, 2, 3, 4, -1], bias=3)
    ids[:] = edge[rng.integers(0, len(edge), len(ids))]
    r["history"][:] = edge[rng.integers(0, len(edge), r["history"].shape)]
    check(ctx, (rng.standard_normal((len(ids), V)) * 4).astype(np.float32), ids, q_start, r, in_place=in_place)
    ctx.check()
