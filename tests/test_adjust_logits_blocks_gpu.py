"""Rules on logits (srhpm_adjust_logits) where all rows of a sequence are one block's, over vocabularies of several slices: windows
that move from row to row, masked rows beside free ones, in place and not; against the plain form in 64 bits with the bounds of
test_adjust_logits_gpu."""
import numpy as np
import pytest

from test_adjust_logits_gpu import check, rules

pytestmark = pytest.mark.gpu


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
