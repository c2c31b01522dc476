"""Paged caches of q4_0 rows: the store (srhpm_rope_kv_paged) and attention over them (srhpm_flash_attn_paged) against plain forms
in 64 bits, at the lengths, masks, layouts and values where they can go wrong. The attention's bounds are those of
test_paged_gpu (the roundings are the same: a cache value is d * (q - 8) rounded to f16, and the references use that)."""
import numpy as np
import pytest
import torch

import paged_ref as R
import share_ref as X
import srhpm_b200 as S
from srhpm_b200 import _lib as L
from test_paged_gpu import attn_bound, attn_case, attn_check, attn_run, cu

pytestmark = pytest.mark.gpu
Q4 = L.Q4_0


def case4(rng, past, new, H, Hkv, D, P, qt, poison=True, **kw):
    """attn_case with q4_0 pages; slots behind the sequences hold NaN steps."""
    q, caches, vals, table, q_start, kv_len = attn_case(rng, past, new, H, Hkv, D, P, L.F16, qt, poison=poison, **kw)
    packed, values = [], []
    for v in vals:
        b = X.q4_pack(np.nan_to_num(v.astype(np.float32)))
        if poison:
            b[np.isnan(v[:, :, 0, 0])] = 0x7f  # f16 0x7f7f is NaN
        packed.append(b)
        values.append(X.q4_values(b))
    return q, packed, values, table, q_start, kv_len


# ---- store -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,H,Hkv,P,n,qt", [
    (256, 24, 4, 64, 9, torch.float32), (128, 7, 7, 48, 33, torch.float16), (64, 5, 1, 16, 1, torch.float32),
    (256, 6, 2, 32, 700, torch.float16), (64, 3, 3, 16, 5, torch.float32), (128, 32, 8, 16, 3000, torch.float16)])
def test_store(ctx, D, H, Hkv, P, n, qt):
    """Values as ggml rounds them, byte for byte; keys as it rounds the exactly turned ones (numbers equal, the step off by
    one f16 rounding at most); queries as for other caches; everything else untouched."""
    rng = np.random.default_rng(n + D)
    row = D // 32 * 18
    pages = -(-n // P) + 2
    x = rng.standard_normal((n, (H + 2 * Hkv) * D)).astype(np.float32)
    pos = rng.integers(0, 1 << 18, n).astype(np.int32)
    slots = rng.permutation(pages * P)[:n].astype(np.int64)
    slots[n // 2] = [-1, pages * P][n % 2]  # padding, or behind the cache
    kc0, vc0 = (rng.integers(0, 256, (pages, P, Hkv, row), dtype=np.uint8) for _ in range(2))
    kc, vc = cu(kc0), cu(vc0)
    qo = torch.zeros((n, H, D), device="cuda", dtype=qt)
    ctx.rope_kv_paged(cu(x), cu(pos), cu(slots), kc, vc, Q4, qo, theta_base=1e6)
    torch.cuda.synchronize()
    xs = x.reshape(n, H + 2 * Hkv, D)
    want = R.turn(xs[:, :H + Hkv], pos, 1e6)
    tol = 2.0 ** -20 * (np.abs(xs[:, :H + Hkv]) + np.abs(np.roll(xs[:, :H + Hkv], D // 2, -1)))
    half = 2.0 ** -11 if qt == torch.float16 else 2.0 ** -24
    got = qo.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want[:, :H]) <= tol[:, :H] + half * np.abs(want[:, :H]) + 2.0 ** -25).all()
    ok = (slots >= 0) & (slots < pages * P)
    at = slots[ok]
    gk, gv = kc.cpu().numpy().reshape(-1, Hkv, row), vc.cpu().numpy().reshape(-1, Hkv, row)
    assert np.array_equal(gv[at], X.q4_pack(np.ascontiguousarray(xs[ok][:, H + Hkv:])))
    d, num = X.q4_parts(gk[at])
    dw, numw = X.q4_parts(X.q4_pack(want[ok][:, H:].astype(np.float32)))
    assert np.array_equal(num, numw)
    assert (np.abs(d.astype(np.float64) - dw.astype(np.float64)) <= 2.0 ** -10 * np.abs(dw.astype(np.float64))).all()
    rest = np.setdiff1d(np.arange(pages * P), at)
    assert np.array_equal(gk[rest], kc0.reshape(-1, Hkv, row)[rest])
    assert np.array_equal(gv[rest], vc0.reshape(-1, Hkv, row)[rest])


def test_store_borders_and_head_major_pages(ctx):
    """Ties for the largest size, zeros, values on the borders of two numbers, tiny and huge ones; pages of [head][token];
    two contexts' worth of turns that change nothing (position 0)."""
    n, H, Hkv, D, P = 7, 2, 2, 128, 16
    rng = np.random.default_rng(3)
    x = (rng.integers(-4, 5, (n, H + 2 * Hkv, D)) * 0.5).astype(np.float32)
    x[1] = 0
    x[2] *= np.float32(1e-6)
    x[3] *= np.float32(1e4)
    x[4, :, ::32] = -7.0
    x[4, :, 1::32] = 7.0
    x[5] = np.tile(np.linspace(-1, 1, 64, dtype=np.float32), (H + 2 * Hkv, 2))
    x[6] = 1e-30  # steps below f16
    kc, vc = (torch.zeros((2, Hkv, P, D // 32 * 18), dtype=torch.uint8, device="cuda").transpose(1, 2) for _ in range(2))
    ctx.rope_kv_paged(cu(x.reshape(n, -1)), cu(np.zeros(n, np.int32)), cu(np.arange(13, 13 + n)), kc, vc, Q4,
                      torch.zeros((n, H, D), device="cuda"))
    for c, w in ((kc, x[:, H:H + Hkv]), (vc, x[:, H + Hkv:])):
        got = c.cpu().numpy().reshape(2 * P, Hkv, -1)[13:13 + n]
        assert np.array_equal(got, X.q4_pack(np.ascontiguousarray(w)))


def test_store_keys_next_to_a_border(ctx):
    """Keys whose turned values stand on borders by design: the numbers are those of the exactly turned values."""
    rng = np.random.default_rng(4)
    n, D, P = 512, 64, 16
    pos = rng.integers(1, 100000, n).astype(np.int32)
    target = (rng.integers(-8, 8, (n, 1, D)) + 0.5) / 8.0  # halves of steps where the block's largest value is -1
    target[:, :, ::32] = -1.0
    back = R.turn(target, -pos.astype(np.int64), 1e6)  # turned back, so that the store turns it there (but for 2^-24)
    x = np.zeros((n, 3, D), np.float32)
    x[:, 1:2] = back
    kc, vc = (torch.zeros((n // P, P, 1, D // 32 * 18), dtype=torch.uint8, device="cuda") for _ in range(2))
    ctx.rope_kv_paged(cu(x.reshape(n, -1)), cu(pos), cu(np.arange(n)), kc, vc, Q4, torch.zeros((n, 1, D), device="cuda"))
    exact = R.turn(x[:, 1:2], pos, 1e6)
    num = X.q4_parts(kc.cpu().numpy().reshape(n, 1, -1))[1]
    want = X.q4_parts(X.q4_pack(exact.astype(np.float32)))[1]
    # what 64 bits leave open: two libraries' sines differ in their last places, which f32 shows once in 2^28
    assert (num != want).sum() <= 2
    assert np.abs(num.astype(int) - want.astype(int)).max() <= 1


# ---- attention -------------------------------------------------------------------------------------------------------
SHAPES = [(256, 24, 4), (128, 8, 2), (64, 4, 4), (256, 3, 1), (128, 7, 1), (64, 16, 1), (128, 28, 4)]


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,Hkv", SHAPES)
@pytest.mark.parametrize("P,past,new", [
    (16, [0], [1]), (32, [127], [1]), (64, [128], [1]), (16, [255, 0, 31], [2, 1, 97]), (48, [130, 5], [9, 61]),
    (256, [500, 3], [1, 0]), (80, [0, 300, 63, 0], [0, 16, 65, 0]), (16, [15, 16, 31, 33], [1, 1, 1, 1])])
def test_attention_lengths(ctx, qt, D, H, Hkv, P, past, new):
    rng = np.random.default_rng(D + H + P)
    attn_run(ctx, case4(rng, past, new, H, Hkv, D, P, qt, pad_rows=3), Q4, D ** -0.5)
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,Hkv", SHAPES[:4])
@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (16, 0.0, True), (100, 5.0, False), (129, 0.0, False),
                                                 (0, 30.0, True), (5000, 0.0, True)])
@pytest.mark.parametrize("past,new", [([300, 1000], [3, 120]), ([700, 4, 250], [1, 2, 1])])
def test_attention_window_softcap_sinks(ctx, qt, D, H, Hkv, window, softcap, sink, past, new):
    rng = np.random.default_rng(D + window)
    case = case4(rng, past, new, H, Hkv, D, 32, qt, spread=2.0)
    kw = dict(window=window, softcap=softcap)
    if sink:
        kw["sinks"] = np.where(np.arange(H) % 3 == 1, -np.inf, rng.standard_normal(H) * 4).astype(np.float32)
    attn_run(ctx, case, Q4, D ** -0.5, **kw)
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,Hkv", [(256, 24, 4), (128, 32, 8), (64, 8, 1), (128, 8, 8)])
@pytest.mark.parametrize("past,new,window", [
    ([9000], [9], 0), ([20011], [1], 0), ([40000], [40], 0), ([3000, 10, 900] * 6, [1] * 18, 0),
    ([1326, 2666, 2194, 237, 153, 0, 1738], [13, 441, 97, 7, 229, 165, 1], 1024)])
def test_attention_cut_items(ctx, qt, D, H, Hkv, past, new, window):
    """Items cut between CTAs and several per CTA, five runs with the same bits."""
    rng = np.random.default_rng(D + len(past))
    P = 48
    q, caches, vals, table, q_start, kv_len = case4(rng, past, new, H, Hkv, D, P, qt)
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    runs = [ctx.flash_attn_paged(d[0], d[1], d[2], Q4, d[3], d[4], d[5], scale=D ** -0.5, window=window) for _ in range(5)]
    torch.cuda.synchronize()
    ctx.check()
    seqs = [[], []]
    for c, v in zip(seqs, vals):
        vt = cu(v)
        for s, n in enumerate(kv_len):
            c.append(vt[cu(table[s, :-(-int(n) // P)].astype(np.int64))].flatten(0, 1)[:int(n)])
    attn_bound(runs[0].cpu().numpy(), q, R.attention_dense(d[0], seqs[0], seqs[1], q_start, kv_len, D ** -0.5, window), q_start, kv_len)
    for r in runs[1:]:
        assert torch.equal(r, runs[0])


def test_attention_released_pages_before_the_window(ctx):
    """Pages wholly before the window are given away: their entries are no pages, and nothing of them is read."""
    rng = np.random.default_rng(5)
    P, W = 16, 40
    for D in (64, 128, 256):
        q, caches, vals, table, q_start, kv_len = case4(rng, [400, 1000, 333], [4, 130, 1], 4, 2, D, P, torch.float16)
        held = table.copy()
        for s, past in enumerate((400, 1000, 333)):
            first = max(0, past - W + 1)
            table[s, :first // P] = [-1, 2 ** 30, -5][s]
            b, slot = held[s, first // P], first % P  # slots of the first kept page before the window
            for c in caches:
                c[b, :slot] = 0x7f
            for v in vals:
                v[b, :slot] = np.nan
        attn_run(ctx, (q, caches, vals, table, q_start, kv_len), Q4, D ** -0.5, window=W)
        ctx.check()


def test_attention_rows_that_see_nothing(ctx):
    """kv_len smaller than the rows: rows before position 0 give 0, with sinks too."""
    rng = np.random.default_rng(6)
    for D in (64, 256):
        q, caches, vals, table, q_start, kv_len = case4(rng, [0, 0, 50], [5, 140, 2], 4, 2, D, 16, torch.float16, poison=False)
        kv_len[0], kv_len[1] = 0, 133
        for kw in ({}, {"sinks": np.ones(4, np.float32)}):
            attn_run(ctx, (q, caches, vals, table, q_start, kv_len), Q4, 0.1, **kw)
    ctx.check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [2, 70])
def test_attention_entries_that_are_no_page(ctx, D, new):
    """Inside the visible range: read as zeros, and the context's status says so."""
    rng = np.random.default_rng(7)
    q, caches, vals, table, q_start, kv_len = case4(rng, [300], [new], 4, 2, D, 16, torch.float16, poison=False)
    table[0, 3], table[0, 9], table[0, 12] = -1, vals[0].shape[0], 2 ** 31 - 1
    attn_run(ctx, (q, caches, vals, table, q_start, kv_len), Q4, D ** -0.5)
    with pytest.raises(S.SrhpmError) as e:
        ctx.check()
    assert e.value.status == L.ERR_DEVICE
    ctx.check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [3, 90])
def test_attention_layouts(ctx, D, new):
    """Pages of [head][token]; K and V side by side in one pool; queries as columns of wider rows, output rows with strides
    of their own."""
    rng = np.random.default_rng(8)
    H, Hkv, P = 6, 3, 32
    q, caches, vals, table, q_start, kv_len = case4(rng, [77, 10], [new, 40], H, Hkv, D, P, torch.float16)
    T = q.shape[0]
    wide = torch.zeros((T, H + 2, D), device="cuda", dtype=torch.float16)
    wide[:, 1:H + 1] = cu(q)
    heads = [cu(c).transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    both = torch.stack([cu(c) for c in caches], 2)  # [pages, P, 2, Hkv, row]
    tb = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    tb[:, 2:2 + table.shape[1]] = cu(table)
    for k, v in (heads, (both[:, :, 0], both[:, :, 1]), (heads[0], both[:, :, 1])):
        out = torch.full((T, H + 1, D), 7.0, device="cuda", dtype=torch.float16)
        ctx.flash_attn_paged(wide[:, 1:H + 1], k, v, Q4, tb[:, 2:2 + table.shape[1]], cu(q_start), cu(kv_len), scale=D ** -0.5,
                             out=out[:, :H])
        torch.cuda.synchronize()
        attn_check(out[:, :H].cpu().numpy(), q, vals, table, q_start, kv_len, D ** -0.5)
        assert (out[:, H] == 7.0).all()
    ctx.check()


def test_attention_far_pages(ctx):
    """Pages behind 2^32 bytes of a pool."""
    P, Hkv, D, H = 64, 8, 128, 8
    row = D // 32 * 18
    pages = (1 << 32) // (P * Hkv * row) + 40
    kc, vc = (torch.zeros((pages, P, Hkv, row), dtype=torch.uint8, device="cuda") for _ in range(2))
    rng = np.random.default_rng(9)
    use = [pages - 1, 0, pages - 30]
    small = [X.q4_pack(rng.standard_normal((3, P, Hkv, D)).astype(np.float32)) for _ in range(2)]
    for c, v in ((kc, small[0]), (vc, small[1])):
        c[use] = cu(v)
    for n in (1, 5, 100):
        q = rng.standard_normal((n, H, D)).astype(np.float16)
        out = ctx.flash_attn_paged(cu(q), kc, vc, Q4, cu(np.array([use], np.int32)), cu(np.array([0, n], np.int32)),
                                   cu(np.array([150], np.int32)), scale=D ** -0.5)
        attn_check(out.cpu().numpy(), q, [X.q4_values(v) for v in small], np.array([[0, 1, 2]]), np.array([0, n]), np.array([150]), D ** -0.5)
    ctx.check()


def test_attention_many_sequences(ctx):
    rng = np.random.default_rng(10)
    n = 700
    case = case4(rng, rng.integers(0, 60, n).tolist(), rng.integers(0, 3, n).tolist(), 2, 1, 64, 16, torch.float16, pad_rows=2)
    attn_run(ctx, case, Q4, 0.125)
    ctx.check()


@pytest.mark.parametrize("D,H,Hkv", [(128, 8, 2), (256, 6, 1)])
def test_attention_streams_and_replay(ctx, D, H, Hkv):
    """Two calls at once on two streams, then captured once and replayed with other lengths, tables and rows."""
    rng = np.random.default_rng(11)
    a = case4(rng, [3000, 500], [4, 100], H, Hkv, D, 16, torch.float16)
    b = case4(rng, [2000, 900], [90, 3], H, Hkv, D, 16, torch.float16, pad_rows=11)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    dev = [[cu(x) for x in (c[0], c[1][0], c[1][1], c[3], c[4], c[5])] for c in (a, b)]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [ctx.flash_attn_paged(d[0], d[1], d[2], Q4, d[3], d[4], d[5], scale=0.1, stream=s) for d, s in zip(dev, streams)]
    torch.cuda.synchronize()
    for o, c in zip(outs, (a, b)):
        attn_check(o.cpu().numpy(), c[0], c[2], c[3], c[4], c[5], 0.1)
    T, pages, cols = (max(x, y) for x, y in zip((a[0].shape[0], a[1][0].shape[0], a[3].shape[1]),
                                                (b[0].shape[0], b[1][0].shape[0], b[3].shape[1])))
    q = torch.zeros((T, H, D), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((pages,) + a[1][0].shape[1:], dtype=torch.uint8, device="cuda") for _ in range(2))
    tb = torch.zeros((2, cols), dtype=torch.int32, device="cuda")
    qs, kl = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)

    def put(c):
        q[:c[0].shape[0]] = cu(c[0])
        kc[:c[1][0].shape[0]], vc[:c[1][1].shape[0]] = cu(c[1][0]), cu(c[1][1])
        tb[:, :c[3].shape[1]] = cu(c[3])
        qs.copy_(cu(c[4]))
        kl.copy_(cu(c[5]))

    put(a)
    g = torch.cuda.CUDAGraph()
    ctx.flash_attn_paged(q, kc, vc, Q4, tb, qs, kl, scale=0.1, out=out)
    with torch.cuda.graph(g):
        ctx.flash_attn_paged(q, kc, vc, Q4, tb, qs, kl, scale=0.1, out=out)
    for c in (a, b, a):
        put(c)
        g.replay()
        torch.cuda.synchronize()
        attn_check(out.cpu().numpy()[:c[0].shape[0]], c[0], c[2], c[3], c[4], c[5], 0.1)
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("past,new,at", [([300], [3], 301), ([9000, 40], [2, 1], 100), ([0], [500], 130), ([20000], [40], 7), ([5000, 5], [1, 1], 4999)])
def test_attention_nan_keys(ctx, qt, D, past, new, at):
    """A NaN step among the keys of KV head 0: the rows of its heads that see it are NaN, whole and cut items alike, all
    others keep their bits."""
    rng = np.random.default_rng(14)
    P, H, Hkv = 32, 4, 2
    q, caches, vals, table, q_start, kv_len = case4(rng, past, new, H, Hkv, D, P, qt)
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    clean = ctx.flash_attn_paged(d[0], d[1], d[2], Q4, d[3], d[4], d[5], scale=0.1).cpu().numpy()
    d[1][int(table[0, at // P]), at % P, 0, :2] = 0x7e
    got = ctx.flash_attn_paged(d[0], d[1], d[2], Q4, d[3], d[4], d[5], scale=0.1).cpu().numpy()
    ctx.check()
    sees = np.zeros((q.shape[0], H, 1), bool)
    sees[max(0, at - past[0]):new[0], :H // Hkv] = True
    assert np.isnan(got[np.broadcast_to(sees, got.shape)]).all()
    keep = ~np.broadcast_to(sees, got.shape)
    assert np.array_equal(got[keep], clean[keep]) and np.isfinite(clean).all()


def test_attention_large_steps(ctx):
    """Steps of either sign over the range of f16, so that products round and scores differ widely."""
    rng = np.random.default_rng(15)
    for D, n in ((128, 1), (128, 60), (256, 3), (64, 9)):
        q, caches, vals, table, q_start, kv_len = case4(rng, [700, 90], [n, 1], 4, 2, D, 16, torch.float16, poison=False)
        for c, scale in ((caches[0], 1.0), (caches[1], 900.0)):
            b = c.reshape(c.shape[:-1] + (-1, 18))
            d = (rng.standard_normal(b.shape[:-1]) * scale).astype(np.float16)
            b[..., :2] = d[..., None].view(np.uint8)
        vals = [X.q4_values(c) for c in caches]
        attn_run(ctx, (q, caches, vals, table, q_start, kv_len), Q4, 0.05)
    ctx.check()


@pytest.mark.parametrize("D,H,Hkv", [(256, 6, 1), (256, 6, 3), (128, 14, 2), (64, 4, 4), (64, 1, 1)])
@pytest.mark.parametrize("window", [0, 1, 100, 600])
def test_attention_prompts(ctx, D, H, Hkv, window):
    """Sequences that share the pages of a common beginning and bring rows by the hundred; one brings none, one has fewer cached tokens
    than rows; released entries before a window; pages of [head][token] and K/V in one pool."""
    rng = np.random.default_rng(16)
    P, new = 48, [500, 0, 410, 390]
    q, caches, vals, table, q_start, kv_len = case4(rng, [700, 5, 301, 0], new, H, Hkv, D, P, torch.float16, pad_rows=3)
    table[2, :4] = table[0, :4]
    kv_len[3] = 333
    if window == 100:
        table[0, :(700 - window + 1) // P] = [-1, 2 ** 30, -7, vals[0].shape[0]] * 3
    heads = [cu(c).transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    both = torch.stack([cu(c) for c in caches], 2)
    first = None
    for k, v in ((cu(caches[0]), cu(caches[1])), heads, (both[:, :, 0], both[:, :, 1])):
        out = torch.full(q.shape, 7.0, device="cuda", dtype=torch.float16)
        ctx.flash_attn_paged(cu(q), k, v, Q4, cu(table), cu(q_start), cu(kv_len), scale=D ** -0.5, window=window, out=out)
        assert (out[-3:] == 7.0).all()  # rows behind the last sequence
        if first is None:
            first = out
            attn_check(out.cpu().numpy(), q, vals, table, q_start, kv_len, D ** -0.5, window=window)
        assert torch.equal(out, first)
    ctx.check()
