"""The paged-cache operators (srhpm_page_plan, srhpm_rope_kv_paged, srhpm_flash_attn_paged, srhpm_verify_sample) against
plain forms in 64 bits (paged_ref), at the lengths, masks, layouts and values where they can go wrong.

Whole-number results have to be equal. Attention's bounds are counted from its roundings (f16 eps 2^-10, half a step
2^-11). With A = sum p |v| / sum p of a row and B its largest sum |q k| * scale:
  scores: the product's f32 sum over D terms is off by at most (D / 8 + 2) 2^-23 B (one step per 16 terms, two passes),
          with f32 rows also 2 * 2^-22 B from the two-part split of q; a score's error e moves every p by a factor
          within exp(+-e), the result by at most 2 e A; the exponential adds 2^-21 A;
  f16 rows: probabilities round to f16 (2^-11 A in the product, and the sum may count them unrounded: 2^-11 |o| <=
          2^-11 A), the output rounds (2^-11 |o|), so 3 * 2^-11 A together;
  f32 rows: two f16 parts keep 2^-22 of p, the output rounds to 2^-24: 2^-21 A together;
  sums over n tokens in f32: one step per 16-term product and per tile rescale: (n / 16 + n / 64 + 4) 2^-23 A at most.
"""
import ctypes

import numpy as np
import pytest
import torch

import oracle as O
import paged_ref as R
import srhpm_b200 as S
from srhpm_b200 import _lib as L

pytestmark = pytest.mark.gpu


def cu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- page plan -------------------------------------------------------------------------------------------------------
def plan_case(rng, S, P, past_hi, new_hi, spare=3, extra_cols=1):
    past = rng.integers(0, past_hi + 1, S).astype(np.int32)
    new = rng.integers(0, new_hi + 1, S).astype(np.int32)
    have = -(-past // P)
    want = -(-(past + new) // P)
    cols = max(1, int(want.max()) + extra_cols)
    pool = rng.permutation(int(want.sum()) + spare).astype(np.int32)
    table = np.full((S, cols), -7, np.int32)
    at = 0
    for s in range(S):
        table[s, :have[s]] = pool[at:at + have[s]]
        at += have[s]
    return past, new, table, pool[at:]


def check_plan(ctx, past, new, table, free, P, n_rows, head=None):
    tb = cu(table)
    hd = None if head is None else cu(np.array([head], np.int32))
    r = ctx.page_plan(cu(past), cu(new), tb, cu(free), P, n_rows, free_head=hd)
    torch.cuda.synchronize()
    want = R.plan(past, new, table, free, P, n_rows, head or 0)
    got = (tb, r.q_start, r.kv_len, r.pos, r.slots, r.status, r.n_taken)
    for name, g, w in zip(("table", "q_start", "kv_len", "pos", "slots", "status", "n_taken"), got, want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
    return r


@pytest.mark.parametrize("S,P,past_hi,new_hi", [(1, 16, 0, 1), (1, 1, 5, 9), (2, 48, 100, 64), (33, 16, 300, 17),
                                                (1000, 64, 5000, 40), (1025, 16, 64, 3), (8192, 256, 900, 300)])
def test_plan_lengths(ctx, S, P, past_hi, new_hi):
    rng = np.random.default_rng(S + P)
    past, new, table, free = plan_case(rng, S, P, past_hi, new_hi)
    check_plan(ctx, past, new, table, free, P, int(new.sum()) + 11)


def test_plan_refusals_per_sequence(ctx):
    """Every status, sequences behind refused ones, an empty step, and a head into the free list."""
    P = 16
    past = np.array([30, -1, 16, 15, 100, 0, 32, 3, 16, 31], np.int32)
    new = np.array([3, 4, -2, 2, 60, 33, 0, 40, 0, 1], np.int32)
    table = np.arange(10 * 8, dtype=np.int32).reshape(10, 8)
    free = np.arange(500, 509, dtype=np.int32)
    r = check_plan(ctx, past, new, table, free, P, 200, head=2)
    # pages needed: 1 (30 + 3), 1 (15 + 2), 3 (0 + 33), 2 (3 + 40): 7, the 7 behind head 2
    assert r.status.cpu().tolist() == [0, 3, 3, 0, 1, 0, 0, 0, 0, 0]
    r = check_plan(ctx, past, new, table, free, P, 200, head=3)
    assert r.status.cpu().tolist() == [0, 3, 3, 0, 1, 0, 0, 2, 0, 0]
    check_plan(ctx, past, new, table, free, P, 40)          # rows run out inside sequence 5
    check_plan(ctx, past, new, table, free, P, 200, head=9)   # nothing free at all
    check_plan(ctx, past, new, table, free[:0], P, 200)
    check_plan(ctx, past, np.zeros_like(new), table, free, P, 0)
    check_plan(ctx, past, new, table, free, P, 200, head=-3)
    table[3, 0] = -1                                          # a hole in the cached part: no slot there
    check_plan(ctx, past, new, table, free, P, 200)


def test_plan_strided_table_and_largest_lengths(ctx):
    big = torch.full((3, 40), -5, dtype=torch.int32, device="cuda")
    past, new = np.array([2 ** 31 - 1, 2 ** 31 - 20, 5], np.int32), np.array([1, 19, 2 ** 31 - 1], np.int32)
    r = ctx.page_plan(cu(past), cu(new), big[:, 3:20], cu(np.arange(50, dtype=np.int32)), 2 ** 28, 30)
    # 1 + 19 rows fit, then the third ends behind the buffer; the first is longer than an int32 holds
    assert r.status.cpu().tolist() == [1, 0, 4]
    assert r.kv_len.cpu().tolist() == [0, 2 ** 31 - 1, 0]
    assert r.pos.cpu().tolist()[1:20] == list(range(2 ** 31 - 20, 2 ** 31 - 1))
    assert r.slots.cpu().tolist()[1:20] == [-1] * 19  # its entry (7) is -5
    assert (big == -5).all()


# ---- RoPE and the paged store ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("S,P", [(1, 16), (5, 1), (40, 16), (1500, 64)])
def test_plan_pages_held_behind_the_cache(ctx, S, P):
    """Pages of rejected tokens stay the sequence's: its next tokens go into them before it takes new ones."""
    rng = np.random.default_rng(S)
    past, drafted, new = (rng.integers(0, 6 * P, S), rng.integers(0, 3 * P + 2, S), rng.integers(0, 4 * P, S))
    past, new = past.astype(np.int32), new.astype(np.int32)
    held = (-(-(past + drafted) // P)).astype(np.int32)
    held[::7] = rng.integers(-3, 1, len(held[::7]))  # fewer than the cache fills: the cache's count stands
    named = np.maximum(held, -(-past // P))
    cols = int(np.maximum(named, -(-(past + new) // P)).max()) + 1
    pool = rng.permutation(S * cols).astype(np.int32)
    table, at = np.full((S, cols), -7, np.int32), 0
    for s in range(S):
        table[s, :named[s]] = pool[at:at + named[s]]
        at += int(named[s])
    free, rows = pool[at:], int(new.sum()) + 2
    tb = cu(table)
    r = ctx.page_plan(cu(past), cu(new), tb, cu(free), P, rows, n_held=cu(held))
    torch.cuda.synchronize()
    want = R.plan(past, new, table, free, P, rows, held=held)
    for g, w in zip((tb, r.q_start, r.kv_len, r.pos, r.slots, r.status, r.n_taken), want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1))
    used = tb.cpu().numpy()  # no page twice
    used = used[used >= 0]
    assert len(np.unique(used)) == len(used)


@pytest.mark.parametrize("head", [-1, -2 ** 31, 2 ** 31 - 1])
def test_plan_heads_outside_the_list(ctx, head):
    """A sequence that needs no page keeps its rows; one that needs a page is refused."""
    table = np.array([[4, -1, -1], [9, 2, -1], [7, -1, -1]], np.int32)
    past, new = np.array([3, 17, 16], np.int32), np.array([5, 2, 1], np.int32)
    r = check_plan(ctx, past, new, table, np.arange(5, dtype=np.int32), 16, 9, head)
    assert r.status.cpu().tolist() == [0, 0, 2]


def test_plan_steps_that_take_turns(ctx):
    """Inputs and outputs side by side in one buffer, and each step's lengths from the step before, whose kv_len stays as it
    is: two plans in turn. The plan that holds this step's lengths is refused as its output."""
    rng = np.random.default_rng(17)
    S_, P, T, cols = 5, 16, 64, 30
    buf = torch.zeros(S_ + 2 * (3 * S_ + 2 + T), dtype=torch.int32, device="cuda")
    new, *parts = buf.split([S_, S_ + 1, S_, T, S_, 1, S_ + 1, S_, T, S_, 1])
    slots = torch.zeros(2, T, dtype=torch.int64, device="cuda")
    plans = [S.PagePlan(*parts[:3], slots[0], *parts[3:5]), S.PagePlan(*parts[5:8], slots[1], *parts[8:])]
    table = torch.full((S_, cols), -1, dtype=torch.int32, device="cuda")
    free, head = cu(rng.permutation(S_ * cols).astype(np.int32)), torch.zeros(1, dtype=torch.int32, device="cuda")
    ref, past, at = table.cpu().numpy(), np.zeros(S_, np.int64), 0
    for i in range(6):
        n = rng.integers(0, 13, S_).astype(np.int32)
        new.copy_(cu(n))
        before, pl = plans[(i + 1) % 2], plans[i % 2]
        ctx.page_plan(before.kv_len, new, table, free, P, T, free_head=head, out=pl)
        with pytest.raises(S.SrhpmError) as e:
            ctx.page_plan(pl.kv_len, new, table, free, P, T, free_head=head, out=pl)
        assert e.value.status == L.ERR_INVALID
        torch.cuda.synchronize()
        w = R.plan(past, n, ref, free.cpu().numpy(), P, T, at)
        for g, x in zip((table, pl.q_start, pl.kv_len, pl.pos, pl.slots, pl.status, pl.n_taken), w):
            assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(x).reshape(-1))
        ref, past, at = w[0], w[2], at + w[6]
        head += pl.n_taken


@pytest.mark.parametrize("kv,D,H,Hkv,P,n,qt", [
    (L.F16, 256, 24, 4, 64, 9, torch.float32), (L.F16, 128, 7, 7, 48, 33, torch.float16),
    (L.F16, 64, 5, 1, 16, 1, torch.float32), (L.Q8_0, 256, 6, 2, 32, 70, torch.float16),
    (L.Q8_0, 64, 3, 3, 16, 5, torch.float32), (L.Q8_0, 128, 32, 8, 80, 17, torch.float32),
    (L.F16, 128, 4, 2, 16, 3000, torch.float16)])
def test_store(ctx, kv, D, H, Hkv, P, n, qt):
    """Angles at far positions within the bound, keys stored from the turned rows, values bit for bit, everything else
    untouched. A turned value's error: angle 2^-23 turns * 2 pi at most, sine and cosine 2 ulp each, two products and a
    sum: under 2^-20 of |x_j| + |x_j'|."""
    rng = np.random.default_rng(n + D)
    row = D * 2 if kv == L.F16 else D // 32 * 34
    pages = -(-n // P) + 2
    x = rng.standard_normal((n, (H + 2 * Hkv) * D)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, n).astype(np.int32)
    pos[0] = 2 ** 31 - 1
    slots = rng.permutation(pages * P)[:n].astype(np.int64)
    slots[n // 2] = [-1, pages * P][n % 2]  # padding, or behind the cache
    base = 1e6
    kc0, vc0 = (rng.integers(0, 256, (pages, P, Hkv, row), dtype=np.uint8) for _ in range(2))
    kc, vc = cu(kc0), cu(vc0)
    wide = torch.zeros((n, (H + 2 * Hkv) * D + 4), device="cuda")  # rows with a stride of their own
    wide[:, 4:] = cu(x)
    qo = torch.zeros((n, H + 1, D), device="cuda", dtype=qt)[:, :H]
    ctx.rope_kv_paged(wide[:, 4:], cu(pos), cu(slots), kc, vc, kv, qo, theta_base=base)
    torch.cuda.synchronize()
    xs = x.reshape(n, H + 2 * Hkv, D)
    want = R.turn(xs[:, :H + Hkv], pos, base)
    tol = 2.0 ** -20 * (np.abs(xs[:, :H + Hkv]) + np.abs(np.roll(xs[:, :H + Hkv], D // 2, -1)))
    half = 2.0 ** -11 if qt == torch.float16 else 2.0 ** -24
    got = qo.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want[:, :H]) <= tol[:, :H] + half * np.abs(want[:, :H]) + 2.0 ** -25).all()
    assert np.array_equal(wide[:, 4:].cpu().numpy(), x)
    ok = (slots >= 0) & (slots < pages * P)
    at = slots[ok]
    gk, gv = kc.cpu().numpy().reshape(-1, Hkv, row), vc.cpu().numpy().reshape(-1, Hkv, row)
    assert np.array_equal(gv[at], O.cache_rows(kv, np.ascontiguousarray(xs[ok][:, H + Hkv:])))
    wk = want[ok][:, H:]
    if kv == L.F16:
        g = np.ascontiguousarray(gk[at]).view(np.float16).astype(np.float64)
        assert (np.abs(g - wk) <= tol[ok][:, H:] + 2.0 ** -11 * np.abs(wk) + 2.0 ** -25).all()
    else:  # half a step of the block's scale, one f16 rounding of that scale (2^-11 of 127 steps)
        step = np.abs(wk).reshape(wk.shape[:2] + (-1, 32)).max(-1).repeat(32, -1) / 127
        assert (np.abs(R.q8_values(gk[at]) - wk) <= step * (0.5 + 0.08 + 0.002) + tol[ok][:, H:]).all()
    rest = np.setdiff1d(np.arange(pages * P), at)
    assert np.array_equal(gk[rest], kc0.reshape(-1, Hkv, row)[rest])
    assert np.array_equal(gv[rest], vc0.reshape(-1, Hkv, row)[rest])


def test_store_modes_and_head_major_pages(ctx):
    """The context's q8_0 mode, and a cache whose pages hold [head][token]."""
    rng = np.random.default_rng(3)
    n, H, Hkv, D, P = 6, 2, 2, 256, 16
    x = (rng.integers(-3, 4, (n, (H + 2 * Hkv) * D)) * 0.5).astype(np.float32)  # ties of the rounding
    for mode in (L.Q8_0_ACT_REF, L.Q8_0_ACT_SIMD):
        kc, vc = (torch.zeros((2, Hkv, P, 272), dtype=torch.uint8, device="cuda").transpose(1, 2) for _ in range(2))
        ctx.set_q8_0_act_mode(mode)
        try:
            ctx.rope_kv_paged(cu(x), cu(np.zeros(n, np.int32)), cu(np.arange(14, 20)), kc, vc, L.Q8_0,
                              torch.zeros((n, H, D), device="cuda"))
        finally:
            ctx.set_q8_0_act_mode(L.Q8_0_ACT_SIMD)
        rows = x.reshape(n, -1, D)
        for c, w in ((kc, rows[:, H:H + Hkv]), (vc, rows[:, H + Hkv:])):  # position 0: keys are not turned
            got = c.cpu().numpy().reshape(2 * P, Hkv, 272)[14:20]
            assert np.array_equal(got, O.cache_rows(L.Q8_0, np.ascontiguousarray(w), mode))


def test_store_threads_with_bases_of_their_own(ctx):
    """Two host threads on one context, two streams, two bases: each gets its own angles every time."""
    import threading
    n, H, Hkv, D, P = 5, 2, 1, 64, 16
    x = torch.randn((n, (H + 2 * Hkv) * D), device="cuda")
    pos, slots = (torch.arange(n, device="cuda", dtype=t) for t in (torch.int32, torch.int64))
    kc, vc = (torch.zeros((4, P, Hkv, D * 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    bases = (1e4, 1e6)
    outs = [[torch.zeros((n, H, D), device="cuda") for _ in range(100)] for _ in bases]
    want = [ctx.rope_kv_paged(x, pos + 40000, slots, kc, vc, L.F16, torch.zeros((n, H, D), device="cuda"), theta_base=b)
            for b in bases]
    at = pos + 40000
    streams = [torch.cuda.Stream() for _ in bases]
    torch.cuda.synchronize()

    def run(i):
        for o in outs[i]:
            ctx.rope_kv_paged(x, at, slots, kc, vc, L.F16, o, theta_base=bases[i], stream=streams[i])

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ctx.check()
    for w, os_ in zip(want, outs):
        for o in os_:
            assert torch.equal(o, w)


# ---- attention over pages --------------------------------------------------------------------------------------------
def attn_case(rng, past, new, H, Hkv, D, P, kv, qt, poison=True, pad_rows=0, spread=1.0):
    """Caches whose slots behind each sequence hold NaN (f16) or huge steps, table entries behind it that are no page."""
    S_ = len(past)
    nb = [-(-(a + b) // P) for a, b in zip(past, new)]
    pages = sum(nb) + 2
    cols = max(max(nb), 1) + 1
    perm = rng.permutation(pages)
    table = np.full((S_, cols), -1, np.int32)
    if poison:
        table[:, :] = rng.choice([-1, 2 ** 31 - 1, -2 ** 31], (S_, cols))
    at, held = 0, np.zeros((pages, P), bool)
    for s in range(S_):
        table[s, :nb[s]] = perm[at:at + nb[s]]
        for b in range(nb[s]):
            held[perm[at + b], :max(0, min(P, past[s] + new[s] - b * P))] = True
        at += nb[s]
    caches, vals = [], []
    for _ in range(2):
        v = (rng.standard_normal((pages, P, Hkv, D)) * spread).astype(np.float16)
        if kv == L.F16:
            if poison:
                v[~held] = np.nan
            caches.append(v.view(np.uint8))
            vals.append(v)
        else:
            b = O.cache_rows(L.Q8_0, v.astype(np.float32).reshape(-1, Hkv, D)).reshape(pages, P, Hkv, -1).copy()
            if poison:
                b[~held] = 0x7f  # f16 0x7f7f is NaN
            caches.append(b)
            vals.append(R.q8_values(b))
    T = int(sum(new)) + pad_rows
    q = rng.standard_normal((T, H, D)).astype(np.float16 if qt == torch.float16 else np.float32)
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    kv_len = (np.array(past) + np.array(new)).astype(np.int32)
    return q, caches, vals, table, q_start, kv_len


def attn_check(got, q, vals, table, q_start, kv_len, scale, **kw):
    attn_bound(got, q, R.attention(q.astype(np.float64), np.nan_to_num(vals[0].astype(np.float64), posinf=0, neginf=0),
                                   np.nan_to_num(vals[1].astype(np.float64), posinf=0, neginf=0), table, q_start,
                                   kv_len, scale, **kw), q_start, kv_len)


def attn_bound(got, q, ref, q_start, kv_len):
    want, A, B = ref
    used = int(q_start[-1])
    D, n = q.shape[2], int(max(kv_len.max(), 1))
    e = (D / 8 + 2) * 2.0 ** -23 * B
    if q.dtype == np.float16:
        tol = A * (2 * e + 2.0 ** -21 + 3 * 2.0 ** -11) + 2.0 ** -25
    else:
        tol = A * (2 * (e + 2.0 ** -21 * B) + 2.0 ** -21 + 2.0 ** -21)
    tol = tol + A * (n / 16 + n / 64 + 4) * 2.0 ** -23 + 1e-30
    err = np.abs(got.astype(np.float64) - want)[:used]
    assert np.isfinite(got[:used]).all()
    worst = (err / tol[:used]).max() if used else 0.0
    assert worst <= 1.0, worst


def attn_run(ctx, case, kv, scale, **kw):
    q, caches, vals, table, q_start, kv_len = case
    out = torch.full(q.shape, 77.0, device="cuda", dtype=torch.float16 if q.dtype == np.float16 else torch.float32)
    ctx.flash_attn_paged(cu(q), cu(caches[0]), cu(caches[1]), kv, cu(table), cu(q_start), cu(kv_len), scale=scale,
                         out=out, **{k: cu(v) if k == "sinks" else v for k, v in kw.items()})
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[int(q_start[-1]):] == 77.0).all()  # padding rows as they were
    attn_check(got, q, vals, table, q_start, kv_len, scale, **kw)


SHAPES = [(L.F16, 256, 24, 4), (L.F16, 128, 8, 2), (L.F16, 64, 4, 4), (L.Q8_0, 256, 6, 2), (L.F16, 256, 3, 1),
          (L.F16, 128, 7, 1), (L.F16, 64, 16, 1)]


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D,H,Hkv", SHAPES)
@pytest.mark.parametrize("P,past,new", [
    (16, [0], [1]), (32, [127], [1]), (64, [128], [1]), (16, [255, 0, 31], [2, 1, 97]), (48, [130, 5], [9, 61]),
    (256, [500, 3], [1, 0]), (80, [0, 300, 63, 0], [0, 16, 65, 0])])
def test_attention_lengths(ctx, qt, kv, D, H, Hkv, P, past, new):
    rng = np.random.default_rng(D + H + P)
    case = attn_case(rng, past, new, H, Hkv, D, P, kv, qt, pad_rows=3)
    attn_run(ctx, case, kv, D ** -0.5)
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D,H,Hkv", SHAPES[:4])
@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (16, 0.0, True), (100, 5.0, False), (129, 0.0, False),
                                                 (100000, 30.0, True)])
def test_attention_window_softcap_sinks(ctx, qt, kv, D, H, Hkv, window, softcap, sink):
    rng = np.random.default_rng(window + D)
    case = attn_case(rng, [260, 0, 700], [3, 150, 1], H, Hkv, D, 32, kv, qt)
    kw = dict(window=window, softcap=softcap)
    if sink:
        kw["sinks"] = (rng.standard_normal(H) * 2).astype(np.float32)
    attn_run(ctx, case, kv, D ** -0.5, **kw)
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D,H,Hkv", SHAPES[:4])
def test_attention_long_rows_split(ctx, qt, kv, D, H, Hkv):
    """Caches long enough that a row's tokens are shared out and joined again; scores that rise along the cache."""
    rng = np.random.default_rng(D)
    case = attn_case(rng, [9000, 40], [2, 1], H, Hkv, D, 64, kv, qt, spread=1.0)
    attn_run(ctx, case, kv, D ** -0.5)
    q, caches, vals, table, q_start, kv_len = case
    attn_run(ctx, (q * 4,) + case[1:], kv, D ** -0.5)  # peaked rows: few tokens carry the sum
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,Hkv", [(64, 8, 2), (128, 8, 1), (128, 3, 3), (256, 12, 2), (64, 18, 2)])
@pytest.mark.parametrize("window,softcap,sink", [(0, 0.0, False), (1, 0.0, True), (100, 20.0, True), (5000, 0.0, True)])
def test_attention_few_rows(ctx, qt, D, H, Hkv, window, softcap, sink):
    """Decoding and short drafts: items of 3 to 18 rows side by side, empty caches, whole and cut items, with every mask."""
    rng = np.random.default_rng(D + H + window)
    case = attn_case(rng, [0, 5, 130, 0, 3000, 12000, 127], [1, 2, 1, 0, 2, 1, 1], H, Hkv, D, 16, L.F16, qt, pad_rows=2)
    kw = dict(window=window, softcap=softcap)
    if sink:
        kw["sinks"] = (rng.standard_normal(H) * 2).astype(np.float32)
        kw["sinks"][0] = -np.inf
    attn_run(ctx, case, L.F16, D ** -0.5, **kw)
    q, caches, vals, table, q_start, kv_len = case
    kv_len[1], kv_len[2] = 1, 0  # a row before position 0, a row that sees nothing
    caches = [np.nan_to_num(c.view(np.float16)).view(np.uint8) for c in caches]
    vals = [np.nan_to_num(v) for v in vals]
    attn_run(ctx, (q, caches, vals, table, q_start, kv_len), L.F16, D ** -0.5, **kw)
    ctx.check()


def test_attention_released_pages_before_the_window(ctx):
    """Pages wholly before the window are given away: their entries are no pages, and nothing of them is read."""
    rng = np.random.default_rng(5)
    P, W = 16, 40
    for kv, D in ((L.F16, 128), (L.Q8_0, 256)):
        case = attn_case(rng, [400, 1000], [4, 130], 4, 2, D, P, kv, torch.float16)
        q, caches, vals, table, q_start, kv_len = case
        held = table.copy()
        for s, past in enumerate((400, 1000)):
            first = max(0, past - W + 1)
            table[s, :first // P] = [-1, 2 ** 30][s]
            b, slot = held[s, first // P], first % P  # slots of the first kept page before the window
            for c in caches:
                c[b, :slot] = 0x7f
            for v in vals:
                v[b, :slot] = np.nan
        attn_run(ctx, (q, caches, vals, table, q_start, kv_len), kv, D ** -0.5, window=W)
        ctx.check()


def test_attention_rows_that_see_nothing(ctx):
    """kv_len smaller than the rows (the plan refused the sequence: 0; or a shorter cache): rows before position 0 give
    0, with sinks too."""
    rng = np.random.default_rng(6)
    q, caches, vals, table, q_start, kv_len = attn_case(rng, [0, 0, 50], [5, 140, 2], 4, 2, 128, 16, L.F16,
                                                        torch.float16)
    kv_len[0], kv_len[1] = 0, 133
    caches = [np.nan_to_num(c.view(np.float16)).view(np.uint8) for c in caches]
    vals = [np.nan_to_num(v) for v in vals]
    for kw in ({}, {"sinks": np.ones(4, np.float32)}):
        attn_run(ctx, (q, caches, vals, table, q_start, kv_len), L.F16, 0.1, **kw)
    ctx.check()


@pytest.mark.parametrize("kv,D", [(L.F16, 256), (L.F16, 128), (L.Q8_0, 256)])
def test_attention_entries_that_are_no_page(ctx, kv, D):
    """Inside the visible range: read as zeros, and the context's status says so."""
    rng = np.random.default_rng(7)
    q, caches, vals, table, q_start, kv_len = attn_case(rng, [300], [2], 4, 2, D, 16, kv, torch.float16, poison=False)
    table[0, 3], table[0, 9], table[0, 12] = -1, vals[0].shape[0], 2 ** 31 - 1
    attn_run(ctx, (q, caches, vals, table, q_start, kv_len), kv, D ** -0.5)
    with pytest.raises(S.SrhpmError) as e:
        ctx.check()
    assert e.value.status == L.ERR_DEVICE
    ctx.check()


@pytest.mark.parametrize("kv,D", [(L.F16, 128), (L.F16, 256), (L.Q8_0, 256)])
def test_attention_layouts(ctx, kv, D):
    """Pages of [head][token], queries as columns of wider rows, output rows with strides of their own."""
    rng = np.random.default_rng(8)
    H, Hkv, P = 6, 3, 32
    q, caches, vals, table, q_start, kv_len = attn_case(rng, [77, 10], [3, 40], H, Hkv, D, P, kv, torch.float16)
    T = q.shape[0]
    wide = torch.zeros((T, H + 2, D), device="cuda", dtype=torch.float16)
    wide[:, 1:H + 1] = cu(q)
    heads = [cu(c).transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    out = torch.full((T, H + 1, D), 7.0, device="cuda", dtype=torch.float16)
    tb = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    tb[:, 2:2 + table.shape[1]] = cu(table)
    ctx.flash_attn_paged(wide[:, 1:H + 1], heads[0], heads[1], kv, tb[:, 2:2 + table.shape[1]], cu(q_start),
                         cu(kv_len), scale=D ** -0.5, out=out[:, :H])
    torch.cuda.synchronize()
    attn_check(out[:, :H].cpu().numpy(), q, vals, table, q_start, kv_len, D ** -0.5)
    assert (out[:, H] == 7.0).all()
    ctx.check()


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D,H,Hkv,P,past,new,window", [
    (L.F16, 128, 32, 8, 48, [1326, 2666, 2194, 237, 153, 0, 1738], [13, 441, 297, 7, 229, 565, 1], 1024),
    (L.F16, 64, 8, 8, 16, [0, 3000, 10, 900] * 5, [700, 40, 1, 129] * 5, 0),
    (L.F16, 256, 24, 4, 64, [700, 5, 3000, 129], [300, 9, 1, 128], 0),
    (L.Q8_0, 256, 12, 4, 32, [700, 5, 3000, 129], [300, 9, 1, 128], 200),
    (L.F16, 128, 16, 8, 16, [0, 1, 2, 6000, 5000, 4000, 3000, 20] * 4, [1, 2, 3, 4, 1, 1, 9, 20] * 4, 0)])
def test_attention_many_tiles_per_cta(ctx, qt, kv, D, H, Hkv, P, past, new, window):
    """Far more tiles than SMs: every CTA takes several items of several tiles each, whole ones and cut ones, one row tile
    and two; ten times over, since what a slow warp meets depends on its timing."""
    rng = np.random.default_rng(D + P)
    q, caches, vals, table, q_start, kv_len = attn_case(rng, past, new, H, Hkv, D, P, kv, qt)
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    runs = [ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=D ** -0.5, window=window)
            for _ in range(10)]
    torch.cuda.synchronize()
    ctx.check()
    seqs = [[], []]
    for c, v in zip(seqs, vals):
        vt = cu(v)
        for s, L_ in enumerate(kv_len):
            pages = cu(table[s, :-(-int(L_) // P)].astype(np.int64))
            c.append(vt[pages].flatten(0, 1)[:int(L_)])
    ref = R.attention_dense(d[0], seqs[0], seqs[1], q_start, kv_len, D ** -0.5, window)
    attn_bound(runs[0].cpu().numpy(), q, ref, q_start, kv_len)
    for r in runs[1:]:
        assert torch.equal(r, runs[0])


@pytest.mark.parametrize("kv,qt,D,H,Hkv,past,new,window,shared", [
    (L.F16, torch.float32, 256, 24, 4, [16001], [1500], 0, 0), (L.F16, torch.float16, 256, 24, 4, [16001], [1500], 0, 0),
    (L.F16, torch.float32, 256, 24, 4, [16001], [1500], 9001, 0), (L.F16, torch.float16, 256, 24, 4, [16001], [1500], 9001, 0),
    (L.F16, torch.float16, 128, 32, 8, [15000, 3], [1501, 700], 0, 0), (L.F16, torch.float32, 128, 32, 8, [16001], [1500], 8999, 0),
    (L.F16, torch.float16, 64, 32, 16, [12345], [3000], 0, 0),
    (L.Q8_0, torch.float16, 256, 24, 4, [16001], [1500], 0, 0), (L.Q8_0, torch.float32, 256, 24, 4, [11000], [700], 9001, 0),
    (L.F16, torch.float32, 256, 24, 4, [8960 + 7 * i % 150 for i in range(90)], [1 + i % 3 for i in range(90)], 0, 8960),
    (L.F16, torch.float16, 256, 24, 4, [8960 + 7 * i % 150 for i in range(90)], [1 + i % 3 for i in range(90)], 0, 8960),
    (L.F16, torch.float16, 128, 32, 8, [8960 + 7 * i % 150 for i in range(60)], [1 + i % 2 for i in range(60)], 8300, 8960)])
def test_attention_turned_order(ctx, kv, qt, D, H, Hkv, past, new, window, shared):
    """Whole items of 64 tiles and more, whose tiles come in a turned order: the tile at the cache's end (or at the window's
    beginning), with NaN in the slots that no row sees, stands in the middle. Ten runs with the same bits. `shared`: the
    sequences' first tokens stand in the same pages."""
    rng = np.random.default_rng(D + H + window)
    P = 64
    sh = shared // P
    q, caches, vals, table, q_start, kv_len = attn_case(rng, [p - shared for p in past], new, H, Hkv, D, P, kv, qt)
    if sh:  # pages of the common beginning, in front of each sequence's own
        kv_len = kv_len + np.int32(shared)
        table = np.concatenate([np.tile(np.arange(sh, dtype=np.int32) + caches[0].shape[0], (len(past), 1)), table], 1)
        for i in range(2):
            v = rng.standard_normal((sh, P, Hkv, D)).astype(np.float16)
            caches[i], vals[i] = np.concatenate([caches[i], v.view(np.uint8)]), np.concatenate([vals[i], v])
    n_sm = torch.cuda.get_device_properties(0).multi_processor_count
    _, turned, inside = R.turned_items(q_start, kv_len, H, Hkv, D, kv == L.Q8_0, qt == torch.float32, window, n_sm)
    assert turned >= 20 and inside >= 20, (turned, inside)
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    runs = [ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=D ** -0.5, window=window)
            for _ in range(10)]
    torch.cuda.synchronize()
    ctx.check()
    seqs = [[], []]
    for c, v in zip(seqs, vals):
        vt = cu(v)
        for s, L_ in enumerate(kv_len):
            pages = cu(table[s, :-(-int(L_) // P)].astype(np.int64))
            c.append(vt[pages].flatten(0, 1)[:int(L_)])
    ref = R.attention_dense(d[0], seqs[0], seqs[1], q_start, kv_len, D ** -0.5, window)
    attn_bound(runs[0].cpu().numpy(), q, ref, q_start, kv_len)
    for r in runs[1:]:
        assert torch.equal(r, runs[0])


def test_attention_far_pages(ctx):
    """Pages behind 2^32 bytes of a pool."""
    P, Hkv, D, H = 64, 8, 128, 8
    pages = (1 << 32) // (P * Hkv * D * 2) + 40
    kc = torch.zeros((pages, P, Hkv, D), dtype=torch.float16, device="cuda")
    vc = torch.zeros((pages, P, Hkv, D), dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(9)
    use = [pages - 1, 0, pages - 30]
    small = [rng.standard_normal((3, P, Hkv, D)).astype(np.float16) for _ in range(2)]
    for c, v in ((kc, small[0]), (vc, small[1])):
        c[use] = cu(v)
    q = rng.standard_normal((5, H, D)).astype(np.float16)
    out = ctx.flash_attn_paged(cu(q), kc.view(torch.uint8), vc.view(torch.uint8), L.F16,
                               cu(np.array([use], np.int32)), cu(np.array([0, 5], np.int32)),
                               cu(np.array([150], np.int32)), scale=D ** -0.5)
    attn_check(out.cpu().numpy(), q, small, np.array([[0, 1, 2]]), np.array([0, 5]), np.array([150]), D ** -0.5)
    ctx.check()


def test_attention_many_sequences(ctx):
    rng = np.random.default_rng(10)
    n = 700
    past = rng.integers(0, 60, n).tolist()
    new = rng.integers(0, 3, n).tolist()
    case = attn_case(rng, past, new, 2, 1, 64, 16, L.F16, torch.float16, pad_rows=2)
    attn_run(ctx, case, L.F16, 0.125)
    ctx.check()


def test_attention_streams_and_replay(ctx):
    """Two calls at once on two streams, then captured once and replayed with other lengths, tables and rows."""
    rng = np.random.default_rng(11)
    a = attn_case(rng, [3000, 500], [4, 100], 8, 2, 128, 16, L.F16, torch.float16)
    b = attn_case(rng, [2000, 900], [90, 3], 8, 2, 128, 16, L.F16, torch.float16, pad_rows=11)
    outs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    dev = [[cu(x) for x in (c[0], c[1][0], c[1][1], c[3], c[4], c[5])] for c in (a, b)]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [ctx.flash_attn_paged(d[0], d[1], d[2], L.F16, d[3], d[4], d[5], scale=0.1, stream=s)
                for d, s in zip(dev, streams)]
    torch.cuda.synchronize()
    for o, c in zip(outs, (a, b)):
        attn_check(o.cpu().numpy(), c[0], c[2], c[3], c[4], c[5], 0.1)
    # replay: buffers of the larger case hold either one's data
    T, pages, cols = (max(x, y) for x, y in zip((a[0].shape[0], a[1][0].shape[0], a[3].shape[1]),
                                                (b[0].shape[0], b[1][0].shape[0], b[3].shape[1])))
    q = torch.zeros((T, 8, 128), dtype=torch.float16, device="cuda")
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
    ctx.flash_attn_paged(q, kc, vc, L.F16, tb, qs, kl, scale=0.1, out=out)
    with torch.cuda.graph(g):
        ctx.flash_attn_paged(q, kc, vc, L.F16, tb, qs, kl, scale=0.1, out=out)
    for c in (a, b, a):
        put(c)
        g.replay()
        torch.cuda.synchronize()
        attn_check(out.cpu().numpy()[:c[0].shape[0]], c[0], c[2], c[3], c[4], c[5], 0.1)
    ctx.check()


def test_attention_same_twice(ctx):
    """Two runs of one call give the same bits, split rows among them."""
    rng = np.random.default_rng(12)
    for kv, D in ((L.F16, 128), (L.Q8_0, 256)):
        q, caches, _, table, q_start, kv_len = attn_case(rng, [5000, 77], [9, 200], 6, 2, D, 48, kv, torch.float32)
        d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
        one, two = (ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=0.1) for _ in range(2))
        assert torch.equal(one, two)


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("kv,D", [(L.F16, 64), (L.F16, 128), (L.F16, 256), (L.Q8_0, 256)])
@pytest.mark.parametrize("past,new,at", [([300], [3], 301), ([9000, 40], [2, 1], 100), ([0], [500], 130), ([20000], [40], 7)])
def test_attention_nan_keys(ctx, qt, kv, D, past, new, at):
    """A NaN among the keys of KV head 0: the rows of its heads that see it are NaN, whole and cut items alike, all others
    keep their bits."""
    rng = np.random.default_rng(14)
    P, H, Hkv = 32, 4, 2
    q, caches, vals, table, q_start, kv_len = attn_case(rng, past, new, H, Hkv, D, P, kv, qt)
    d = [cu(x) for x in (q, caches[0], caches[1], table, q_start, kv_len)]
    clean = ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=0.1).cpu().numpy()
    d[1][int(table[0, at // P]), at % P, 0, :2] = 0x7e  # f16 0x7e7e: a value or a block's step
    got = ctx.flash_attn_paged(d[0], d[1], d[2], kv, d[3], d[4], d[5], scale=0.1).cpu().numpy()
    ctx.check()
    sees = np.zeros((q.shape[0], H, 1), bool)
    sees[max(0, at - past[0]):new[0], :H // Hkv] = True
    assert np.isnan(got[np.broadcast_to(sees, got.shape)]).all()
    keep = ~np.broadcast_to(sees, got.shape)
    assert np.array_equal(got[keep], clean[keep]) and np.isfinite(clean).all()


# ---- acceptance by sampling ------------------------------------------------------------------------------------------
def sample_case(rng, ks, V, draft=True, agree=True):
    T = int(sum(ks)) + len(ks)
    q_start = np.concatenate([[0], np.cumsum(np.array(ks) + 1)]).astype(np.int32)
    lg = rng.standard_normal((T, V)).astype(np.float32) * 2
    near = lg + 0.3 * rng.standard_normal((T, V)).astype(np.float32) if agree else rng.standard_normal((T, V)) * 2
    dp = np.exp(near - near.max(1, keepdims=True))
    dp = (dp / dp.sum(1, keepdims=True)).astype(np.float32)
    pick = np.array([rng.choice(V, p=p.astype(np.float64) / p.astype(np.float64).sum()) for p in dp])
    ids = np.zeros(T, np.int32)
    ids[1:] = pick[:-1]
    u, us = rng.random(T).astype(np.float32), rng.random(len(ks)).astype(np.float32)
    return lg, ids, q_start, u, us, dp if draft else None


def sample_check(ctx, lg, ids, q_start, u, us, dp=None, temp=None, ref_temp=None):
    T = lg.shape[0]
    out = (torch.full((T,), -9, dtype=torch.int32, device="cuda"), torch.full((len(q_start) - 1,), -9,
           dtype=torch.int32, device="cuda"), torch.full((T,), -9.0, device="cuda"))
    ctx.verify_sample(cu(lg), cu(ids), cu(q_start), cu(u), cu(us), draft_probs=None if dp is None else cu(dp),
                      temperature=None if temp is None else cu(temp), out=out)
    torch.cuda.synchronize()
    ctx.check()
    wi, wn, wp = R.sample(lg, ids, q_start, u, us, dp, temp if ref_temp is None else ref_temp)
    assert out[1].cpu().tolist() == wn
    assert out[0].cpu().tolist() == [-9 if i is None else i for i in wi]
    p = out[2].cpu().numpy()
    # exponential 2^-22 of its argument's rounding and its own, sums of positive terms in f32 or more: 2^-18
    for r, w in enumerate(wp):
        assert p[r] == -9.0 if w is None else abs(p[r] - w) <= 2.0 ** -18 * w + 1e-30, (r, p[r], w)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("V", [1, 2, 37, 1000, 4099, 151936])
def test_sample_sizes(ctx, V, draft):
    rng = np.random.default_rng(V)
    ks = [8, 0, 3] if V > 100000 else [8, 0, 3, 16, 1, 40]
    lg, ids, q_start, u, us, dp = sample_case(rng, ks, V, draft)
    sample_check(ctx, lg, ids, q_start, u, us, dp)
    temp = rng.uniform(0.2, 1.5, len(ks)).astype(np.float32)
    temp[0], temp[-1] = 0.0, -1.0
    sample_check(ctx, lg, ids, q_start, u, us, dp, temp)


@pytest.mark.parametrize("draft", [True, False])
def test_sample_edges(ctx, draft):
    """u of 0 and just below 1, masked tokens, rows of -inf, NaN and +inf, tokens outside the vocabulary, equal
    distributions, sequences without rows, padding rows."""
    rng = np.random.default_rng(1)
    V = 333
    lg, ids, q_start, u, us, dp = sample_case(rng, [4] * 12, V, draft)
    u[:10], us[:2], us[2:4] = 0.0, 0.0, np.nextafter(np.float32(1), np.float32(0))
    u[10:20] = us[2]
    lg[20:25, ::2] = -np.inf
    lg[25] = -np.inf
    lg[29] = -np.inf
    lg[30, 5:9] = np.inf
    lg[35, 3] = np.nan
    lg[36, 0] = np.nan
    lg[40] = 3.25
    lg[41, -1] = 300.0
    ids[46], ids[47] = V, -1
    if dp is not None:
        dp[50] = (np.exp(lg[50].astype(np.float64)) / np.exp(lg[50].astype(np.float64)).sum()).astype(np.float32)
        dp[41] = 0.0
    qs = np.concatenate([q_start[:1], q_start, q_start[-1:], q_start[-1:]]).astype(np.int32)  # empty ones around
    us2 = np.concatenate([[0.5], us, [0.5, 0.5]]).astype(np.float32)
    pad = np.zeros((3, V), np.float32)
    sample_check(ctx, np.concatenate([lg, pad]), np.concatenate([ids, [0, 0, 0]]).astype(np.int32), qs,
                 np.concatenate([u, [0, 0, 0]]).astype(np.float32), us2,
                 None if dp is None else np.concatenate([dp, pad]))


def test_sample_strided_rows_and_replay(ctx):
    rng = np.random.default_rng(2)
    V = 5003
    lg, ids, q_start, u, us, dp = sample_case(rng, [5, 2, 8], V)
    wide = torch.zeros((lg.shape[0], V + 6), device="cuda")
    wd = torch.zeros((lg.shape[0], V + 9), device="cuda")
    wide[:, 3:3 + V], wd[:, 1:1 + V] = cu(lg), cu(dp)
    d = [cu(x) for x in (ids, q_start, u, us)]
    ref = ctx.verify_sample(wide[:, 3:3 + V], d[0], d[1], d[2], d[3], draft_probs=wd[:, 1:1 + V])
    wi, wn, _ = R.sample(lg, ids, q_start, u, us, dp)
    assert ref[0].cpu().tolist() == wi and ref[1].cpu().tolist() == wn
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ctx.verify_sample(wide[:, 3:3 + V], d[0], d[1], d[2], d[3], draft_probs=wd[:, 1:1 + V])
    for seed in range(3):
        rng = np.random.default_rng(100 + seed)
        lg, ids, q_start, u, us, dp = sample_case(rng, [[5, 2, 8], [0, 15, 0], [7, 7, 1]][seed], V, agree=seed != 1)
        wide[:, 3:3 + V], wd[:, 1:1 + V] = cu(lg), cu(dp)
        for x, y in zip(d, (ids, q_start, u, us)):
            x.copy_(cu(y))
        g.replay()
        torch.cuda.synchronize()
        wi, wn, _ = R.sample(lg, ids, q_start, u, us, dp)
        assert out[0].cpu().tolist() == wi and out[1].cpu().tolist() == wn


def test_sample_frequencies(ctx):
    """The emitted first tokens of many one-draft sequences follow the target's distribution, whatever the drafter's:
    each count within 5 standard deviations of its mean (8 tokens: 5e-6 of such runs are outside by chance; the seed is
    fixed)."""
    rng = np.random.default_rng(3)
    n, V = 4096, 8
    lg1 = rng.standard_normal(V).astype(np.float32) * 1.5
    q1 = rng.random(V) + 0.05
    q1 = (q1 / q1.sum()).astype(np.float32)
    ids = np.zeros(2 * n, np.int32)
    ids[1::2] = rng.choice(V, n, p=q1.astype(np.float64) / q1.astype(np.float64).sum())
    lg, dp = np.tile(lg1, (2 * n, 1)), np.tile(q1, (2 * n, 1))
    out = ctx.verify_sample(cu(lg), cu(ids), cu(np.arange(0, 2 * n + 1, 2).astype(np.int32)),
                            cu(rng.random(2 * n).astype(np.float32)), cu(rng.random(n).astype(np.float32)),
                            draft_probs=cu(dp))
    got = np.bincount(out[0].cpu().numpy()[::2], minlength=V)
    p = np.exp(lg1.astype(np.float64))
    p /= p.sum()
    assert (np.abs(got - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_sample_temperatures(ctx):
    """From all weight on the maxima (two equal ones) to uniform. The bound of p holds at 1e-9 too: m / t log2 e there is
    rounded to 2^-20, which is the error of a weight's exponent."""
    rng = np.random.default_rng(4)
    temp = np.array([1e-3, 1e-5, 1e-7, 1e-9, 1e-20, 1e-37, 1e3, 1e20, 1e36, np.inf], np.float32)
    for draft in (True, False):
        lg, ids, q_start, u, us, dp = sample_case(rng, [3] * len(temp), 1500, draft)
        lg[:, 700] = lg[:, 90] = lg.max(1) + 0.5
        ids[1::2] = 700
        sample_check(ctx, lg, ids, q_start, u, us, dp, temp)


@pytest.mark.parametrize("V,ks,draft", [(151936, [2, 0, 3, 1, 2, 0], True), (151936, [2, 0, 3, 1, 2, 0], False),
                                        (5003, [3, 0, 4, 2, 1, 0] * 8, True), (5003, [3, 0, 4, 2, 1, 0] * 8, False),
                                        (1200007, [0] * 75, False)])
def test_sample_tokens_without_weight(ctx, V, ks, draft):
    """u_sample of 0 and rows that begin with tokens of weight 0 (masked, NaN, at the type's lowest value, far below the
    maximum at a low temperature): the first token that has a weight, never one of them."""
    rng = np.random.default_rng(V)
    T, S_ = sum(ks) + len(ks), len(ks)
    q_start = np.concatenate([[0], np.cumsum(np.array(ks) + 1)]).astype(np.int32)
    lg = rng.standard_normal((T, V), dtype=np.float32) * 2
    temp = np.array([1.0, 0.7, 0.01, 1.3, 2e-4, 1.0] * S_, np.float32)[:S_]
    lead = V * 2 // 3
    for s in range(S_):
        rows = slice(q_start[s], q_start[s + 1])
        # 200 below: 20000 t and more at the low temperatures. Elsewhere -inf, NaN, the lowest value
        lg[rows, :lead] = np.float32([-np.inf, np.nan, -200.0, np.finfo(np.float32).min, -200.0, -np.inf][s % 6])
        lg[rows, lead + 5 + s % 3] = 30.0  # weight of the low temperatures' rows
    ids = rng.integers(0, V, T).astype(np.int32)
    u = np.full(T, 0.5, np.float32)
    dp = None
    if draft:
        e = np.exp(np.nan_to_num(rng.standard_normal((T, V), dtype=np.float32)))
        dp = (e / e.sum(1, keepdims=True)).astype(np.float32)
    for us in (0.0, 2.0 ** -24, 0.5):
        sample_check(ctx, lg, ids, q_start, u, np.full(S_, us, np.float32), dp, temp)


@pytest.mark.parametrize("draft", [True, False])
def test_sample_high_temperatures_beside_masked_tokens(ctx, draft):
    """Temperatures up to infinity leave a masked token its weight of 0: (l - m) / t of -inf is -inf, and for an infinite
    t (a limit, taken at the largest f32: exp of 1e-36 at most is 1 in 64 bits) the others weigh the same."""
    rng = np.random.default_rng(21)
    temp = np.array([1e30, 1e35, 1e36, 1e37, 3e38, np.inf] * 2, np.float32)
    lg, ids, q_start, u, us, dp = sample_case(rng, [2] * 12, 30011, draft)
    lg[:, rng.permutation(30011)[:20000]] = -np.inf
    lg[:, :4000] = -np.inf
    lg[15:18, [5000, 20000]] = np.inf  # the weight stands on these alone, at t = inf too
    us[::3] = 0.0
    sample_check(ctx, lg, ids, q_start, u, us, dp, temp, np.minimum(temp, np.finfo(np.float32).max))


@pytest.mark.parametrize("V,rows,flat", [(20011, 48, False), (151936, 8, False), (700, 48, False), (151936, 6, True)])
def test_sample_drafter_equal_to_the_target(ctx, V, rows, flat):
    """The drafter's distribution is the target's but for the last places of its f32 values: two steps below p at one token,
    above p (by one step at least, 2^-24 of it) at all others. The replacement of the rejected token (its q is 2 p) can only be that token, whatever
    the random number: weights are told from 0 with the 64-bit sum, not with the f32 one of the acceptance. `flat`: all
    tokens but one at one distance from the maximum, at temperatures where that distance in f32 log2 units is off by
    more than 2^-19.7, and the f32 sum with it."""
    rng = np.random.default_rng(V)
    T = 2 * rows
    lg = rng.standard_normal((T, V)).astype(np.float32) * 3
    temp = rng.uniform(0.3, 1.5, rows).astype(np.float32)
    q_start = np.arange(0, T + 1, 2).astype(np.int32)
    ids, dp = np.zeros(T, np.int32), np.zeros((T, V), np.float32)
    only = rng.integers(0, V, rows)
    if flat:
        t = rng.uniform(0.9, 1.1, 20000).astype(np.float32)
        y = np.float32(-10.5) * (np.float32(1.4426950408889634) / t)
        off = np.log(2) * (y - -10.5 * 1.4426950408889634 / t.astype(np.float64))
        temp = t[np.argsort(-np.abs(off))[:rows]]
        assert np.sort(np.abs(off))[-rows] > 2.0 ** -19.7
        lg[:] = -3.0
        lg[:, 77777] = 7.5
    for s in range(rows):
        l = lg[2 * s].astype(np.float64)
        e = np.exp((l - l.max()) / float(temp[s]))
        p = e / e.sum()
        q = p.astype(np.float32)
        q = np.where(q < p, np.nextafter(q, np.float32(2)), q)  # p or above
        down = np.nextafter(np.nextafter(np.nextafter(q, np.float32(0)), np.float32(0)), np.float32(0))
        q = np.nextafter(q, np.float32(2))
        q[only[s]] = down[only[s]]
        x = int(l.argmax())
        if x == only[s]:
            x = (x + 1) % V
        q[x] *= 2
        ids[2 * s + 1], dp[2 * s] = x, q
    u, us = np.full(T, 0.9, np.float32), rng.random(rows).astype(np.float32)
    us[::4] = 0.0
    out = ctx.verify_sample(cu(lg), cu(ids), cu(q_start), cu(u), cu(us), draft_probs=cu(dp), temperature=cu(temp))
    assert out[1].cpu().tolist() == [1] * rows
    assert out[0].cpu().tolist()[::2] == only.tolist()


# ---- together --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,D", [(L.F16, 128), (L.Q8_0, 256)])
def test_steps_of_a_batch(ctx, kv, D):
    """Four steps of a batch as a server runs them, the whole step captured once: lengths -> plan -> RoPE and store ->
    attention -> logits -> acceptance -> new lengths. Every step's tables, cache, rows and tokens are held to the plain
    forms on the same inputs."""
    rng = np.random.default_rng(13)
    S_, H, Hkv, P, cols, T, V, pages = 3, 4, 2, 16, 12, 40, 211, 60
    i32 = dict(dtype=torch.int32, device="cuda")
    past, new = torch.zeros(S_, **i32), torch.zeros(S_, **i32)
    table, head = torch.full((S_, cols), -1, **i32), torch.zeros(1, **i32)
    free = cu(rng.permutation(pages).astype(np.int32))
    row = 2 * D if kv == L.F16 else D // 32 * 34
    kc, vc = (torch.full((pages, P, Hkv, row), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(2))
    qkv = torch.zeros((T, (H + 2 * Hkv) * D), device="cuda")
    q = torch.zeros((T, H, D), device="cuda")
    att = torch.zeros_like(q)
    Wv = cu((rng.standard_normal((H * D, V)) * 0.5).astype(np.float32))
    lg = torch.zeros((T, V), device="cuda")
    ids, u, us = torch.zeros(T, **i32), torch.zeros(T, device="cuda"), torch.zeros(S_, device="cuda")

    def step():
        pl = ctx.page_plan(past, new, table, free, P, T, free_head=head)
        ctx.rope_kv_paged(qkv, pl.pos, pl.slots, kc, vc, kv, q)
        ctx.flash_attn_paged(q, kc, vc, kv, table, pl.q_start, pl.kv_len, scale=D ** -0.5, out=att)
        torch.mm(att.view(T, H * D), Wv, out=lg)
        return pl, ctx.verify_sample(lg, ids, pl.q_start, u, us)

    step()
    torch.cuda.synchronize()
    table.fill_(-1)
    kc.fill_(0x7f)
    vc.fill_(0x7f)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pl, res = step()
    lens = np.zeros(S_, np.int64)
    ref_table, at = np.full((S_, cols), -1, np.int32), 0
    cache_k, cache_v = (np.zeros((pages, P, Hkv, D)) for _ in range(2))
    for n_new in ([20, 1, 7], [3, 4, 5], [1, 9, 0], [5, 5, 5]):
        x = rng.standard_normal((T, (H + 2 * Hkv) * D)).astype(np.float32)
        ids_n, u_n, us_n = rng.integers(0, V, T).astype(np.int32), rng.random(T).astype(np.float32), rng.random(S_).astype(np.float32)
        past.copy_(cu(lens.astype(np.int32)))
        new.copy_(cu(np.array(n_new, np.int32)))
        qkv.copy_(cu(x))
        ids.copy_(cu(ids_n))
        u.copy_(cu(u_n))
        us.copy_(cu(us_n))
        g.replay()
        torch.cuda.synchronize()
        w = R.plan(lens, n_new, ref_table, free.cpu().numpy(), P, T, at)
        ref_table = w[0]
        at += w[6]
        assert np.array_equal(table.cpu().numpy(), ref_table) and np.array_equal(pl.slots.cpu().numpy(), w[4])
        assert pl.status.cpu().tolist() == [0] * S_ and int(pl.n_taken) == w[6]
        head += pl.n_taken
        n = int(sum(n_new))
        xs = x.reshape(T, H + 2 * Hkv, D)[:n]
        got_q = q.cpu().numpy()[:n]
        wq = R.turn(xs[:, :H + Hkv], w[3][:n], 1e6)
        assert np.abs(got_q - wq[:, :H]).max() <= 2.0 ** -19 * np.abs(xs).max()
        pg, off = w[4][:n] // P, w[4][:n] % P
        raw = [c.cpu().numpy() for c in (kc, vc)]
        vals = [r.view(np.float16) if kv == L.F16 else R.q8_values(r) for r in raw]
        step_ = 2.0 ** -10 if kv == L.F16 else 1.0 / 127
        for have, rows in ((vals[0], wq[:, H:]), (vals[1], xs[:, H + Hkv:])):
            assert np.abs(have[pg, off].astype(np.float64) - rows).max() <= step_ * np.abs(rows).max()
        attn_check(att.cpu().numpy(), np.concatenate([got_q, np.zeros((T - n, H, D), np.float32)]), vals, ref_table,
                   w[1], w[2], D ** -0.5)
        si, sn, _ = R.sample(lg.cpu().numpy(), ids_n, w[1], u_n, us_n)
        assert res[0].cpu().tolist()[:n] == si[:n] and res[1].cpu().tolist() == sn
        lens += np.array(sn)
    ctx.check()


@pytest.mark.parametrize("kv,D", [(L.F16, 128), (L.Q8_0, 256)])
def test_steps_with_prompts_refusals_and_held_pages(ctx, kv, D):
    """The loop as the documents show it, captured once: prompts (only their last row is scored) beside drafts, a sequence that
    finds no rows and comes again, one that finds no page, pages of rejected tokens that stay with their sequence. Lengths
    and held pages are kept on the device and held to the host's."""
    rng = np.random.default_rng(19)
    S_, H, Hkv, P, cols, T, R_, V, pages = 4, 4, 2, 16, 12, 64, 24, 211, 11
    i32 = dict(dtype=torch.int32, device="cuda")
    n_past, n_new, held, head = (torch.zeros(n, **i32) for n in (S_, S_, S_, 1))
    prompt = torch.zeros(S_, dtype=torch.bool, device="cuda")
    table = torch.full((S_, cols), -1, **i32)
    free = cu(rng.permutation(pages).astype(np.int32))
    row = 2 * D if kv == L.F16 else D // 32 * 34
    kc, vc = (torch.full((pages, P, Hkv, row), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(2))
    qkv, ids = torch.zeros((T, (H + 2 * Hkv) * D), device="cuda"), torch.zeros(T, **i32)
    q = torch.zeros((T, H, D), device="cuda")
    att = torch.zeros_like(q)
    Wv = cu((rng.standard_normal((H * D, V)) * 0.5).astype(np.float32))
    u, us = torch.zeros(R_, device="cuda"), torch.zeros(S_, device="cuda")
    r = torch.arange(R_, device="cuda")

    def step():
        pl = ctx.page_plan(n_past, n_new, table, free, P, T, free_head=head, n_held=held)
        ctx.rope_kv_paged(qkv, pl.pos, pl.slots, kc, vc, kv, q)
        ctx.flash_attn_paged(q, kc, vc, kv, table, pl.q_start, pl.kv_len, scale=D ** -0.5, out=att)
        ok = pl.status == 0
        n_score = torch.where(ok, torch.where(prompt, n_new.clamp(max=1), n_new), 0)
        v_start = torch.nn.functional.pad(n_score.cumsum(0), (1, 0)).int()
        s = (torch.searchsorted(v_start, r, right=True) - 1).clamp(max=S_ - 1)
        rows = (pl.q_start[s + 1] - v_start[s + 1] + r).clamp(0, T - 1)
        logits = att.view(T, H * D)[rows] @ Wv
        out = ctx.verify_sample(logits, ids[rows], v_start, u, us)
        n_past.add_(torch.where(ok, n_new - n_score + out[1], 0))
        torch.maximum(held, (pl.kv_len + P - 1) // P, out=held)
        head.add_(pl.n_taken)
        return pl, out, logits, v_start, rows

    step()
    for t, v in ((n_past, 0), (held, 0), (head, 0), (table, -1), (kc, 0x7f), (vc, 0x7f)):
        t.fill_(v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pl, out, logits, v_start, rows = step()
    for t, v in ((n_past, 0), (held, 0), (head, 0), (table, -1), (kc, 0x7f), (vc, 0x7f)):
        t.fill_(v)
    lens, hold, ref_table, at, seen = np.zeros(S_, np.int64), np.zeros(S_, np.int64), np.full((S_, cols), -1, np.int32), 0, []
    for new, pr in (([30, 20, 17, 0], [1, 1, 1, 0]), ([14, 1, 17, 9], [0, 0, 1, 1]), ([5, 3, 6, 9], [0] * 4),
                    ([6, 5, 5, 5], [0] * 4), ([2, 40, 3, 1], [0, 1, 0, 0]), ([3, 4, 5, 9], [0] * 4)):
        x = rng.standard_normal((T, (H + 2 * Hkv) * D)).astype(np.float32)
        ids_n, u_n, us_n = rng.integers(0, V, T).astype(np.int32), rng.random(R_).astype(np.float32), rng.random(S_).astype(np.float32)
        u_n[:6] = 0.0  # some drafts are accepted
        for t, v in ((n_new, np.array(new, np.int32)), (prompt, np.array(pr, bool)), (qkv, x), (ids, ids_n), (u, u_n), (us, us_n)):
            t.copy_(cu(v))
        g.replay()
        torch.cuda.synchronize()
        w = R.plan(lens, new, ref_table, free.cpu().numpy(), P, T, at, hold)
        ref_table, q_start, kv_len, pos, slots, status = w[:6]
        at += w[6]
        seen += status.tolist()
        for a, b in ((table, ref_table), (pl.q_start, q_start), (pl.kv_len, kv_len), (pl.slots, slots), (pl.status, status)):
            assert np.array_equal(a.cpu().numpy(), b)
        raw = [c.cpu().numpy() for c in (kc, vc)]
        vals = [c.view(np.float16) if kv == L.F16 else R.q8_values(c) for c in raw]
        attn_check(att.cpu().numpy(), q.cpu().numpy(), vals, ref_table, np.minimum(q_start, T), kv_len, D ** -0.5)
        score = np.where(status == 0, np.where(np.array(pr, bool), np.minimum(new, 1), new), 0)
        starts = np.concatenate([[0], np.cumsum(score)])
        at_rows = np.concatenate([np.arange(q_start[s + 1] - score[s], q_start[s + 1]) for s in range(S_)])
        n = len(at_rows)
        assert np.array_equal(v_start.cpu().numpy(), starts) and np.array_equal(rows.cpu().numpy()[:n], at_rows)
        si, sn, _ = R.sample(logits.cpu().numpy()[:n], ids_n[at_rows], starts, u_n, us_n)
        assert out[0].cpu().tolist()[:n] == si and out[1].cpu().tolist() == sn
        lens += np.where(status == 0, np.array(new) - score + np.array(sn), 0)
        hold = np.maximum(hold, -(-kv_len // P))
        assert np.array_equal(n_past.cpu().numpy(), lens) and np.array_equal(held.cpu().numpy(), hold)
        # every page that was taken is some sequence's, and no page is two sequences'
        assert int(head) == at == int(hold.sum()) == int((ref_table >= 0).sum()) == len(np.unique(ref_table[ref_table >= 0]))
    assert {0, 2, 4} <= set(seen)
    ctx.check()
