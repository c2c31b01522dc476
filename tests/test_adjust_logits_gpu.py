"""Rules on logits (srhpm_adjust_logits) against the plain form in 64 bits. Roundings of a changed logit: the bias, the
division or product, the penalty (product and sum) and its subtraction, each to f32: 2^-24 of the value at hand, so 5 * 2^-24
of |l| + |bias| (times the repeat factor, where it multiplies) + the penalty."""
import numpy as np
import pytest
import torch

import share_ref as X
from test_paged_gpu import cu

pytestmark = pytest.mark.gpu


def rules(rng, ks, V, cap=200, last=None, bias=0, mask=False, pen=True, hot=50):
    """Rules of len(ks) sequences with ks[s] rows each."""
    S, T = len(ks), int(sum(ks))
    q_start = np.concatenate([[0], np.cumsum(ks)]).astype(np.int32)
    kw = {}
    if cap:
        kw["history"] = rng.integers(0, min(V, hot), (S, cap)).astype(np.int32)
        kw["n_history"] = rng.integers(0, cap + 1, S).astype(np.int32)
    if last is not None:
        kw["last_n"] = np.array([last[i % len(last)] for i in range(S)], np.int32)
    if pen:
        kw["repeat"] = (0.8 + rng.random(S)).astype(np.float32)
        kw["frequency"] = (rng.standard_normal(S) * 0.5).astype(np.float32)
        kw["presence"] = (rng.standard_normal(S) * 0.5).astype(np.float32)
    if bias:
        n = rng.integers(0, bias + 1, S)
        tok = rng.integers(0, V, int(n.sum())).astype(np.int32)
        tok[::3] %= min(V, hot)  # some of the history's tokens
        kw["bias"] = (np.concatenate([[0], np.cumsum(n)]).astype(np.int32), tok, rng.standard_normal(len(tok)).astype(np.float32) * 3)
    if mask:
        m = max(1, T // 2)
        kw["mask"] = rng.integers(-2 ** 31, 2 ** 31, (m, -(-V // 32) + 1)).astype(np.int32)
        kw["mask_row"] = rng.integers(-1, m + 1, T).astype(np.int32)  # m: no mask
    return rng.integers(0, min(V, hot), T).astype(np.int32), q_start, kw


def check(ctx, lg, ids, q_start, kw, in_place=False, pad=0, ld=None):
    T, V = lg.shape
    rows = T + pad
    wide = torch.full((rows, ld or V), 55.0, device="cuda")
    src = wide[:, :V]
    src[:T] = cu(lg)
    out = src if in_place else torch.full((rows, (ld or V) + (3 if ld else 0)), 77.0, device="cuda")[:, :V]
    dev = {k: tuple(cu(x) for x in v) if k == "bias" else cu(v) for k, v in kw.items()}
    if pad and "mask_row" in dev:
        dev["mask_row"] = torch.cat([dev["mask_row"], torch.zeros(pad, dtype=torch.int32, device="cuda")])
    i = torch.cat([cu(ids), torch.zeros(pad, dtype=torch.int32, device="cuda")])
    got = ctx.adjust_logits(src, i, cu(q_start), out=out, **dev)
    torch.cuda.synchronize()
    assert got is out
    assert (out[int(q_start[-1]):] == (55.0 if in_place else 77.0)).all()  # padding rows as they were
    if not in_place:
        assert np.array_equal(src[:T].cpu().numpy(), lg, equal_nan=True)
    if ld:
        assert (wide[:, V:] == 55.0).all()
    want = X.logits(lg, ids, q_start, **kw)
    g = out[:int(q_start[-1])].cpu().numpy().astype(np.float64)
    n = len(want)
    big = np.abs(lg[:n].astype(np.float64)) + 1.0
    scale = np.ones((n, 1))
    extra = np.zeros((n, 1))
    for s in range(len(q_start) - 1):
        a, b = q_start[s], q_start[s + 1]
        if "repeat" in kw:
            scale[a:b] = max(float(kw["repeat"][s]), 1 / float(kw["repeat"][s]), 1.0)
            count = (kw["n_history"][s] if "n_history" in kw else 0) + b - a
            extra[a:b] = count * abs(float(kw["frequency"][s])) + abs(float(kw["presence"][s]))
    if "bias" in kw and len(kw["bias"][2]):
        big = big + np.abs(kw["bias"][2]).max()
    tol = 5 * 2.0 ** -24 * (big * scale + extra)
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(g)) and np.array_equal(want[~fin & ~np.isnan(want)], g[~fin & ~np.isnan(want)])
    assert np.array_equal(np.isnan(want), np.isnan(g))
    assert (np.abs(g[fin] - want[fin]) <= tol[fin]).all()
    # what no rule touches keeps its bits
    same = want == lg[:n]
    assert np.array_equal(out[:n].cpu().numpy()[same], lg[:n][same])
    return out


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("V", [1, 2, 31, 33, 1003, 8191, 8192, 8193, 20011, 151936])
@pytest.mark.parametrize("ks", [[1], [9, 0, 3]])
def test_sizes(ctx, V, ks, in_place):
    rng = np.random.default_rng(V + len(ks))
    for kw in (dict(), dict(mask=True), dict(bias=30, pen=False, cap=0), dict(last=[64, 0, -1], bias=20, mask=True), dict(cap=0)):
        ids, q_start, r = rules(rng, ks, V, **kw)
        lg = (rng.standard_normal((len(ids), V)) * 4).astype(np.float32)
        check(ctx, lg, ids, q_start, r, in_place=in_place, pad=2)
    ctx.check()


@pytest.mark.parametrize("last", [[0], [1], [3, 500, -1], None, [2 ** 31 - 1, -2 ** 31]])
@pytest.mark.parametrize("cap", [0, 1, 700, 9000])
def test_windows(ctx, last, cap):
    """The window ends at the row's own token and reaches back into the history; histories that are empty, full or longer
    than they say; counts out of range are clamped."""
    rng = np.random.default_rng(cap + 3)
    ids, q_start, r = rules(rng, [4, 1, 9, 2], 3000, cap=cap, last=last)
    if cap:
        r["n_history"][:2] = [0, cap]
    check(ctx, (rng.standard_normal((16, 3000)) * 4).astype(np.float32), ids, q_start, r)
    if cap:
        want = dict(r, n_history=np.clip(r["n_history"], 0, cap))
        r["n_history"][0], want["n_history"][0] = -5, 0
        r["n_history"][2], want["n_history"][2] = cap + 9, cap
        lg = (rng.standard_normal((16, 3000)) * 4).astype(np.float32)
        a = ctx.adjust_logits(cu(lg), cu(ids), cu(q_start), **{k: cu(v) for k, v in r.items()})
        b = ctx.adjust_logits(cu(lg), cu(ids), cu(q_start), **{k: cu(v) for k, v in want.items()})
        assert torch.equal(a, b)
    ctx.check()


def test_strides_and_one_rule_at_a_time(ctx):
    rng = np.random.default_rng(5)
    for V, ld in ((1000, 1004), (1000, 1001), (999, 1024), (33, 35)):
        ids, q_start, r = rules(rng, [3, 5], V, bias=9, mask=True)
        lg = (rng.standard_normal((8, V)) * 4).astype(np.float32)
        for in_place in (False, True):
            check(ctx, lg, ids, q_start, r, in_place=in_place, ld=ld)
    for keep in (["repeat"], ["frequency"], ["presence"], ["history", "n_history"]):
        ids, q_start, r = rules(rng, [3, 5], 500)
        kw = {k: v for k, v in r.items() if k in keep + ["history", "n_history"]}
        full = dict(kw)
        S = 2
        if "repeat" in kw or "frequency" in kw or "presence" in kw:
            for k, d in (("repeat", 1.0), ("frequency", 0.0), ("presence", 0.0)):
                full.setdefault(k, np.full(S, d, np.float32))
        lg = (rng.standard_normal((8, 500)) * 4).astype(np.float32)
        a = ctx.adjust_logits(cu(lg), cu(ids), cu(q_start), **{k: cu(v) for k, v in kw.items()})
        b = ctx.adjust_logits(cu(lg), cu(ids), cu(q_start), **{k: cu(v) for k, v in full.items()})
        assert torch.equal(a, b)
        check(ctx, lg, ids, q_start, full)
    ctx.check()


def test_odd_tokens_and_values(ctx):
    """Tokens outside the vocabulary, a token biased twice (the later value counts), infinities and NaN, masks that leave
    nothing, rows without a mask row of their own."""
    rng = np.random.default_rng(6)
    V = 300
    ids, q_start, r = rules(rng, [4, 2, 3], V, bias=12, mask=True)
    r["history"][:, ::5] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31], r["history"][:, ::5].shape)
    ids[1] = -1
    start, tok, val = r["bias"]
    tok[1::2] = tok[::2][:len(tok[1::2])]
    tok[-1] = V
    r["bias"] = (start, tok, val)
    r["mask"][0] = 0
    r["mask_row"][:] = [0, -1, 1, 2, 4, 2 ** 31 - 1, -2 ** 31, 3, 0]
    lg = (rng.standard_normal((9, V)) * 4).astype(np.float32)
    lg[0, :40], lg[1, :40:3], lg[1, 1:40:3], lg[2, :20], lg[3, :50] = np.inf, -np.inf, np.inf, np.nan, -np.inf
    for in_place in (False, True):
        with np.errstate(invalid="ignore"):
            out = check(ctx, lg, ids, q_start, r, in_place=in_place)
        assert (out[0] == -np.inf).all() and (out[8] == -np.inf).all()
    lg[:] = 2.0
    lone = {"mask": np.zeros((9, 10), np.int32)}  # by rows
    lone["mask"][:, 0] = 1 << np.arange(9)
    out = check(ctx, lg, ids, q_start, lone)
    assert [int(x) for x in (out > 0).int().argmax(1)] == list(range(9))
    ctx.check()


def test_many_sequences_streams_and_replay(ctx):
    rng = np.random.default_rng(7)
    ks = rng.integers(0, 4, 1300).tolist()
    ids, q_start, r = rules(rng, ks, 700, cap=40, last=[16, 3, -1], bias=5, mask=True)
    lg = (rng.standard_normal((len(ids), 700)) * 4).astype(np.float32)
    check(ctx, lg, ids, q_start, r, pad=5)
    a, b = (rules(rng, [3, 4, 2], 5000, cap=64, last=[9], bias=20, mask=True) for _ in range(2))
    lgs = [(rng.standard_normal((9, 5000)) * 4).astype(np.float32) for _ in range(2)]

    def dev(c):
        return {k: tuple(cu(x) for x in v) if k == "bias" else cu(v) for k, v in c[2].items()}

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    d = [(cu(l), cu(c[0]), cu(c[1]), dev(c)) for l, c in zip(lgs, (a, b))]
    torch.cuda.synchronize()
    outs = [ctx.adjust_logits(x[0], x[1], x[2], stream=s, **x[3]) for x, s in zip(d, streams)]
    torch.cuda.synchronize()
    once = [ctx.adjust_logits(x[0], x[1], x[2], **x[3]) for x in d]
    for o, w in zip(outs, once):
        assert torch.equal(o, w)
    # captured in place, replayed with the other rows' data
    nb = max(len(c[2]["bias"][1]) for c in (a, b))
    buf = [x.clone() if torch.is_tensor(x) else x for x in d[0]]
    kw = {k: v.clone() if torch.is_tensor(v) else tuple(t.clone() for t in v) for k, v in buf[3].items()}
    kw["bias"] = (kw["bias"][0], torch.zeros(nb, dtype=torch.int32, device="cuda"), torch.zeros(nb, device="cuda"))
    ctx.adjust_logits(buf[0], buf[1], buf[2], out=buf[0], **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.adjust_logits(buf[0], buf[1], buf[2], out=buf[0], **kw)
    for x, w in zip(d, once):
        for t, v in zip(buf[:3], x[:3]):
            t.copy_(v)
        for k, v in x[3].items():
            if k == "bias":
                for t, u in zip(kw[k], v):
                    t[:len(u)].copy_(u)
            else:
                kw[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf[0], w)
    ctx.check()


def test_rules_then_acceptance(ctx):
    """As a step uses them: drafted tokens that a grammar forbids are not accepted, penalties shift what is, in place before
    the acceptance by sampling."""
    import paged_ref as P
    rng = np.random.default_rng(8)
    V, ks = 4001, [4, 2, 0, 3]
    rows = [k + 1 for k in ks]
    ids, q_start, r = rules(rng, rows, V, cap=100, last=[64, -1], bias=10, mask=True, hot=V)
    lg = (rng.standard_normal((len(ids), V)) * 3).astype(np.float32)
    for x in range(len(ids) - 1):
        lg[x, ids[x + 1]] += 14.0  # drafts that would be accepted
    r["mask_row"][:] = np.where(np.arange(len(ids)) % 4 == 1, 0, -1)
    r["mask"][0] = -1
    r["mask"][0, ids[2] // 32] &= ~np.int32(1 << (ids[2] % 32)) if ids[2] % 32 < 31 else np.int32(2 ** 31 - 1)
    u, us = (rng.random(len(ids)) * 0.5).astype(np.float32), rng.random(len(ks)).astype(np.float32)
    t = cu(lg)
    dev = {k: tuple(cu(x) for x in v) if k == "bias" else cu(v) for k, v in r.items()}
    ctx.adjust_logits(t, cu(ids), cu(q_start), out=t, **dev)
    oi, on, _ = ctx.verify_sample(t, cu(ids), cu(q_start), cu(u), cu(us))
    wi, wn, _ = P.sample(t.cpu().numpy(), ids, q_start, u, us)
    assert oi.cpu().tolist() == wi and on.cpu().tolist() == wn
    assert int(on[0]) == 2  # row 1 forbids its drafted token
    ctx.check()
