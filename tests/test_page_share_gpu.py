"""Pages that change hands (srhpm_page_fork, srhpm_page_copy, srhpm_page_free, srhpm_page_compact) against plain forms:
whole numbers and bytes, so everything has to be equal."""
import numpy as np
import pytest
import torch

import paged_ref as R
import share_ref as X
import srhpm_b200 as S
from srhpm_b200 import _lib as L
from test_paged_gpu import attn_check, cu

pytestmark = pytest.mark.gpu


def books(rng, n_rows, cols, held, spare=5, share=0.0):
    """A table whose rows hold held[s] pages, some of them the pages of the row before; counts, free list and head."""
    table, refs, at = np.full((n_rows, cols), -1, np.int32), None, 0
    own = []
    for s in range(n_rows):
        k = int(rng.integers(0, min(held[s], held[s - 1]) + 1)) if s and rng.random() < share else 0
        own.append(held[s] - k)
    pages = int(sum(own)) + spare
    perm, refs = rng.permutation(pages).astype(np.int32), np.zeros(pages, np.int32)
    for s in range(n_rows):
        k = held[s] - own[s]
        table[s, :k] = table[s - 1, :k]
        refs[table[s, :k]] += 1
        table[s, k:held[s]] = perm[at:at + own[s]]
        at += own[s]
    return table, refs, perm, at


def eq(*pairs):
    for i, (a, b) in enumerate(pairs):
        assert np.array_equal(a.cpu().numpy().reshape(-1), np.asarray(b).reshape(-1)), i


def fork_check(ctx, parent, child, keep, table, refs, free, P, head, wide=0):
    tb = torch.full((table.shape[0], table.shape[1] + wide), -9, dtype=torch.int32, device="cuda")
    tb[:, :table.shape[1]] = cu(table)
    rf = cu(refs)
    f = ctx.page_fork(cu(parent), cu(child), cu(keep), tb[:, :table.shape[1]], rf, cu(free), P,
                      free_head=None if head is None else cu(np.array([head], np.int32)))
    torch.cuda.synchronize()
    w = X.fork(parent, child, keep, table, refs, free, P, head or 0)
    eq((tb[:, :table.shape[1]], w[0]), (rf, w[1]), (f.src, w[2]), (f.dst, w[3]), (f.status, w[4]), (f.n_taken, w[5]))
    assert (tb[:, table.shape[1]:] == -9).all()
    return f, w


@pytest.mark.parametrize("n,parents,P,longest", [(1, 1, 16, 5), (3, 1, 16, 1000), (64, 24, 64, 900), (5, 2, 1, 40), (700, 60, 16, 300),
                                                 (2000, 7, 48, 20000), (33, 33, 256, 256)])
def test_fork(ctx, n, parents, P, longest):
    rng = np.random.default_rng(n + P)
    lens = rng.integers(0, longest + 1, parents)
    lens[0] = longest
    held = -(-lens // P)
    cols = int(held.max()) + 1
    table, refs, perm, at = books(rng, parents + n, cols, list(held) + [0] * n, spare=n + 3, share=0.3)
    refs += rng.integers(0, 3, len(refs)).astype(np.int32)
    parent = rng.integers(0, parents, n).astype(np.int32)
    child = (parents + rng.permutation(n)).astype(np.int32)
    keep = np.where(rng.random(n) < 0.5, lens[parent], rng.integers(0, lens[parent] + 1)).astype(np.int32)
    fork_check(ctx, parent, child, keep, table, refs, perm, P, at, wide=3)
    ctx.check()


def test_fork_refusals(ctx):
    """Negative lengths, rows the table lacks, a row forked from itself, too few entries, an empty list: these write nothing and
    take nothing, the others do; a list without room refuses every later fork that needs a page."""
    rng = np.random.default_rng(2)
    table, refs, perm, at = books(rng, 12, 6, [6, 4, 3] + [0] * 9, spare=3)
    parent = np.array([0, 1, -1, 12, 5, 0, 1, 2, 0, 1, 2], np.int32)
    child = np.array([3, 4, 6, 7, 5, 8, 9, 10, 12, -1, 11], np.int32)
    keep = np.array([16 * 6, -5, 3, 3, 3, 16 * 6 + 1, 17, 16, 3, 3, 2 ** 31 - 1], np.int32)
    for head in (at, at + 2, len(perm), len(perm) + 7, -1, -2 ** 31, 2 ** 31 - 1, None):
        fork_check(ctx, parent, child, keep, table, refs, perm, 16, head)
    parent, child = np.array([0, 1, 2, 0, 1, 2], np.int32), np.arange(3, 9, dtype=np.int32)
    keep = np.array([5, 16, 20, 7, 32, 9], np.int32)
    for head in range(len(perm) - 4, len(perm) + 2):
        fork_check(ctx, parent, child, keep, table, refs, perm, 16, head)
    f, _ = fork_check(ctx, parent, child, keep, table, refs, perm[:0], 16, None)
    assert f.status.cpu().tolist() == [2, 0, 2, 2, 0, 2]
    ctx.check()


def test_fork_entries_that_are_no_page(ctx):
    rng = np.random.default_rng(3)
    table, refs, perm, at = books(rng, 6, 5, [4, 4, 0, 0, 0, 0])
    table[0, 1], table[0, 2], table[1, 3] = -1, len(refs), 2 ** 31 - 1
    fork_check(ctx, np.array([0, 1, 0, 1], np.int32), np.array([2, 3, 4, 5], np.int32), np.array([60, 60, 40, 48], np.int32), table, refs,
               perm, 16, at)


# ---- copy ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,D,Hkv,P,layers", [(L.F16, 256, 4, 64, 3), (L.Q8_0, 64, 1, 16, 2), (L.Q4_0, 64, 1, 16, 1), (L.Q4_0, 128, 3, 48, 2),
                                               (L.F16, 64, 2, 1, 200), (L.Q8_0, 32, 3, 5, 2), (L.Q4_0, 32, 1, 1, 3)])
@pytest.mark.parametrize("layout", ["plain", "heads", "both", "padded"])
def test_copy(ctx, kv, D, Hkv, P, layers, layout):
    """Every type's rows, odd pages, pages of [head][token], K and V in one pool, rows and pages with gaps."""
    rng = np.random.default_rng(D + P)
    row, pages, n = L.load().srhpm_row_size(kv, D), 23, 9
    pools = []
    for _ in range(layers):
        if layout == "plain":
            pools += [torch.empty((pages, P, Hkv, row), dtype=torch.uint8, device="cuda") for _ in range(2)]
        elif layout == "heads":
            pools += [torch.empty((pages, Hkv, P, row), dtype=torch.uint8, device="cuda").transpose(1, 2) for _ in range(2)]
        elif layout == "both":
            p = torch.empty((pages, P, 2, Hkv, row), dtype=torch.uint8, device="cuda")
            pools += [p[:, :, 0], p[:, :, 1]]
        else:
            p = torch.empty((pages, P, Hkv + 1, row + 2), dtype=torch.uint8, device="cuda")
            pools += [p[:, :, :Hkv, :row]]
    whole = {id(p): p for p in pools}
    for p in whole.values():
        p.copy_(torch.randint(0, 256, p.shape, dtype=torch.uint8, device="cuda"))
    before = [p.clone() for p in pools]
    at = rng.permutation(pages)
    src, dst = at[:n].astype(np.int32), at[n:2 * n].astype(np.int32)
    src[2], dst[3], src[4], dst[5], dst[6] = -1, -1, pages, 2 ** 31 - 1, src[6]
    for moves in (None, 7, 0, -3, 100):
        for p, b in zip(pools, before):
            p.copy_(b)
        k = n if moves is None else min(max(moves, 0), n)
        ctx.page_copy(pools, kv, cu(src), cu(dst), n_moves=None if moves is None else cu(np.array([moves], np.int32)))
        torch.cuda.synchronize()
        for p, b in zip(pools, before):
            w = b.clone()
            for s, d in zip(src[:k], dst[:k]):
                if 0 <= s < pages and 0 <= d < pages:
                    w[d] = b[s]
            assert torch.equal(p, w)
    ctx.check()


def test_copy_leaves_the_gaps(ctx):
    """Bytes between rows and pages are nobody's."""
    p = torch.randint(0, 256, (9, 16, 5, 80), dtype=torch.uint8, device="cuda")
    b = p.clone()
    ctx.page_copy([p[:, :, 1:4, 4:76]], L.Q4_0, cu(np.array([0, 4], np.int32)), cu(np.array([8, 2], np.int32)))
    b[8, :, 1:4, 4:76], b[2, :, 1:4, 4:76] = b[0, :, 1:4, 4:76], b[4, :, 1:4, 4:76]
    assert torch.equal(p, b)


def test_copy_far_pages_and_many_pools(ctx):
    """Pages behind 2^32 bytes of a pool; more pools than one launch takes."""
    pages, P, Hkv, D = (1 << 32) // (64 * 8 * 256) + 9, 64, 8, 128
    p = torch.zeros((pages, P, Hkv, 2 * D), dtype=torch.uint8, device="cuda")
    p[3] = torch.randint(0, 256, p.shape[1:], dtype=torch.uint8, device="cuda")
    ctx.page_copy([p], L.F16, cu(np.array([3], np.int32)), cu(np.array([pages - 2], np.int32)))
    assert torch.equal(p[pages - 2], p[3]) and not p[pages - 1].any() and not p[pages - 3].any()
    del p
    many = torch.randint(0, 256, (600, 4, 16, 1, 36), dtype=torch.uint8, device="cuda")
    want = many.clone()
    want[:, 3] = many[:, 1]
    ctx.page_copy(list(many.unbind(0)), L.Q4_0, cu(np.array([1], np.int32)), cu(np.array([3], np.int32)))
    assert torch.equal(many, want)


# ---- free ------------------------------------------------------------------------------------------------------------
def free_check(ctx, rows, begin, end, table, refs, lst, head):
    tb, rf, fl = cu(table), cu(refs), cu(lst)
    n = ctx.page_free(cu(rows), None if begin is None else cu(begin), cu(end), tb, rf, fl, cu(np.array([head], np.int32)))
    torch.cuda.synchronize()
    w = X.free(rows, np.zeros(len(rows), int) if begin is None else begin, end, table, refs, lst, head)
    eq((tb, w[0]), (rf, w[1]), (fl, w[2]), (n, w[3]))
    return w


@pytest.mark.parametrize("S_,done,longest", [(1, 1, 1), (8, 3, 40), (1024, 48, 512), (300, 300, 300), (40, 0, 9), (5, 5, 3000)])
@pytest.mark.parametrize("share", [0.0, 0.6])
def test_free(ctx, S_, done, longest, share):
    """Sequences that are done, pages that others hold stay; every page of the list is somebody's or free afterwards."""
    rng = np.random.default_rng(S_ + done)
    held = rng.integers(0, longest + 1, S_)
    held[0] = longest
    table, refs, perm, at = books(rng, S_, longest + 1, held, share=share)
    rows = rng.permutation(S_)[:done].astype(np.int32)
    w = free_check(ctx, rows, None, held[rows].astype(np.int32), table, refs, perm, at)
    holders = np.bincount(w[0][w[0] >= 0], minlength=len(refs))
    listed = w[2][at - w[3]:]
    assert np.array_equal(np.sort(np.concatenate([np.nonzero(holders)[0], listed])), np.arange(len(refs)))
    assert np.array_equal(w[1], np.maximum(holders - 1, 0))
    ctx.check()


def test_free_ranges(ctx):
    """Parts of rows (before a window, behind a cache), a row twice, rows the table lacks, ranges that leave it."""
    rng = np.random.default_rng(4)
    table, refs, perm, at = books(rng, 9, 20, [20, 5, 0, 12, 20, 7, 1, 19, 20], share=0.5)
    table[3, 4], table[3, 5] = -1, len(refs)  # no pages
    rows = np.array([0, 0, 0, 1, 3, 4, -1, 9, 7, 2 ** 31 - 1, 5, 8], np.int32)
    begin = np.array([0, 3, 5, -4, 2, 19, 0, 0, 10, 0, 9, 2 ** 31 - 1], np.int32)
    end = np.array([5, 9, 9, 3, 8, 2 ** 31 - 1, 5, 5, 4, 5, 1, 2 ** 31 - 1], np.int32)
    free_check(ctx, rows, begin, end, table, refs, perm, at)
    ctx.check()


def test_free_more_than_was_taken(ctx):
    """A list without room in front of its head: what fits is written, the rest lost, and the status says so."""
    table, refs = np.arange(6, dtype=np.int32).reshape(1, 6), np.zeros(6, np.int32)
    for head, keep in ((2, [4, 5]), (0, []), (-5, [])):
        tb, rf, fl = cu(table), cu(refs), torch.full((8,), -7, dtype=torch.int32, device="cuda")
        n = ctx.page_free(cu(np.array([0], np.int32)), None, cu(np.array([6], np.int32)), tb, rf, fl, cu(np.array([head], np.int32)))
        assert int(n) == len(keep) and fl.cpu().tolist() == keep + [-7] * (8 - len(keep)) and (tb == -1).all()
        with pytest.raises(S.SrhpmError):
            ctx.check()
        ctx.check()


def test_free_many_pages(ctx):
    """Page numbers up to the limit, shared out among all CTAs."""
    pages = 1 << 22
    rng = np.random.default_rng(5)
    names = np.unique(np.concatenate([[0, pages - 1], rng.integers(0, pages, 5000)])).astype(np.int32)
    held = rng.permutation(names)[:5000].reshape(50, 100)
    refs = np.zeros(pages, np.int32)
    refs[held[::2, ::7]] = 1
    lst = np.full(pages, -3, np.int32)
    free_check(ctx, np.arange(50, dtype=np.int32), None, np.full(50, 100, np.int32), held, refs, lst, pages - 11)
    ctx.check()


# ---- compact ---------------------------------------------------------------------------------------------------------
def compact_check(ctx, table, held, refs, lst):
    tb, rf, fl = cu(table), cu(refs), cu(lst)
    n = len(refs)
    src, dst = (torch.full((max(n // 2, 1),), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    m = ctx.page_compact(tb, cu(held), rf, fl, out=(src, dst))
    torch.cuda.synchronize()
    w = X.compact(table, held, refs, lst)
    pad = [-5] * (len(src) - len(w[3]))
    eq((tb, w[0]), (rf, w[1]), (fl, w[2]), (src, w[3] + pad), (dst, w[4] + pad), (m.n_moves, [len(w[3])]), (m.n_used, [w[5]]))
    return w


@pytest.mark.parametrize("S_,longest,spare", [(1, 1, 0), (1, 0, 9), (8, 40, 100), (300, 60, 3), (48, 64, 4000), (3, 700, 1), (2, 5, 60000)])
@pytest.mark.parametrize("share", [0.0, 0.5])
def test_compact(ctx, S_, longest, spare, share):
    rng = np.random.default_rng(S_ + spare)
    held = rng.integers(0, longest + 1, S_)
    held[0] = longest
    table, refs, perm, _ = books(rng, S_, longest + 2, held, spare=max(spare, 1), share=share)
    gone = rng.random(S_) < 0.4  # given back before; their entries stay as they are
    left = np.where(gone, 0, held).astype(np.int32)
    w = compact_check(ctx, table, left, refs, perm)
    assert {int(p) for r, h in zip(w[0], left) for p in r[:h]} == set(range(w[5]))
    ctx.check()


def test_compact_odd_entries(ctx):
    """No pages among the entries, lengths that leave the table, every page in use, none."""
    rng = np.random.default_rng(6)
    table, refs, perm, _ = books(rng, 6, 10, [10, 3, 0, 8, 9, 1], spare=70)
    table[0, 2], table[3, 3], table[4, 0] = -1, len(refs), 2 ** 31 - 1
    compact_check(ctx, table, np.array([50, 3, -4, 8, 9, 2 ** 31 - 1], np.int32), refs, perm)
    compact_check(ctx, table, np.zeros(6, np.int32), refs, perm)
    full = rng.permutation(96).astype(np.int32).reshape(4, 24)
    compact_check(ctx, full, np.full(4, 24, np.int32), np.zeros(96, np.int32), np.arange(96, dtype=np.int32))
    ctx.check()


def test_compact_many_pages(ctx):
    pages = 1 << 22
    rng = np.random.default_rng(7)
    table = rng.choice(pages, 60000, replace=False).astype(np.int32).reshape(60, 1000)
    refs = np.zeros(pages, np.int32)
    refs[table[::3, ::3]] = 2
    compact_check(ctx, table, np.full(60, 1000, np.int32), refs, np.zeros(pages, np.int32))
    ctx.check()


# ---- together --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,D", [(L.F16, 128), (L.Q8_0, 256), (L.Q4_0, 128), (L.Q4_0, 256), (L.Q4_0, 64)])
def test_life_of_a_batch(ctx, kv, D):
    """A server's steps, captured as three graphs that replay with new data: a step of all sequences (plan, store, attention);
    forks of a prompt into branches with their page copies; branches that end, whose pages go back, and the pool compacted with the
    bytes moved. Books are held to the plain forms, and every attention to the tokens that the sequence's own history
    says are in its cache, whatever page they are in by now."""
    rng = np.random.default_rng(D)
    S_, H, Hkv, P, cols, T, pages = 5, 4, 2, 16, 9, 70, 40
    i32 = dict(dtype=torch.int32, device="cuda")
    past, new, held = (torch.zeros(S_, **i32) for _ in range(3))
    head, table, refs = torch.zeros(1, **i32), torch.full((S_, cols), -1, **i32), torch.zeros(pages, **i32)
    lst = cu(rng.permutation(pages).astype(np.int32))
    row = L.load().srhpm_row_size(kv, D)
    pools = [torch.full((pages, P, Hkv, row), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(2)]
    qkv, q = torch.zeros((T, (H + 2 * Hkv) * D), device="cuda"), torch.zeros((T, H, D), device="cuda")
    att = torch.zeros_like(q)
    parent, child, keep = (torch.zeros(2, **i32) for _ in range(3))
    rows, end = torch.zeros(2, **i32), torch.zeros(2, **i32)
    src, dst = (torch.full((pages // 2,), -1, **i32) for _ in range(2))

    def step():
        pl = ctx.page_plan(past, new, table, lst, P, T, free_head=head, n_held=held)
        ctx.rope_kv_paged(qkv, pl.pos, pl.slots, pools[0], pools[1], kv, q)
        ctx.flash_attn_paged(q, pools[0], pools[1], kv, table, pl.q_start, pl.kv_len, scale=D ** -0.5, out=att)
        past.copy_(pl.kv_len)
        torch.maximum(held, (pl.kv_len + P - 1) // P, out=held)
        head.add_(pl.n_taken)
        return pl

    def fork():
        f = ctx.page_fork(parent, child, keep, table, refs, lst, P, free_head=head)
        ctx.page_copy(pools, kv, f.src, f.dst)
        past.index_copy_(0, child.long(), keep)
        held.index_copy_(0, child.long(), (keep + P - 1) // P)
        head.add_(f.n_taken)
        return f

    def end_some():
        head.sub_(ctx.page_free(rows, None, end, table, refs, lst, head))
        past.index_fill_(0, rows.long(), 0)
        held.index_fill_(0, rows.long(), 0)
        m = ctx.page_compact(table, held, refs, lst, out=(src, dst))
        ctx.page_copy(pools, kv, m.src, m.dst, n_moves=m.n_moves)
        head.copy_(m.n_used)
        return m

    def clear():
        for t, v in ((past, 0), (new, 0), (held, 0), (head, 0), (table, -1), (refs, 0), (parent, 0), (keep, 0), (rows, 0), (end, 0),
                     *((p, 0x7f) for p in pools)):
            t.fill_(v)
        child.copy_(cu(np.array([3, 4], np.int32)))
        lst.copy_(cu(order))

    order = lst.cpu().numpy()
    graphs, outs = [], []
    for f in (step, fork, end_some):
        clear()
        f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    clear()
    told = [[np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))] for _ in range(S_)]  # each sequence's stored values
    b_table, b_refs, b_list, b_head = table.cpu().numpy(), refs.cpu().numpy(), lst.cpu().numpy(), 0
    lens, hold = np.zeros(S_, np.int64), np.zeros(S_, np.int64)

    def same():
        eq((table, b_table), (refs, b_refs), (lst, b_list), (head, [b_head]), (past, lens), (held, hold))
        ctx.check()

    def run_step(n_new):
        nonlocal b_table, b_head
        new.copy_(cu(np.array(n_new, np.int32)))
        x = rng.standard_normal((T, (H + 2 * Hkv) * D)).astype(np.float32)
        qkv.copy_(cu(x))
        graphs[0].replay()
        torch.cuda.synchronize()
        w = R.plan(lens, n_new, b_table, b_list, P, T, b_head, hold)
        b_table, q_start, kv_len = w[0], w[1], w[2]
        b_head += w[6]
        assert (w[5] == 0).all()
        lens[:] = kv_len
        hold[:] = np.maximum(hold, -(-kv_len // P))
        same()
        n = q_start[-1]
        pg, off = w[4][:n] // P, w[4][:n] % P
        raw = [p.cpu().numpy() for p in pools]
        vals = [r.view(np.float16) if kv == L.F16 else R.q8_values(r) if kv == L.Q8_0 else X.q4_values(r) for r in raw]
        for s in range(S_):
            a, b = q_start[s], q_start[s + 1]
            for i in range(2):
                told[s][i] = np.concatenate([told[s][i], vals[i][pg[a:b], off[a:b]].astype(np.float64)])
        # the sequences' own histories as pools of their own
        mine = [np.concatenate([np.concatenate([t[i], np.zeros((cols * P - len(t[i]), Hkv, D))]).reshape(cols, P, Hkv, D) for t in told])
                for i in range(2)]
        attn_check(att.cpu().numpy(), q.cpu().numpy(), mine, np.arange(S_ * cols).reshape(S_, cols), q_start, kv_len, D ** -0.5)

    def run_fork(pa, ch, ke):
        nonlocal b_table, b_refs, b_head
        for t, v in ((parent, pa), (child, ch), (keep, ke)):
            t.copy_(cu(np.array(v, np.int32)))
        graphs[1].replay()
        torch.cuda.synchronize()
        w = X.fork(pa, ch, ke, b_table, b_refs, b_list, P, b_head)
        b_table, b_refs = w[0], w[1]
        b_head += w[5]
        eq((outs[1].src, w[2]), (outs[1].dst, w[3]), (outs[1].status, w[4]))
        for p, c, k in zip(pa, ch, ke):
            told[c] = [t[:k].copy() for t in told[p]]
            lens[c], hold[c] = k, -(-k // P)
        same()

    def run_end(who):
        nonlocal b_table, b_refs, b_list, b_head
        rows.copy_(cu(np.array(who, np.int32)))
        end.copy_(cu(hold[who].astype(np.int32)))
        graphs[2].replay()
        torch.cuda.synchronize()
        w = X.free(who, [0, 0], hold[who], b_table, b_refs, b_list, b_head)
        for s in who:
            lens[s] = hold[s] = 0
            told[s] = [np.zeros((0, Hkv, D))] * 2
        w = X.compact(w[0], hold, w[1], w[2])
        b_table, b_refs, b_list, b_head = w[0], w[1], w[2], w[5]
        same()
        return len(w[3])

    run_step([37, 16, 0, 0, 0])
    run_fork([0, 1], [2, 3], [37, 16])  # a partly filled page is copied, a whole one shared
    run_step([1, 2, 3, 4, 0])
    run_step([20, 0, 9, 1, 30])
    moved = run_end([0, 4])
    run_step([50, 1, 1, 1, 0])
    moved += run_end([3, 1])
    run_fork([0, 2], [3, 1], [33, 20])
    run_step([3, 20, 5, 11, 1])
    moved += run_end([4, 0])
    run_fork([1, 2], [4, 0], [7, 0])
    run_step([1, 1, 1, 1, 1])
    moved += run_end([2, 3])
    run_step([9, 9, 9, 9, 9])
    assert moved > 0
