"""What the operators of q4_0 caches, of pages that change hands and of rules on logits refuse, through the C ABI and through
ops.Context, without a device: every check comes before anything touches the context or the GPU, so a block of zeros
stands in for a context."""
import ctypes

import numpy as np
import pytest
import torch

import share_ref as R
from srhpm_b200 import _lib as L
from srhpm_b200.ops import Context, _paged

lib = L.load()
_ctx = ctypes.create_string_buffer(8192)
CTX = ctypes.cast(_ctx, ctypes.c_void_p)
A = 1 << 20  # an aligned address that nothing reads
GAP = 1 << 16


def view(type_, ne, nb, data=A):
    ne, nb = list(ne) + [1] * (4 - len(ne)), list(nb) + [nb[-1]] * (4 - len(nb))
    return L.SrhpmTensor(type_, (ctypes.c_int64 * 4)(*ne), (ctypes.c_size_t * 4)(*nb), data)


def cache4(D=128, P=16, Hkv=3, n=10, data=A, **over):
    row = D // 32 * 18
    nb = [18, Hkv * row, row, P * Hkv * row]
    for k, v in over.items():
        nb[int(k[2])] = v
    return view(L.Q4_0, [D, P, Hkv, n], nb, data)


def rows(D=128, T=9, H=6, type_=L.F16, head_first=False):
    e = 2 if type_ == L.F16 else 4
    ne = [D, H, T] if head_first else [D, T, H]
    return view(type_, ne + [1], [e, D * e, H * D * e, T * H * D * e] if head_first else [e, H * D * e, D * e, T * H * D * e])


def table(cols=8, S=2, data=A, nb1=None, type_=L.I32):
    return view(type_, [cols, S], [4, nb1 if nb1 is not None else cols * 4], data)


def test_type_facts():
    assert lib.srhpm_blck_size(L.Q4_0) == 32 and lib.srhpm_type_size(L.Q4_0) == 18 and lib.srhpm_row_size(L.Q4_0, 256) == 144
    w = np.ones((2, 64), np.float32)
    out = np.zeros(4096, np.uint8)
    assert lib.srhpm_quantize_chunk(L.Q4_0, w.ctypes.data, out.ctypes.data, 0, 2, 64, None) == 0  # no weight type
    W, X = view(L.Q4_0, [256, 8], [18, 144]), view(L.F32, [256, 1], [4, 1024])
    size = ctypes.c_size_t()
    assert lib.srhpm_mul_mat_work_size(ctypes.byref(W), ctypes.byref(X), ctypes.byref(size)) == L.UNSUPPORTED


def attn(D=128, k=None, v=None, q=None, tb=None, cols=8, T=9, H=6):
    q = q or rows(D=D, T=T, H=H)
    k, v, tb = k or cache4(D=D), v or cache4(D=D), tb or table(cols=cols)
    return lib.srhpm_flash_attn_paged(CTX, ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), ctypes.byref(tb), A, A, None, 0.1, 0.0, 0,
                                      ctypes.byref(rows(D=D, T=q.ne[1], H=q.ne[2], head_first=True)), A, 0, None)


@pytest.mark.parametrize("o,st", [
    (dict(k=cache4(data=A + 4)), L.ERR_ALIGN), (dict(k=cache4(nb1=220)), L.ERR_ALIGN),
    (dict(k=cache4(nb2=76)), L.ERR_ALIGN), (dict(v=cache4(nb2=64)), L.ERR_INVALID),
    (dict(D=64, k=cache4(D=64, data=A + 2)), L.ERR_ALIGN), (dict(D=256, k=cache4(D=256, data=A + 8)), L.ERR_ALIGN),
    (dict(D=96), L.UNSUPPORTED), (dict(k=cache4(P=24), v=cache4(P=24)), L.UNSUPPORTED),
    (dict(v=view(L.Q8_0, [128, 16, 3, 10], [34, 408, 136, 6528])), L.UNSUPPORTED),
    # rows of a KV head and tiles of 8 of them
    (dict(q=rows(T=1 << 24, H=1536), k=cache4(), v=cache4()), L.UNSUPPORTED), (dict(q=rows(T=1 << 24), cols=1 << 13), L.UNSUPPORTED)])
def test_flash_attn_paged(o, st):
    assert attn(**o) == st


def test_q4_strides_that_are_fine_for_their_rows():
    """Rows of 36 and 72 bytes need their copies' alignment only; without a work buffer that is what the call stops at."""
    lib_st = [attn(D=64, k=cache4(D=64, data=A + 4), v=cache4(D=64, data=A + 4)), attn(D=128, k=cache4(data=A + 8), v=cache4())]
    assert lib_st == [L.ERR_WORKSPACE] * 2


def store(k=None, v=None, W=(6 + 6) * 128):
    k, v = k or cache4(), v or cache4()
    return lib.srhpm_rope_kv_paged(CTX, ctypes.byref(view(L.F32, [W, 9], [4, W * 4])), 6, 3, A, A, 1e6, ctypes.byref(rows()),
                                   ctypes.byref(k), ctypes.byref(v), None)


@pytest.mark.parametrize("o,st", [
    (dict(k=cache4(data=A + 1)), L.ERR_ALIGN), (dict(v=cache4(nb1=217)), L.ERR_ALIGN), (dict(v=cache4(nb1=70)), L.ERR_INVALID),
    (dict(v=cache4(n=9)), L.ERR_INVALID), (dict(v=view(L.F16, [128, 16, 3, 10], [2, 768, 256, 12288])), L.UNSUPPORTED),
    (dict(k=cache4(D=96), v=cache4(D=96)), L.UNSUPPORTED)])
def test_rope_kv_paged(o, st):
    assert store(**o) == st


def places(names):
    return {n: A + GAP * (i + 1) for i, n in enumerate(names)}


FORK = dict(parent=12, child=12, keep=12, table=64, refs=40, free=20, head=4, src=12, dst=12, status=12, taken=4)


def fork(n=3, P=16, tb=None, n_pages=10, n_free=5, **at):
    p = places(FORK) | at
    tb = tb or table(data=p["table"])
    return lib.srhpm_page_fork(CTX, p["parent"], p["child"], p["keep"], n, P, ctypes.byref(tb), p["refs"], n_pages, p["free"], n_free,
                               p["head"], p["src"], p["dst"], p["status"], p["taken"], None)


@pytest.mark.parametrize("o,st", [
    (dict(parent=None), L.ERR_INVALID), (dict(child=None), L.ERR_INVALID), (dict(keep=None), L.ERR_INVALID), (dict(refs=None), L.ERR_INVALID),
    (dict(src=None), L.ERR_INVALID), (dict(dst=None), L.ERR_INVALID), (dict(status=None), L.ERR_INVALID), (dict(taken=None), L.ERR_INVALID),
    (dict(n=0), L.ERR_INVALID), (dict(n=8193, src=1 << 24, dst=1 << 25, status=1 << 26), L.UNSUPPORTED), (dict(P=0), L.ERR_INVALID),
    (dict(n_pages=0), L.ERR_INVALID), (dict(n_free=-1), L.ERR_INVALID), (dict(free=None), L.ERR_INVALID),
    (dict(tb=table(type_=L.F32)), L.ERR_INVALID), (dict(tb=table(nb1=30)), L.ERR_ALIGN), (dict(tb=table(data=0)), L.ERR_INVALID)])
def test_page_fork(o, st):
    assert fork(**o) == st


FREE = dict(rows=12, begin=12, end=12, table=64, refs=40, free=40, head=4, freed=4)


def free(n=3, tb=None, n_pages=10, n_free=10, **at):
    p = places(FREE) | at
    tb = tb or table(data=p["table"])
    return lib.srhpm_page_free(CTX, p["rows"], p["begin"], p["end"], n, ctypes.byref(tb), p["refs"], n_pages, p["free"], n_free,
                               p["head"], p["freed"], None)


@pytest.mark.parametrize("o,st", [
    (dict(rows=None), L.ERR_INVALID), (dict(end=None), L.ERR_INVALID), (dict(refs=None), L.ERR_INVALID), (dict(head=None), L.ERR_INVALID),
    (dict(freed=None), L.ERR_INVALID), (dict(n=-1), L.ERR_INVALID), (dict(n_pages=0), L.ERR_INVALID), (dict(n_free=-1), L.ERR_INVALID),
    (dict(free=None), L.ERR_INVALID), (dict(tb=table(type_=L.F32)), L.ERR_INVALID), (dict(n_pages=(1 << 22) + 1), L.UNSUPPORTED)])
def test_page_free(o, st):
    assert free(**o) == st


COMPACT = dict(table=64, held=8, refs=40, free=40, src=20, dst=20, moves=4, used=4)


def compact(tb=None, n_pages=10, **at):
    p = places(COMPACT) | at
    tb = tb or table(data=p["table"])
    return lib.srhpm_page_compact(CTX, ctypes.byref(tb), p["held"], p["refs"], n_pages, p["free"], p["src"], p["dst"], p["moves"], p["used"],
                                  None)


@pytest.mark.parametrize("o,st", [
    (dict(held=None), L.ERR_INVALID), (dict(refs=None), L.ERR_INVALID), (dict(free=None), L.ERR_INVALID), (dict(src=None), L.ERR_INVALID),
    (dict(dst=None), L.ERR_INVALID), (dict(moves=None), L.ERR_INVALID), (dict(used=None), L.ERR_INVALID), (dict(n_pages=0), L.ERR_INVALID),
    (dict(tb=table(nb1=2)), L.ERR_ALIGN), (dict(n_pages=(1 << 22) + 1), L.UNSUPPORTED)])
def test_page_compact(o, st):
    assert compact(**o) == st


CALLS = [(fork, FORK, ("parent", "child", "keep", "free", "head")), (free, FREE, ("rows", "begin", "end", "head")),
         (compact, COMPACT, ("held",))]


@pytest.mark.parametrize("call,sizes,inputs", CALLS)
def test_outputs_that_share_memory(call, sizes, inputs):
    """Every output against every other vector: one byte too many at either end."""
    at = places(sizes)
    for o in sizes:
        if o in inputs:
            continue
        for v in sizes:
            if v == o:
                continue
            for where in (at[v], at[v] + 4 - sizes[o], at[v] + sizes[v] - 4):
                assert call(**{o: where}) == L.ERR_INVALID, (o, v, where - at[v])


def copy(caches, n=2, src=A, dst=A, count=None):
    arr = (L.SrhpmTensor * max(len(caches), 1))(*caches)
    return lib.srhpm_page_copy(CTX, ctypes.byref(arr), len(caches) if count is None else count, src, dst, n, None, None)


@pytest.mark.parametrize("o,st", [
    (dict(caches=[], count=0), L.ERR_INVALID), (dict(caches=[cache4()], n=-1), L.ERR_INVALID), (dict(caches=[cache4()], src=None), L.ERR_INVALID),
    (dict(caches=[cache4()], dst=None), L.ERR_INVALID), (dict(caches=[cache4(), cache4(n=9)]), L.ERR_INVALID),
    (dict(caches=[cache4(), cache4(nb1=432)]), L.ERR_INVALID), (dict(caches=[cache4(nb1=217)]), L.ERR_ALIGN),
    (dict(caches=[cache4(data=A + 1)]), L.ERR_ALIGN), (dict(caches=[cache4(), cache4(data=0)]), L.ERR_INVALID),
    (dict(caches=[cache4(), view(L.F16, [128, 16, 3, 10], [2, 768, 256, 12288])]), L.ERR_INVALID),
    (dict(caches=[view(L.F32, [128, 16, 3, 10], [4, 1536, 512, 24576])]), L.UNSUPPORTED),
    (dict(caches=[view(L.Q8_0, [40, 16, 3, 10], [34, 408, 136, 6528])]), L.ERR_INVALID),
    (dict(caches=[cache4(nb2=36)]), L.ERR_INVALID), (dict(caches=[cache4()], n=0, src=None, dst=None), L.OK)])
def test_page_copy(o, st):
    assert copy(**o) == st


LOGITS = dict(logits=1 << 15, ids=20, q_start=12, history=64, n_history=8, last_n=8, repeat=8, frequency=8, presence=8, starts=12,
              tokens=16, values=16, mask=2560, mask_row=20, out=1 << 15)


def adjust(S=2, T=5, V=1000, n_bias=4, ov=None, lv=None, hist=None, mask=None, **at):
    p = {n: (1 << 24) + (1 << 20) * (i + 1) for i, n in enumerate(LOGITS)} | at
    lv = lv or view(L.F32, [V, T], [4, 4 * V], p["logits"])
    ov = ov or view(L.F32, [V, T], [4, 4 * V], p["out"])
    hist = hist or (table(cols=8, S=2, data=p["history"]) if p["history"] else None)
    mask = mask or (table(cols=32, S=20, data=p["mask"]) if p["mask"] else None)
    return lib.srhpm_adjust_logits(CTX, ctypes.byref(lv), p["ids"], p["q_start"], S, ctypes.byref(hist) if hist else None, p["n_history"],
                                   p["last_n"], p["repeat"], p["frequency"], p["presence"], p["starts"], p["tokens"], p["values"], n_bias,
                                   ctypes.byref(mask) if mask else None, p["mask_row"], ctypes.byref(ov), None)


@pytest.mark.parametrize("o,st", [
    (dict(ids=None), L.ERR_INVALID), (dict(q_start=None), L.ERR_INVALID), (dict(S=0), L.ERR_INVALID), (dict(S=(1 << 24) + 1), L.ERR_INVALID),
    (dict(n_bias=-1), L.ERR_INVALID), (dict(starts=None), L.ERR_INVALID), (dict(tokens=None), L.ERR_INVALID), (dict(values=None), L.ERR_INVALID),
    (dict(n_history=None), L.ERR_INVALID), (dict(hist=table(S=3)), L.ERR_INVALID), (dict(hist=table(type_=L.F32)), L.ERR_INVALID),
    (dict(mask=table(cols=31, S=20)), L.ERR_INVALID), (dict(mask=table(cols=32, S=4), mask_row=None), L.ERR_INVALID),
    (dict(lv=view(L.F16, [1000, 5], [2, 2000])), L.ERR_INVALID), (dict(ov=view(L.F32, [1000, 4], [4, 4000])), L.ERR_INVALID),
    (dict(ov=view(L.F32, [999, 5], [4, 4000])), L.ERR_INVALID), (dict(ov=view(L.F32, [1000, 5], [4, 3996])), L.ERR_INVALID),
    (dict(lv=view(L.F32, [1 << 29, 1 << 16], [4, 1 << 31]), ov=view(L.F32, [1 << 29, 1 << 16], [4, 1 << 31], 1 << 50),
          mask=table(cols=1 << 24, S=20)), L.UNSUPPORTED)])
def test_adjust_logits(o, st):
    assert adjust(**o) == st


def test_adjust_logits_output_that_shares_memory():
    at = {n: (1 << 24) + (1 << 20) * (i + 1) for i, n in enumerate(LOGITS)}
    size = 4 * 5000
    for v, n in LOGITS.items():
        if v == "out":
            continue
        n = size if v == "logits" else n
        for where in (at[v] + 4 - size, at[v] + n - 4):
            assert adjust(out=where) == L.ERR_INVALID, v
    wide = view(L.F32, [1000, 5], [4, 4096], at["logits"])  # the logits' place, other strides
    assert adjust(ov=wide) == L.ERR_INVALID


def test_python_layer():
    with pytest.raises(ValueError):
        _paged(torch.zeros((2, 16, 4, 70), dtype=torch.uint8), L.Q4_0)
    c = Context.__new__(Context)
    c._index, c.handle = -1, None  # tensors of the host are this context's

    def raises(f):
        with pytest.raises(ValueError):
            f()

    i = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    c.lib = lib
    c._new = lambda shape, dtype, stream: torch.empty(shape, dtype=dtype)
    raises(lambda: c.page_fork(i(3), i(2), i(3), i(4, 5), i(9), i(9), 16))
    raises(lambda: c.page_fork(i(3), i(3), i(3).long(), i(4, 5), i(9), i(9), 16))
    raises(lambda: c.page_fork(i(3), i(3), i(3), i(5, 4).t(), i(9), i(9), 16))
    raises(lambda: c.page_free(i(3), None, i(2), i(4, 5), i(9), i(9), i(1)))
    raises(lambda: c.page_free(i(3), None, i(3), i(4, 5), i(9).long(), i(9), i(1)))
    raises(lambda: c.page_compact(i(4, 5), i(3), i(9), i(9)))
    raises(lambda: c.page_compact(i(4, 5), i(4), i(9), i(8)))  # a list of all pages
    raises(lambda: c.page_compact(i(4, 5), i(4), i(9), i(9), out=(i(3), i(4))))
    raises(lambda: c.page_copy([torch.zeros((2, 16, 4, 71), dtype=torch.uint8)], L.Q8_0, i(1), i(1)))
    raises(lambda: c.page_copy([torch.zeros((2, 16, 4, 72), dtype=torch.uint8)], L.Q4_0, i(2), i(1)))
    lg, qs = torch.zeros((5, 100)), i(3)
    raises(lambda: c.adjust_logits(lg, i(4), qs))
    raises(lambda: c.adjust_logits(lg.double(), i(5), qs))
    raises(lambda: c.adjust_logits(lg, i(5), qs, history=i(2, 7).long(), n_history=i(2)))
    raises(lambda: c.adjust_logits(lg, i(5), qs, repeat=torch.zeros(1)))
    raises(lambda: c.adjust_logits(lg, i(5), qs, bias=(i(3), i(4), torch.zeros(3))))
    raises(lambda: c.adjust_logits(lg, i(5), qs, mask_row=i(5)))
    raises(lambda: c.adjust_logits(lg, i(5), qs, out=torch.zeros((5, 200))[:, ::2]))
    with pytest.raises(ValueError):
        c._index = 0
        c.page_fork(i(3), i(3), i(3), i(4, 5), i(9), i(9), 16)


def test_the_plain_forms_agree_on_a_rounding():
    """Blocks with a tie for the largest size, zeros, and values at the borders of two numbers."""
    x = np.zeros((4, 32), np.float32)
    x[0, :3] = [-4, 4, 2]
    x[1, :4] = [3, -8, 0.5, -0.5]
    x[3] = np.linspace(-1, 1, 32)
    v = R.q4_values(R.q4_pack(x)).astype(np.float64)
    assert v[0, :3].tolist() == [-4, 3.5, 2] and not v[2].any()
    assert v[1, :4].tolist() == [3, -8, 1, 0]  # 8.5 steps up from -8 count as 9, 8 steps as 8
    assert np.abs(v[3] - x[3]).max() <= 0.125 + 1e-3
