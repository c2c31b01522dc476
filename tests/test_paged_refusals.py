"""What the paged-cache operators refuse, through the C ABI and through ops.Context, without a device: every check comes
before anything touches the context or the GPU, so a block of zeros stands in for a context."""
import ctypes

import pytest
import torch

from srhpm_b200 import _lib as L
from srhpm_b200.ops import _head_rows, _ints, _paged

lib = L.load()
_ctx = ctypes.create_string_buffer(4096)
CTX = ctypes.cast(_ctx, ctypes.c_void_p)
A = 1 << 20  # an aligned address that nothing reads


def view(type_, ne, nb, data=A):
    ne, nb = list(ne) + [1] * (4 - len(ne)), list(nb) + [nb[-1]] * (4 - len(nb))
    return L.SrhpmTensor(type_, (ctypes.c_int64 * 4)(*ne), (ctypes.c_size_t * 4)(*nb), data)


def cache(D=256, P=64, Hkv=4, n=10, type_=L.F16, data=A, **over):
    row = D * 2 if type_ == L.F16 else D // 32 * 34
    nb = [2 if type_ == L.F16 else 34, Hkv * row, row, P * Hkv * row]
    for k, v in over.items():
        nb[int(k[2])] = v
    return view(type_, [D, P, Hkv, n], nb, data)


def rows(D=256, T=9, H=24, type_=L.F16, data=A, head_first=False, **over):
    e = 2 if type_ == L.F16 else 4
    ne = [D, H, T] if head_first else [D, T, H]
    nb = [e, D * e, H * D * e, T * H * D * e] if head_first else [e, H * D * e, D * e, T * H * D * e]
    for k, v in over.items():
        nb[int(k[2])] = v
    return view(type_, ne + [1], nb, data)


def table(cols=8, S=2, type_=L.I32, data=A, nb1=None):
    return view(type_, [cols, S], [4, nb1 if nb1 is not None else cols * 4], data)


def plan(**o):
    a = dict(past=A, new=A, S=2, P=16, table=table(), free=A, n_free=5, n_rows=7, q=A, kv=A, pos=A, slots=A, st=A, nt=A)
    a.update(o)
    return lib.srhpm_page_plan(CTX, a["past"], a["new"], None, a["S"], a["P"], ctypes.byref(a["table"]), a["free"], a["n_free"],
                               None, a["n_rows"], a["q"], a["kv"], a["pos"], a["slots"], a["st"], a["nt"], None)


@pytest.mark.parametrize("o,st", [
    (dict(past=None), L.ERR_INVALID), (dict(nt=None), L.ERR_INVALID), (dict(S=0), L.ERR_INVALID),
    (dict(P=0), L.ERR_INVALID), (dict(n_free=-1), L.ERR_INVALID), (dict(free=None), L.ERR_INVALID),
    (dict(slots=None), L.ERR_INVALID), (dict(slots=A + 4), L.ERR_ALIGN), (dict(S=3), L.ERR_INVALID),
    (dict(table=table(type_=L.F32)), L.ERR_INVALID), (dict(table=table(nb1=30)), L.ERR_ALIGN),
    (dict(table=table(nb1=16)), L.ERR_INVALID), (dict(table=table(data=0)), L.ERR_INVALID),
    (dict(S=8193, table=table(S=8193)), L.UNSUPPORTED)])
def test_page_plan(o, st):
    assert plan(**o) == st


def store(qkv=None, H=24, Hkv=4, pos=A, slots=A, base=1e6, q=None, k=None, v=None):
    qkv = qkv or view(L.F32, [32 * 256, 9], [4, 32 * 256 * 4])
    q, k, v = q or rows(), k or cache(), v or cache()
    return lib.srhpm_rope_kv_paged(CTX, ctypes.byref(qkv), H, Hkv, pos, slots, base, ctypes.byref(q), ctypes.byref(k),
                                   ctypes.byref(v), None)


W = 32 * 256


@pytest.mark.parametrize("o,st", [
    (dict(pos=None), L.ERR_INVALID), (dict(base=0.0), L.ERR_INVALID), (dict(H=23), L.ERR_INVALID),
    (dict(Hkv=2), L.ERR_INVALID), (dict(slots=A + 4), L.ERR_ALIGN),
    (dict(qkv=view(L.F16, [W, 9], [2, W * 2])), L.UNSUPPORTED), (dict(qkv=view(L.F32, [W, 9], [4, W * 4 - 16])), L.ERR_INVALID),
    (dict(qkv=view(L.F32, [W, 9], [4, W * 4 + 4])), L.ERR_ALIGN), (dict(qkv=view(L.F32, [W, 9], [4, W * 4], A + 4)), L.ERR_ALIGN),
    (dict(q=rows(T=8)), L.ERR_INVALID), (dict(q=rows(data=A + 8)), L.ERR_ALIGN), (dict(q=rows(type_=L.I32)), L.UNSUPPORTED),
    (dict(k=cache(type_=L.Q8_0)), L.UNSUPPORTED), (dict(k=cache(D=96), v=cache(D=96)), L.UNSUPPORTED),
    (dict(k=cache(n=11)), L.ERR_INVALID), (dict(k=cache(nb1=W + 8)), L.ERR_ALIGN), (dict(v=cache(nb2=256)), L.ERR_INVALID),
    (dict(v=cache(data=A + 2)), L.ERR_ALIGN)])
def test_rope_kv_paged(o, st):
    assert store(**o) == st


def attn(q=None, k=None, v=None, tb=None, qs=A, kl=A, sinks=None, scale=0.1, cap=0.0, window=0, dst=None, w=A, ws=0):
    q, k, v, tb = q or rows(), k or cache(), v or cache(), tb or table()
    dst = dst or rows(head_first=True)
    return lib.srhpm_flash_attn_paged(CTX, ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), ctypes.byref(tb), qs, kl,
                                      ctypes.byref(sinks) if sinks else None, scale, cap, window, ctypes.byref(dst), w,
                                      ws, None)


@pytest.mark.parametrize("o,st", [
    (dict(qs=None), L.ERR_INVALID), (dict(window=-1), L.ERR_INVALID), (dict(scale=0.0), L.ERR_INVALID),
    (dict(scale=float("nan")), L.ERR_INVALID), (dict(cap=-1.0), L.ERR_INVALID), (dict(q=rows(H=22)), L.ERR_INVALID),
    (dict(q=rows(type_=L.F32)), L.ERR_INVALID), (dict(q=rows(nb1=24)), L.ERR_ALIGN), (dict(q=rows(D=128)), L.ERR_INVALID),
    (dict(k=cache(P=24), v=cache(P=24)), L.UNSUPPORTED), (dict(k=cache(P=8), v=cache(P=8)), L.UNSUPPORTED),
    (dict(k=cache(D=128, type_=L.Q8_0, nb1=1024, nb2=256, nb3=1 << 16),
          v=cache(D=128, type_=L.Q8_0, nb1=1024, nb2=256, nb3=1 << 16), q=rows(D=128)), L.UNSUPPORTED),
    (dict(v=cache(type_=L.Q8_0)), L.UNSUPPORTED), (dict(k=cache(data=A + 8)), L.ERR_ALIGN),
    (dict(tb=table(type_=L.F32)), L.ERR_INVALID), (dict(dst=rows(head_first=True, T=8)), L.ERR_INVALID),
    (dict(dst=rows(head_first=True, nb2=24)), L.ERR_ALIGN), (dict(sinks=view(L.F32, [23], [4])), L.ERR_INVALID),
    (dict(sinks=view(L.F16, [24], [2])), L.ERR_INVALID)])
def test_flash_attn_paged(o, st):
    assert attn(**o) == st


@pytest.mark.parametrize("o", [
    dict(tb=table(S=8193)),  # sequences
    dict(q=rows(T=1 << 24, H=512, nb1=256 * 1024), dst=rows(T=1 << 24, H=512, head_first=True)),  # rows of a KV head
    dict(q=rows(T=1 << 24), dst=rows(T=1 << 24, head_first=True), tb=table(cols=1200)),  # tiles: 1797560 x 1201
    dict(q=rows(T=1 << 16), dst=rows(T=1 << 16, head_first=True), tb=table(cols=1 << 30))])  # 7022 x 2^25 (2^31 tokens)
def test_flash_attn_paged_too_large(o):
    assert attn(**o) == L.UNSUPPORTED


def sample(lg=None, ids=A, qs=A, S=2, dp=None, u=A, us=A, oi=A, on=A, w=A, ws=1 << 30):
    lg = lg or view(L.F32, [1000, 5], [4, 4000])
    return lib.srhpm_verify_sample(CTX, ctypes.byref(lg), ids, qs, S, ctypes.byref(dp) if dp else None, None, u, us, oi,
                                   on, None, w, ws, None)


@pytest.mark.parametrize("o,st", [
    (dict(ids=None), L.ERR_INVALID), (dict(us=None), L.ERR_INVALID), (dict(on=None), L.ERR_INVALID),
    (dict(S=0), L.ERR_INVALID), (dict(lg=view(L.F16, [1000, 5], [2, 2000])), L.ERR_INVALID),
    (dict(lg=view(L.F32, [1000, 5], [4, 3996])), L.ERR_INVALID), (dict(lg=view(L.F32, [0, 5], [4, 4000])), L.ERR_INVALID),
    (dict(dp=view(L.F32, [1000, 4], [4, 4000])), L.ERR_INVALID), (dict(dp=view(L.F32, [999, 5], [4, 4000])), L.ERR_INVALID)])
def test_verify_sample(o, st):
    assert sample(**o) == st


def test_verify_sample_too_many_sequences():
    assert sample(S=(1 << 24) + 1) == L.ERR_INVALID
    size = ctypes.c_size_t()
    lg = view(L.F32, [1000, 5], [4, 4000])
    assert lib.srhpm_verify_sample_work_size(CTX, ctypes.byref(lg), (1 << 24) + 1, ctypes.byref(size)) == L.ERR_INVALID


def test_python_layer():
    with pytest.raises(ValueError):
        _head_rows(torch.zeros(3, 4, 64, dtype=torch.bfloat16), False)
    with pytest.raises(ValueError):
        _head_rows(torch.zeros(3, 64, 4).transpose(1, 2), False)
    with pytest.raises(ValueError):
        _paged(torch.zeros((2, 16, 4, 271), dtype=torch.uint8), L.Q8_0)
    with pytest.raises(ValueError):
        _paged(torch.zeros((2, 16, 4), dtype=torch.uint8), L.F16)
    with pytest.raises(ValueError):
        _ints(torch.zeros(4, dtype=torch.int64), torch.int32, 4, "ids")
    with pytest.raises(ValueError):
        _ints(torch.zeros(3, dtype=torch.int32), torch.int32, 4, "ids")
    with pytest.raises(ValueError):
        _ints(torch.zeros(8, dtype=torch.int32)[::2], torch.int32, 4, "ids")


# vectors a page apart; n_seqs 2, n_rows 7, n_free 5
PLAN_IN = {"n_past": 8, "n_new": 8, "n_held": 8, "free": 20, "free_head": 4}
PLAN_OUT = {"q_start": 12, "kv_len": 8, "pos": 28, "slots": 56, "status": 8, "n_taken": 4}


@pytest.mark.parametrize("i", PLAN_IN)
@pytest.mark.parametrize("o", PLAN_OUT)
@pytest.mark.parametrize("where", ["same", "first byte", "last byte"])
def test_page_plan_outputs_that_share_memory_with_inputs(i, o, where):
    """kv_len as the next step's n_past, above all: other CTAs read lengths that this one has written over."""
    at = {n: A + 4096 * k for k, n in enumerate([*PLAN_IN, *PLAN_OUT])}
    if o == "slots":  # stays aligned: the input moves instead
        at[i] = at[o] + {"same": 0, "first byte": 4 - PLAN_IN[i], "last byte": PLAN_OUT[o] - 4}[where]
    else:
        at[o] = at[i] + {"same": 0, "first byte": 4 - PLAN_OUT[o], "last byte": PLAN_IN[i] - 4}[where]
    st = lib.srhpm_page_plan(CTX, at["n_past"], at["n_new"], at["n_held"], 2, 16, ctypes.byref(table(data=A + (1 << 18))), at["free"], 5,
                             at["free_head"], 7, at["q_start"], at["kv_len"], at["pos"], at["slots"], at["status"],
                             at["n_taken"], None)
    assert st == L.ERR_INVALID


SAMPLE_IN = {"ids": 20, "q_start": 12, "temperature": 8, "u": 20, "us": 8}
SAMPLE_OUT = {"out_ids": 20, "out_n": 8, "p_draft": 20}


@pytest.mark.parametrize("i", SAMPLE_IN)
@pytest.mark.parametrize("o", SAMPLE_OUT)
@pytest.mark.parametrize("where", ["same", "first byte", "last byte"])
def test_verify_sample_outputs_that_share_memory_with_inputs(i, o, where):
    at = {n: A + 4096 * k for k, n in enumerate([*SAMPLE_IN, *SAMPLE_OUT])}
    at[o] = at[i] + {"same": 0, "first byte": 4 - SAMPLE_OUT[o], "last byte": SAMPLE_IN[i] - 4}[where]
    st = lib.srhpm_verify_sample(CTX, ctypes.byref(view(L.F32, [1000, 5], [4, 4000])), at["ids"], at["q_start"], 2, None,
                                 at["temperature"], at["u"], at["us"], at["out_ids"], at["out_n"], at["p_draft"], A,
                                 1 << 30, None)
    assert st == L.ERR_INVALID
