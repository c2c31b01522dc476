"""Plain forms, on the CPU (numpy), of q4_0 rows, of pages that change hands between steps, and of the rules on logits,
written from their definitions."""
import math

import numpy as np


def q4_pack(x):
    """q4_0 blocks (uint8 [..., D / 32 * 18]) of f32 rows, block by block as ggml's reference rounds them."""
    b = np.ascontiguousarray(x, np.float32).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    at = np.abs(b).argmax(-1)[..., None]
    d = np.take_along_axis(b, at, -1) * np.float32(-0.125)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    q = np.clip(np.trunc((b * inv).astype(np.float32) + np.float32(8.5)), 0, 15).astype(np.uint8)
    out = np.empty(b.shape[:-1] + (18,), np.uint8)
    out[..., :2] = np.ascontiguousarray(d.astype(np.float16)).view(np.uint8)
    out[..., 2:] = q[..., :16] | q[..., 16:] << 4
    return out.reshape(x.shape[:-1] + (x.shape[-1] // 32 * 18,))


def q4_parts(rows):
    """(d [..., D / 32] f16, numbers [..., D / 32, 32]) of q4_0 rows."""
    b = rows.reshape(rows.shape[:-1] + (rows.shape[-1] // 18, 18))
    d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0]
    return d, np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1)


def q4_values(rows):
    """The f16 values of q4_0 rows uint8 [..., D / 32 * 18]."""
    d, q = q4_parts(rows)
    with np.errstate(invalid="ignore"):
        v = (d.astype(np.float64)[..., None] * (q.astype(np.float64) - 8.0)).astype(np.float16)
    return v.reshape(rows.shape[:-1] + (rows.shape[-1] // 18 * 32,))


def fork(parent, child, keep, table, refs, free, P, head=0):
    """(table, refs, src, dst, status, taken), fork by fork."""
    table, refs = table.copy(), refs.copy()
    old = table.copy()
    src, dst, status, at, taken = [], [], [], head, 0
    for p, c, k in zip(parent, child, keep):
        p, c, k = int(p), int(c), int(k)
        s = d = -1
        if k < 0 or not (0 <= p < len(table) and 0 <= c < len(table)) or p == c:
            st = 3
        elif k > table.shape[1] * P:
            st = 1
        else:
            st = 0
            if k % P:
                at += 1
                if head < 0 or at > len(free):
                    st = 2
        if st == 0:
            full = k // P
            for j in range(full):
                table[c, j] = old[p, j]
                if 0 <= old[p, j] < len(refs):
                    refs[old[p, j]] += 1
            if k % P:
                s, d = int(old[p, full]), int(free[at - 1])
                table[c, full] = d
                taken = at - head
                if not 0 <= s < len(refs):
                    s = d = -1
        src.append(s)
        dst.append(d)
        status.append(st)
    return table, refs, np.array(src), np.array(dst), np.array(status), taken


def free(rows, begin, end, table, refs, lst, head):
    """(table, refs, list, freed), entry by entry."""
    table, refs, lst = table.copy(), refs.copy(), lst.copy()
    gone = []
    for r, b, e in zip(rows, begin, end):
        if not 0 <= r < len(table):
            continue
        for j in range(max(int(b), 0), min(int(e), table.shape[1])):
            p = int(table[r, j])
            table[r, j] = -1
            if 0 <= p < len(refs):
                refs[p] -= 1
                if refs[p] < 0:
                    gone.append(p)
    gone = sorted(set(gone))
    refs[gone] = 0
    lst[head - len(gone):head] = gone
    return table, refs, lst, len(gone)


def compact(table, held, refs, lst):
    """(table, refs, list, src, dst, used)."""
    table, refs, lst = table.copy(), refs.copy(), lst.copy()
    n = len(refs)
    used = sorted({int(p) for r, h in zip(table, held) for p in r[:max(int(h), 0)] if 0 <= p < n})
    u = len(used)
    src = [p for p in used if p >= u]
    dst = [p for p in range(u) if p not in set(used)]
    to = dict(zip(src, dst))
    for r, h in zip(table, held):
        for j in range(min(max(int(h), 0), table.shape[1])):
            r[j] = to.get(int(r[j]), r[j])
    for s, d in to.items():
        refs[d], refs[s] = refs[s], 0
    lst[u:] = np.arange(u, n)
    return table, refs, lst, src, dst, u


def logits(lg, ids, q_start, history=None, n_history=None, last_n=None, repeat=None, frequency=None, presence=None, bias=None,
           mask=None, mask_row=None):
    """The adjusted rows in 64 bits; rows behind the last sequence are left out."""
    V, out = lg.shape[1], []
    for s in range(len(q_start) - 1):
        for r in range(q_start[s], q_start[s + 1]):
            l = lg[r].astype(np.float64)
            if bias is not None:
                start, tok, val = bias
                for x, b in dict(zip(tok[start[s]:start[s + 1]].tolist(), val[start[s]:start[s + 1]].tolist())).items():
                    if 0 <= x < V:
                        l[x] += b
            said = [] if history is None else history[s, :n_history[s]].tolist()
            said += ids[q_start[s]:r + 1].tolist()
            if last_n is not None and last_n[s] >= 0:
                said = said[len(said) - min(int(last_n[s]), len(said)):]
            if repeat is not None or frequency is not None or presence is not None:
                rep, fr, pr = (float(v[s]) if v is not None else d for v, d in ((repeat, 1.0), (frequency, 0.0), (presence, 0.0)))
                toks, count = np.unique(np.array([x for x in said if 0 <= x < V], np.int64), return_counts=True)
                for x, c in zip(toks, count):
                    l[x] = (l[x] / rep if l[x] > 0 else l[x] * rep) - c * fr - pr
            if mask is not None:
                m = r if mask_row is None else int(mask_row[r])
                if 0 <= m < len(mask):
                    words = mask[m].astype(np.int64) & 0xffffffff
                    x = np.arange(V)
                    l[(words[x // 32] >> (x % 32)) & 1 == 0] = -math.inf
            out.append(l)
    return np.array(out).reshape(-1, V)
