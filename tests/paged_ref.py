"""Plain 64-bit forms of the paged-cache operators, on the CPU (numpy), written from their definitions."""
import math

import numpy as np


def plan(past, new, table, free, P, n_rows, head=0, held=None):
    """(table, q_start, kv_len, pos, slots, status, n_taken) of srhpm_page_plan, sequence by sequence."""
    table = table.copy()
    S, cols = table.shape
    q_start, kv_len, status = [0], [], []
    pos, slots = np.zeros(n_rows, np.int64), np.full(n_rows, -1, np.int64)
    at, taken = head, 0
    for s in range(S):
        a, n = int(past[s]), int(new[s])
        q_start.append(q_start[-1] + max(n, 0))
        have, want = max(-(-a // P), int(held[s]) if held is not None else 0), -(-(a + n) // P)
        if a < 0 or n < 0:
            st = 3
        elif q_start[-1] > n_rows:
            st = 4
        elif want > cols or a + n > 2 ** 31 - 1:
            st = 1
        else:
            st = 0
            need = max(want - have, 0)
            at += need
            if need and (head < 0 or at > len(free)):
                st = 2
            elif need:
                table[s, have:want] = free[at - need:at]
                taken = at - head
        status.append(st)
        kv_len.append(a + n if st == 0 else 0)
        if st == 0:
            p = np.arange(a, a + n)
            pos[q_start[s]:q_start[s] + n] = p
            page = table[s, p // P].astype(np.int64)
            slots[q_start[s]:q_start[s] + n] = np.where(page < 0, -1, page * P + p % P)
    return table, np.array(q_start), np.array(kv_len), pos, slots, np.array(status), taken


def turn(x, pos, base):
    """NeoX rotation of x [n, heads, D] in 64 bits."""
    D = x.shape[-1]
    ang = np.asarray(pos, np.float64)[:, None] * base ** (-2.0 * np.arange(D // 2) / D)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def q8_values(rows):
    """The f16 values of q8_0 cache rows uint8 [..., D / 32 * 34]."""
    b = rows.reshape(rows.shape[:-1] + (-1, 34))
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    v = (d * np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)).astype(np.float16)
    return v.reshape(rows.shape[:-1] + (-1,))


def attention(q, kc, vc, table, q_start, kv_len, scale, softcap=0.0, window=0, sinks=None):
    """q [T, H, D]; kc, vc [pages, P, Hkv, D] values. Returns (out, |v| average, largest sum |q k| scale) per row: the
    last two size the rounding bounds."""
    T, H, D = q.shape
    P, Hkv = kc.shape[1], kc.shape[2]
    G = H // Hkv
    out, mag, big = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H, 1))
    for s in range(len(kv_len)):
        n = q_start[s + 1] - q_start[s]
        for i in range(n):
            t, p = q_start[s] + i, kv_len[s] - n + i
            lo = max(0, p - window + 1) if window > 0 else 0
            j = np.arange(lo, max(p + 1, lo))
            page = np.asarray(table)[s, j // P]
            ok = (page >= 0) & (page < kc.shape[0])
            pg = np.where(ok, page, 0)
            for g in range(Hkv):
                k = kc[pg, j % P, g].astype(np.float64) * ok[:, None]
                v = np.where(ok[:, None], vc[pg, j % P, g].astype(np.float64), 0.0)
                for h in range(g * G, (g + 1) * G):
                    qq = q[t, h].astype(np.float64)
                    sc = k @ qq * scale
                    if len(j):
                        big[t, h] = (np.abs(k) @ np.abs(qq)).max() * scale
                    if softcap:
                        sc = softcap * np.tanh(sc / softcap)
                    sk = -math.inf if sinks is None else float(sinks[h])
                    m = max([sk] + ([sc.max()] if len(j) else []))
                    if m == -math.inf:
                        continue
                    w = np.exp(sc - m)
                    z = w.sum() + math.exp(sk - m)
                    out[t, h], mag[t, h] = w @ v / z, w @ np.abs(v) / z
    return out, mag, big


def attention_dense(q, k, v, q_start, kv_len, scale, window=0):
    """The same for long inputs, on the inputs' device (torch): k, v [S][L, Hkv, D] values of each sequence. Returns
    (out, |v| average, largest sum |q k| scale) in 64 bits."""
    import torch
    T, H, D = q.shape
    out, mag = (torch.zeros((T, H, D), dtype=torch.float64, device=q.device) for _ in range(2))
    big = torch.zeros((T, H, 1), dtype=torch.float64, device=q.device)
    for s in range(len(kv_len)):
        r0, r1 = int(q_start[s]), int(q_start[s + 1])
        L, G = int(kv_len[s]), H // k[s].shape[1]
        p = torch.arange(L - (r1 - r0), L, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)
        hide = (j > p) | ((j <= p - window) if window > 0 else (j < 0))
        for h in range(H):
            kk, vv = k[s][:, h // G].double(), v[s][:, h // G].double()
            qq = q[r0:r1, h].double()
            sc = (qq @ kk.T * scale).masked_fill(hide, -math.inf)
            w = torch.softmax(sc, 1)
            out[r0:r1, h], mag[r0:r1, h] = w @ vv, w @ vv.abs()
            big[r0:r1, h] = (qq.abs() @ kk.abs().T).masked_fill(hide, 0).amax(1, keepdim=True) * scale
    return out.cpu().numpy(), mag.cpu().numpy(), big.cpu().numpy()


def sample(logits, ids, q_start, u, us, dp=None, temp=None):
    """(out_ids with -1 for what is not emitted and None behind the last sequence, out_n, p_draft)."""
    T, V = logits.shape
    out, cnt, pd = [None] * T, [], [None] * T
    for s in range(len(q_start) - 1):
        r0, r1 = q_start[s], q_start[s + 1]
        t = 1.0 if temp is None else float(temp[s])
        open_, n = True, 0
        for r in range(r0, r1):
            l = logits[r].astype(np.float64)
            l = np.where(np.isnan(l), -math.inf, l)
            m = l.max()
            top = int(l.argmax()) if m > -math.inf else 0
            if m == -math.inf:
                e = np.zeros(V)
            elif t <= 0:
                e = np.zeros(V)
                e[top] = 1.0
            else:
                with np.errstate(invalid="ignore"):
                    e = np.where(l == m, 1.0, np.exp((l - m) / t))
            z = e.sum()
            last = r == r1 - 1
            x = -1 if last else int(ids[r + 1])
            inside = 0 <= x < V
            p = e[x] / z if inside and z > 0 else 0.0
            b = (float(dp[r, x]) if dp is not None else 1.0) if inside else 0.0
            pd[r] = p
            out[r] = -1
            if not open_:
                continue
            n += 1
            if not last and float(u[r]) * b < p:
                out[r] = x
                continue
            open_ = False
            if last:
                w = e
            elif dp is not None:
                w = np.maximum((e / z if z > 0 else e) - dp[r].astype(np.float64), 0.0)
            else:
                w = e.copy()
                if inside:
                    w[x] = 0.0
            c = w.cumsum()
            if not c[-1] > 0:
                out[r] = top
            else:
                over = np.nonzero(c > float(us[s]) * c[-1])[0]
                out[r] = int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
        cnt.append(n)
    return out, cnt, pd


def turned_items(q_start, kv_len, n_head, n_head_kv, head_dim, q8, f32, window, n_cta):
    """(items, turned, inside): work items of srhpm_flash_attn_paged, those that one CTA takes whole but not from their first
    tile on, and those among them with a tile that holds slots no row sees (behind the cache or before the window) and
    does not come last. Units of all items in one line, cut into n_cta equal parts (every item here has a unit or more)."""
    S, G, T = len(kv_len), n_head // n_head_kv, int(q_start[-1])
    few = (q8 and f32) or T * G <= S * 56
    rows = 56 if few else 256 if head_dim <= 128 else 128
    bn = 64 if q8 and f32 else 128
    items = []
    for s in range(S):
        n, kv = int(q_start[s + 1] - q_start[s]), int(kv_len[s])
        for _ in range(n_head_kv):
            for r in range(0, n * G, rows):
                hi = kv - n + (min(n * G, r + rows) - 1) // G + 1
                lo = max(0, kv - n + r // G - window + 1) if window > 0 else 0
                items.append((lo // bn, -(-hi // bn), bool(lo % bn), bool(hi % bn)))
    W = sum(b - a for a, b, _, _ in items)
    parts, at = min(n_cta, W), 0
    turned = inside = 0
    for a, b, first, last in items:
        n = b - a
        c = ((at + 1) * parts - 1) // W  # the part that holds unit `at`
        while W * (c + 1) // parts <= at:
            c += 1
        start = W * c // parts
        if n >= 64 and at + n <= W * (c + 1) // parts:
            turn = (at - start) % n
            if turn:
                turned += 1
                # the order: turn .. n - 1, 0 .. turn - 1
                inside += last or (first and turn != 1)
        at += n
    return len(items), turned, inside
