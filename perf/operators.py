"""Workloads of the batched paged-cache operators: page plans, RoPE with a paged store, attention of new tokens over
pages, and verification of drafted tokens by sampling. Each is given in plain torch (`own` false) and as the calls that
a serving loop makes of this package (`own` true)."""
import math
import os
import random
import sys

import torch

own = False  # True: the package's operators; False: their plain forms
DEV = "cuda"
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sr-hpm_b200")
_kept = {}


def _context():
    """The package and its context, made once as a program makes them at its start."""
    if "ctx" not in _kept:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        import srhpm_b200 as S
        _kept["S"], _kept["ctx"] = S, S.Context(torch.cuda.current_device())
    return _kept["S"], _kept["ctx"]


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one scheduling step of a small server: every sequence verifies 8 drafted tokens
        {"name": "plan_verify", "op": "plan", "seqs": 8, "new_lo": 9, "new_hi": 9, "past_hi": 4096, "page": 16,
         "lens": 1},
        # a step of a large one: prompts of any length come in beside sequences that decode
        {"name": "plan_prompts", "op": "plan", "seqs": 1024, "new_lo": 1, "new_hi": 1200, "past_hi": 8192, "page": 64,
         "lens": 2},
        # the 9 token rows of one verify step of the 27B-class decoder (24 query, 4 KV heads of 256)
        {"name": "store_verify", "op": "store", "rows": 9, "H": 24, "Hkv": 4, "D": 256, "kv": "f16", "q": "f32",
         "page": 64, "pos_hi": 131072},
        # a prompt chunk of a decoder with 32 query and 8 KV heads of 128
        {"name": "store_prompt", "op": "store", "rows": 8192, "H": 32, "Hkv": 8, "D": 128, "kv": "f16", "q": "f16",
         "page": 16, "pos_hi": 32768},
        # a prompt chunk into a q8_0 cache
        {"name": "store_q8", "op": "store", "rows": 4001, "H": 24, "Hkv": 4, "D": 256, "kv": "q8_0", "q": "f16",
         "page": 64, "pos_hi": 32768},
        # plain decoding of a batch: one token each over caches of unequal lengths
        {"name": "attn_decode", "op": "attn", "seqs": 32, "new_lo": 1, "new_hi": 1, "past_lo": 500, "past_hi": 8192,
         "H": 32, "Hkv": 8, "D": 128, "kv": "f16", "q": "f16", "page": 16, "window": 0, "lens": 3},
        # one verify step at the long-context length of the 27B-class decoder, full precision rows
        {"name": "attn_verify_long", "op": "attn", "seqs": 1, "new_lo": 9, "new_hi": 9, "past_lo": 131063,
         "past_hi": 131063, "H": 24, "Hkv": 4, "D": 256, "kv": "f16", "q": "f32", "page": 64, "window": 0, "lens": 4},
        # a batch of verify steps over q8_0 caches
        {"name": "attn_verify_q8", "op": "attn", "seqs": 4, "new_lo": 2, "new_hi": 9, "past_lo": 2048,
         "past_hi": 16384, "H": 24, "Hkv": 4, "D": 256, "kv": "q8_0", "q": "f16", "page": 32, "window": 0, "lens": 5},
        # a chunk of a long prompt: 2048 new tokens behind 30720 cached ones
        {"name": "attn_chunk", "op": "attn", "seqs": 1, "new_lo": 2048, "new_hi": 2048, "past_lo": 30720,
         "past_hi": 30720, "H": 24, "Hkv": 4, "D": 256, "kv": "f16", "q": "f16", "page": 64, "window": 0, "lens": 6},
        # prompts, verify steps and single tokens in one batch, sliding-window layer
        {"name": "attn_mixed", "op": "attn", "seqs": 7, "new_lo": 1, "new_hi": 1000, "past_lo": 0, "past_hi": 4000,
         "H": 32, "Hkv": 8, "D": 128, "kv": "f16", "q": "f16", "page": 48, "window": 1024, "lens": 7},
        # one sequence, 8 drafted tokens of a greedy drafter, the 27B-class vocabulary
        {"name": "sample_one", "op": "sample", "seqs": 1, "k_lo": 8, "k_hi": 8, "V": 151936, "draft": False, "lens": 8},
        # a batch whose drafter sampled: its distributions take part
        {"name": "sample_batch", "op": "sample", "seqs": 64, "k_lo": 2, "k_hi": 8, "V": 151936, "draft": True,
         "lens": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "attn", "attn", "sample"])
    page = rng.choice([16, 32, 48, 64, 80, 128, 256])
    lens = rng.randrange(1 << 30)
    H, Hkv, D = rng.choice([(24, 4, 256), (16, 16, 64), (32, 8, 128), (6, 2, 256), (28, 4, 128), (8, 1, 64)])
    if op == "plan":
        return {"op": op, "seqs": _log(rng, 1, 1024), "new_lo": 0, "new_hi": _log(rng, 1, 1200),
                "past_hi": _log(rng, 16, 8192), "page": page, "lens": lens}
    if op == "store":
        kv = rng.choice(["f16", "f16", "q8_0"])
        return {"op": op, "rows": _log(rng, 1, 4000), "H": H, "Hkv": Hkv, "D": D, "kv": kv,
                "q": rng.choice(["f16", "f32"]), "page": page, "pos_hi": _log(rng, 8192, 131072)}
    if op == "attn":
        kv = rng.choice(["f16", "q8_0"]) if D == 256 else "f16"
        seqs = _log(rng, 1, 32)
        past_hi = _log(rng, 1, 65536 // seqs)
        return {"op": op, "seqs": seqs, "new_lo": 1, "new_hi": _log(rng, 1, min(2000, 8192 // seqs)), "past_lo": 0,
                "past_hi": past_hi, "H": H, "Hkv": Hkv, "D": D, "kv": kv, "q": rng.choice(["f16", "f16", "f32"]),
                "page": page, "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "lens": lens}
    V = _log(rng, 500, 151936)
    return {"op": op, "seqs": _log(rng, 1, 60), "k_lo": 0, "k_hi": rng.randrange(1, 9), "V": V,
            "draft": rng.random() < 0.6, "lens": lens}


def _lengths(case):
    """(past, new) of each sequence: part of the case, not of its inputs."""
    rng = random.Random(case["lens"])
    past, new = [], []
    for _ in range(case["seqs"]):
        past.append(rng.randint(case.get("past_lo", 0), case["past_hi"]))
        hi, lo = case["new_hi"], case["new_lo"]
        # most sequences of a batch decode or verify, some bring a prompt
        new.append(rng.randint(lo, hi if hi <= 16 or rng.random() < 0.4 else max(lo, 16)))
    return past, new


def _drafts(case):
    rng = random.Random(case["lens"])
    return [rng.randint(case["k_lo"], case["k_hi"]) for _ in range(case["seqs"])]


# ---- inputs --------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _q_start(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return _i32(at)


ROW = {"f16": lambda D: 2 * D, "q8_0": lambda D: D // 32 * 34}


def _cache(kv, pages, page, Hkv, D, g):
    """A pool of pages uint8 [pages, page, Hkv, row bytes] holding values of unit size."""
    if kv == "f16":
        return torch.randn((pages, page, Hkv, D), device=DEV, generator=g, dtype=torch.float16).view(torch.uint8)
    b = torch.randint(-127, 128, (pages, page, Hkv, D // 32, 34), device=DEV, generator=g, dtype=torch.int8)
    b = b.view(torch.uint8)
    d = (torch.rand((pages, page, Hkv, D // 32, 1), device=DEV, generator=g) * 0.01 + 0.01).half()
    b[..., :2] = d.view(torch.uint8)
    return b.view(pages, page, Hkv, -1)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    if case["op"] == "plan":
        past, new = _lengths(case)
        P = case["page"]
        cols = max(-(-(a + b) // P) for a, b in zip(past, new)) + 1
        have = [-(-a // P) for a in past]
        need = sum(-(-(a + b) // P) for a, b in zip(past, new)) - sum(have)
        pool = torch.randperm(sum(have) + need + 7, device=DEV, generator=g).int()
        table = torch.full((case["seqs"], cols), -1, dtype=torch.int32, device=DEV)
        held = torch.arange(cols, device=DEV)[None, :] < _i32(have)[:, None]
        table[held] = pool[:sum(have)]
        T = sum(new) + 5  # a few padded rows, as a captured step has them
        st |= {"past": _i32(past), "new": _i32(new), "table": table, "free": pool[sum(have):].contiguous(), "T": T,
               "head": _i32([int(seed) % 7])}
    elif case["op"] == "store":
        n, H, Hkv, D, P = (case[k] for k in ("rows", "H", "Hkv", "D", "page"))
        pages = -(-n // P) + 3
        st |= {"qkv": torch.randn((n, (H + 2 * Hkv) * D), device=DEV, generator=g),
               "pos": torch.randint(0, case["pos_hi"], (n,), device=DEV, generator=g).int(),
               "slots": torch.randperm(pages * P, device=DEV, generator=g)[:n].contiguous(),
               "k": _cache(case["kv"], pages, P, Hkv, D, g), "v": _cache(case["kv"], pages, P, Hkv, D, g),
               "q_out": torch.empty((n, H, D), device=DEV, dtype=torch.float16 if case["q"] == "f16" else torch.float32)}
    elif case["op"] == "attn":
        past, new = _lengths(case)
        H, Hkv, D, P = (case[k] for k in ("H", "Hkv", "D", "page"))
        nb = [-(-(a + b) // P) for a, b in zip(past, new)]
        pages = sum(nb) + 3
        table = torch.full((case["seqs"], max(nb)), -1, dtype=torch.int32, device=DEV)
        held = torch.arange(max(nb), device=DEV)[None, :] < _i32(nb)[:, None]
        table[held] = torch.randperm(pages, device=DEV, generator=g)[:sum(nb)].int()
        t = torch.float16 if case["q"] == "f16" else torch.float32
        T = sum(new)
        st |= {"table": table, "q_start": _q_start(new), "kv_len": _i32([a + b for a, b in zip(past, new)]),
               "Lmax": max(a + b for a, b in zip(past, new)), "Nmax": max(new), "T": T,
               "q": torch.randn((T, H, D), device=DEV, generator=g).to(t),
               "k": _cache(case["kv"], pages, P, Hkv, D, g), "v": _cache(case["kv"], pages, P, Hkv, D, g),
               "out": torch.empty((T, H, D), device=DEV, dtype=t)}
    else:
        ks = _drafts(case)
        T, V = sum(ks) + len(ks), case["V"]
        # logits of a confident model: a wide body and a few high tokens; the drafter sees them through noise
        lg = torch.randn((T, V), device=DEV, generator=g) * 2.0
        top = torch.randint(0, V, (T, 8), device=DEV, generator=g)
        lg.scatter_add_(1, top, 6.0 + 8.0 * torch.rand((T, 8), device=DEV, generator=g))
        near = lg + 0.5 * torch.randn((T, V), device=DEV, generator=g)
        dp = torch.softmax(near, 1) if case["draft"] else None
        if case["draft"]:  # tokens drawn from the drafter's distributions
            noise = torch.rand((T, V), device=DEV, generator=g).clamp_(1e-10, 1.0)
            pick = (near - (-noise.log()).log()).argmax(1)
            del noise
        else:
            pick = near.argmax(1)
        ids = torch.zeros(T, dtype=torch.int32, device=DEV)
        ids[1:] = pick[:-1].int()  # row r scores the token behind ids[r]; the drafted token is ids[r + 1]
        st |= {"logits": lg, "ids": ids, "q_start": _q_start([k + 1 for k in ks]), "dp": dp,
               "temp": 0.5 + torch.rand((len(ks),), device=DEV, generator=g),
               "u": torch.rand((T,), device=DEV, generator=g), "us": torch.rand((len(ks),), device=DEV, generator=g)}
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _plan(st):
    P, T, S = st["page"], st["T"], st["seqs"]
    past, new, table, free = st["past"].long(), st["new"].long(), st["table"], st["free"].long()
    dev = past.device
    q_start = torch.zeros(S + 1, dtype=torch.int64, device=dev)
    q_start[1:] = new.clamp(min=0).cumsum(0)
    have, want = (past + P - 1) // P, (past + new + P - 1) // P
    status = torch.where(want > table.shape[1], 1, 0)
    status = torch.where(q_start[1:] > T, 4, status)
    status = torch.where((past < 0) | (new < 0), 3, status)
    need = torch.where(status == 0, want - have, 0)
    end = need.cumsum(0)
    head = st["head"].long()
    status = torch.where((need > 0) & (head + end > free.numel()), 2, status)
    ok = status == 0
    taken = torch.where(ok & (need > 0), end, 0).amax()
    col = torch.arange(table.shape[1], device=dev)[None, :]
    src = (head + (end - need)[:, None] + col - have[:, None]).clamp(0, free.numel() - 1)
    fresh = ok[:, None] & (col >= have[:, None]) & (col < want[:, None])
    table.copy_(torch.where(fresh, free[src], table.long()))
    t = torch.arange(T, device=dev)
    s = (torch.searchsorted(q_start, t, right=True) - 1).clamp(max=S - 1)
    used = (t < q_start[-1]) & ok[s]
    pos = torch.where(used, past[s] + t - q_start[s], 0)
    page = table.long()[s, (pos // P).clamp(max=table.shape[1] - 1)]
    slots = torch.where(used, page * P + pos % P, -1)
    kv_len = torch.where(ok, past + new, 0)
    return table, q_start.int(), kv_len.int(), pos.int(), slots, status.int(), taken.int().view(1)


BASE = 1e6


def _turn(x, pos):
    """NeoX rotation of rows x [n, heads, D] at positions pos, angles in 64 bits."""
    half = x.shape[-1] // 2
    j = torch.arange(half, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None] * torch.exp(-math.log(BASE) * 2.0 * j / (2 * half))
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _pack_q8(x):
    """q8_0 blocks of rows x [..., D]: uint8 [..., D / 32 * 34]."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    q = torch.round(b * torch.where(amax > 0, 127.0 / amax, 0.0)).to(torch.int8)
    d = (amax / 127.0).half()
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], -1).flatten(-2)


def _values(c, kv):
    """The f16 values that cache rows [..., row bytes] stand for; a q8_0 value is d * q rounded to f16."""
    if kv == "f16":
        return c.view(torch.float16)
    b = c.unflatten(-1, (-1, 34))
    d = b[..., :2].contiguous().view(torch.float16)
    return (d.float() * b[..., 2:].view(torch.int8).float()).half().flatten(-2)


def _stored(st):
    """What the caches hold now: whole for f16, the written rows' values for q8_0."""
    if st["kv"] == "f16":
        return st["k"].view(torch.float16), st["v"].view(torch.float16)
    at = st["slots"]
    return tuple(_values(st[c].flatten(0, 1)[at], "q8_0") for c in ("k", "v"))


def _store(st):
    n, H, Hkv, D = (st[k] for k in ("rows", "H", "Hkv", "D"))
    x = st["qkv"].view(n, H + 2 * Hkv, D)
    turned = _turn(x[:, :H + Hkv], st["pos"])
    for c, rows in (("k", turned[:, H:]), ("v", x[:, H + Hkv:])):
        rows = rows.half().view(torch.uint8) if st["kv"] == "f16" else _pack_q8(rows)
        st[c].flatten(0, 1)[st["slots"]] = rows
    st["q_out"].copy_(turned[:, :H])
    return (st["q_out"],) + _stored(st)


def _attn(st):
    H, Hkv, D, P, S, L, N, T = (st[k] for k in ("H", "Hkv", "D", "page", "seqs", "Lmax", "Nmax", "T"))
    G = H // Hkv
    dev = st["q"].device
    qs, kl = st["q_start"].long(), st["kv_len"].long()
    n = qs[1:] - qs[:-1]
    i = torch.arange(N, device=dev)
    rows = (qs[:-1, None] + i).clamp(max=T - 1)
    q = st["q"][rows].float().view(S, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * N, D)
    j = torch.arange(L, device=dev)
    pages = st["table"].long().clamp(min=0)[:, j // P]
    k = _values(st["k"][pages, j % P], st["kv"]).float().permute(0, 2, 3, 1)
    s = torch.matmul(q, k).view(S, Hkv, G, N, L) * (1.0 / math.sqrt(D))
    del k
    p = (kl - n)[:, None] + i  # position of each row
    see = (j[None, None] <= p[..., None]) & (i[None, :, None] < n[:, None, None])
    if st["window"] > 0:
        see &= j[None, None] > p[..., None] - st["window"]
    s.masked_fill_(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m > -math.inf, m, 0.0)).exp_()
    z = s.sum(-1, keepdim=True)
    v = _values(st["v"][pages, j % P], st["kv"]).float().permute(0, 2, 1, 3)
    v = torch.where((j[None] < kl[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(s.view(S, Hkv, G * N, L), v).view(S, Hkv, G, N, D)
    o = (o / torch.where(z > 0, z, 1.0)).permute(0, 3, 1, 2, 4).reshape(S, N, H, D)
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(qs, t, right=True) - 1
    st["out"].copy_(o[seq, t - qs[seq]])
    return st["out"]


def _sample(st):
    S, V, lg, dp = st["seqs"], st["V"], st["logits"], st["dp"]
    T = lg.shape[0]
    dev = lg.device
    qs = st["q_start"].long()
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(qs, t, right=True) - 1
    e = lg.double()
    e = torch.exp((e - e.amax(1, keepdim=True)) / st["temp"].double()[seq][:, None])
    z = e.sum(1)
    last = t == qs[1:][seq] - 1
    x = torch.cat([st["ids"][1:], st["ids"][:1]]).long()
    x = torch.where(last, 0, x)
    px = torch.where(last, 0.0, e[t, x] / z)
    qx = dp[t, x].double() if dp is not None else torch.ones_like(px)
    take = (st["u"].double() * qx < px) & ~last
    stop = torch.where(take, T, t)  # rows that end their sequence's scan
    row = torch.full((S,), T, device=dev).scatter_reduce(0, seq, stop, "amin")
    w = e[row]
    ends = last[row]
    if dp is not None:
        less = torch.clamp(w / z[row][:, None] - dp[row].double(), min=0.0)
        w = torch.where(ends[:, None], w, less)
    else:
        col = torch.arange(V, device=dev)[None]
        w = torch.where(ends[:, None] | (col != x[row][:, None]), w, 0.0)
    c = w.cumsum(1)
    total = c[:, -1:]
    at = (c <= st["us"].double()[:, None] * total).sum(1)
    top = torch.where(w > 0, torch.arange(V, device=dev)[None], -1).amax(1)
    at = torch.where(total[:, 0] > 0, torch.minimum(at, top), lg[row].argmax(1))
    ids = torch.where(t < row[seq], x, torch.where(t == row[seq], at[seq], -1))
    return ids.int(), (row - qs[:-1] + 1).int(), px.float()


# ---- the package's calls -------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if not own:
        return {"plan": _plan, "store": _store, "attn": _attn, "sample": _sample}[op](st)
    S, ctx = _context()
    if op == "plan":
        r = ctx.page_plan(st["past"], st["new"], st["table"], st["free"], st["page"], st["T"], free_head=st["head"])
        return st["table"], r.q_start, r.kv_len, r.pos, r.slots, r.status, r.n_taken
    if op == "store":
        kv = S.F16 if st["kv"] == "f16" else S.Q8_0
        ctx.rope_kv_paged(st["qkv"], st["pos"], st["slots"], st["k"], st["v"], kv, st["q_out"], theta_base=BASE)
        return (st["q_out"],) + _stored(st)
    if op == "attn":
        kv = S.F16 if st["kv"] == "f16" else S.Q8_0
        return ctx.flash_attn_paged(st["q"], st["k"], st["v"], kv, st["table"], st["q_start"], st["kv_len"],
                                    scale=1.0 / math.sqrt(st["D"]), window=st["window"], out=st["out"])
    return ctx.verify_sample(st["logits"], st["ids"], st["q_start"], st["u"], st["us"], draft_probs=st["dp"],
                             temperature=st["temp"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "plan":
        past, new = _lengths(case)
        P = case["page"]
        fresh = sum(-(-(a + b) // P) - -(-a // P) for a, b in zip(past, new))
        # per sequence two lengths in, start, length and status out; a fresh page is read and written; per row its
        # position and slot, and the table entry of each page that rows fall into
        touched = sum((a + b - 1) // P - a // P + 1 for a, b in zip(past, new) if b > 0)
        return {"bytes": 20 * len(past) + 8 * fresh + 4 * touched + 12 * sum(new), "flops": 0}
    if case["op"] == "store":
        n, H, Hkv, D = (case[k] for k in ("rows", "H", "Hkv", "D"))
        qb = 2 if case["q"] == "f16" else 4
        return {"bytes": n * ((H + 2 * Hkv) * D * 4 + 12 + H * D * qb + 2 * Hkv * ROW[case["kv"]](D)),
                "flops": 3 * n * (H + Hkv) * D}
    if case["op"] == "attn":
        past, new = _lengths(case)
        H, Hkv, D, W = (case[k] for k in ("H", "Hkv", "D", "window"))
        seen = read = 0
        for a, b in zip(past, new):
            seen += sum(min(a + i + 1, W) if W > 0 else a + i + 1 for i in range(b))
            read += (min(a + b, W + b - 1) if W > 0 else a + b) if b else 0
        qb = 2 if case["q"] == "f16" else 4
        return {"bytes": 2 * sum(new) * H * D * qb + 2 * read * Hkv * ROW[case["kv"]](D), "flops": 4 * seen * H * D}
    ks = _drafts(case)
    T, S, V = sum(ks) + len(ks), len(ks), case["V"]
    # every row of logits once (each drafted token's probability is asked for), and of the drafter's distributions the
    # one row of each sequence that a rejected token's replacement comes from
    return {"bytes": 4 * V * (T + (S if case["draft"] else 0)) + 16 * T + 12 * S, "flops": 3 * T * V}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "plan":
        return None
    if case["op"] == "store":
        n, H, Hkv, D = (case[k] for k in ("rows", "H", "Hkv", "D"))
        x = st["qkv"].to(f8).view(n, H + 2 * Hkv, D)
        half = D // 2
        freq = torch.tensor([BASE ** (-2.0 * j / D) for j in range(half)], dtype=f8, device=DEV)
        rot = torch.polar(torch.ones((), dtype=f8, device=DEV), st["pos"].to(f8)[:, None] * freq)[:, None, :]
        z = torch.complex(x[:, :H + Hkv, :half], x[:, :H + Hkv, half:]) * rot
        turned = torch.cat([z.real, z.imag], -1)
        parts = []
        for c, rows in ((st["k"], turned[:, H:]), (st["v"], x[:, H + Hkv:])):
            if case["kv"] == "f16":
                flat = c.view(torch.float16).to(f8).flatten(0, 1)
                flat[st["slots"]] = rows
                parts.append(flat.view(c.shape[0], c.shape[1], Hkv, D))
            else:  # the block's step, rounded to f16, times the nearest whole number of 127ths of its largest value
                b = rows.reshape(n, Hkv, D // 32, 32)
                big = b.abs().amax(-1, keepdim=True)
                whole = torch.round(b / big * 127)
                parts.append(((big / 127).to(torch.float16).to(f8) * whole).reshape(n, Hkv, D))
        return (turned[:, :H],) + tuple(parts)
    if case["op"] == "attn":
        past, new = _lengths(case)
        H, Hkv, D, P, W = (case[k] for k in ("H", "Hkv", "D", "page", "window"))
        G, r0 = H // Hkv, 0
        out = torch.zeros((sum(new), H, D), dtype=f8, device=DEV)

        def rows_of(pool, pages, L, h):
            c = pool[pages][:, :, h].flatten(0, 1)[:L]
            if case["kv"] == "f16":
                return c.contiguous().view(torch.float16).to(f8)
            b = c.reshape(L, D // 32, 34)
            step = b[..., :2].contiguous().view(torch.float16).to(f8)
            return (step * b[..., 2:].contiguous().view(torch.int8).to(f8)).to(torch.float16).to(f8).reshape(L, D)

        for s, (a, n) in enumerate(zip(past, new)):
            L = a + n
            pages = st["table"][s, :-(-L // P)].long()
            for h in range(Hkv):
                if n == 0:
                    continue
                k, v = rows_of(st["k"], pages, L, h), rows_of(st["v"], pages, L, h)
                at = torch.arange(L, device=DEV)
                here = torch.arange(a, L, device=DEV)[:, None]
                hide = (at > here) | ((at <= here - W) if W > 0 else (at < 0))
                for g in range(G):
                    sc = st["q"][r0:r0 + n, h * G + g].to(f8) @ k.T / math.sqrt(D)
                    sc[hide] = -math.inf
                    out[r0:r0 + n, h * G + g] = torch.softmax(sc, 1) @ v
            r0 += n
        return out
    ks = _drafts(case)
    T, V = st["logits"].shape
    ids = torch.full((T,), -1, dtype=torch.int32)
    cnt, probs, r0 = [], torch.zeros(T, dtype=f8), 0
    tok, u, us = st["ids"].tolist(), st["u"].tolist(), st["us"].tolist()
    for s, k in enumerate(ks):
        rows = st["logits"][r0:r0 + k + 1].to(f8) / st["temp"][s].to(f8)
        p = torch.softmax(rows, 1)
        xs = torch.tensor(tok[r0 + 1:r0 + k + 1] + [0], device=DEV)
        px = p[torch.arange(k + 1, device=DEV), xs].tolist()
        qx = st["dp"][torch.arange(r0, r0 + k + 1, device=DEV), xs].tolist() if st["dp"] is not None else [1.0] * (k + 1)
        probs[r0:r0 + k] = torch.tensor(px[:k], dtype=f8)
        i = 0
        while i < k and u[r0 + i] * qx[i] < px[i]:
            ids[r0 + i] = tok[r0 + i + 1]
            i += 1
        w = p[i].clone()
        if i < k and st["dp"] is not None:
            w = torch.relu(w - st["dp"][r0 + i].to(f8))
        elif i < k:
            w[tok[r0 + i + 1]] = 0.0
        c = w.cumsum(0)
        ids[r0 + i] = int(torch.searchsorted(c, us[s] * c[-1], right=True).clamp(max=V - 1))
        cnt.append(i + 1)
        r0 += k + 1
    return ids, torch.tensor(cnt, dtype=torch.int32), probs
