"""Workloads of a paged cache held in 4 bits, of pages that sequences share, and of rules on logits: RoPE with a paged
store into q4_0 rows and attention over them; forks of sequences with their page copies, finished sequences' pages given
back and the rest moved together; penalties, biases and token masks on the rows that a step scores. Each is given in plain
torch (`own` false) and as the calls that a serving loop makes of this package (`own` true)."""
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
        # the 9 token rows of one verify step of the 27B-class decoder (24 query, 4 KV heads of 256)
        {"name": "store4_verify", "op": "store", "rows": 9, "H": 24, "Hkv": 4, "D": 256, "q": "f32", "page": 64,
         "pos_hi": 131072},
        # a prompt chunk of a decoder with 32 query and 8 KV heads of 128
        {"name": "store4_prompt", "op": "store", "rows": 8192, "H": 32, "Hkv": 8, "D": 128, "q": "f16", "page": 16,
         "pos_hi": 32768},
        # one chat sequence decoding, a few hundred tokens in: latency
        {"name": "attn4_one", "op": "attn", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 300, "past_hi": 300,
         "H": 28, "Hkv": 4, "D": 128, "q": "f16", "page": 16, "window": 0, "lens": 1},
        # plain decoding of a batch: one token each over caches of unequal lengths
        {"name": "attn4_decode", "op": "attn", "seqs": 32, "new_lo": 1, "new_hi": 1, "past_lo": 500, "past_hi": 8192,
         "H": 32, "Hkv": 8, "D": 128, "q": "f16", "page": 16, "window": 0, "lens": 3},
        # one verify step at the long-context length of the 27B-class decoder, full precision rows
        {"name": "attn4_verify_long", "op": "attn", "seqs": 1, "new_lo": 9, "new_hi": 9, "past_lo": 131063,
         "past_hi": 131063, "H": 24, "Hkv": 4, "D": 256, "q": "f32", "page": 64, "window": 0, "lens": 4},
        # a chunk of a long prompt: 2048 new tokens behind 30720 cached ones
        {"name": "attn4_chunk", "op": "attn", "seqs": 1, "new_lo": 2048, "new_hi": 2048, "past_lo": 30720,
         "past_hi": 30720, "H": 24, "Hkv": 4, "D": 256, "q": "f16", "page": 64, "window": 0, "lens": 6},
        # four answers sampled for one prompt: three forks of it, small model, q8_0 cache
        {"name": "fork_samples", "op": "fork", "parents": 1, "forks": 3, "len_lo": 1000, "len_hi": 1000, "layers": 24,
         "Hkv": 2, "D": 64, "kv": "q8_0", "page": 16, "lens": 5},
        # a batch of prompts that go on as several branches each, f16 cache of the 27B-class decoder's heads
        {"name": "fork_batch", "op": "fork", "parents": 24, "forks": 64, "len_lo": 100, "len_hi": 900, "layers": 24,
         "Hkv": 4, "D": 256, "kv": "f16", "page": 64, "lens": 6},
        # some sequences of a large server's step are done: their pages go back, those that others share stay
        {"name": "release_done", "op": "release", "seqs": 1024, "done": 48, "len_lo": 1, "len_hi": 8192, "page": 16,
         "compact": False, "layers": 1, "Hkv": 1, "D": 64, "kv": "q4_0", "lens": 7},
        # most sequences are done and the pool is to shrink: the pages of the rest move together
        {"name": "release_shrink", "op": "release", "seqs": 48, "done": 28, "len_lo": 100, "len_hi": 4000, "page": 64,
         "compact": True, "layers": 16, "Hkv": 8, "D": 128, "kv": "q8_0", "lens": 8},
        # one sequence, 8 drafted tokens: penalties over the last 64 tokens
        {"name": "logits_one", "op": "logits", "seqs": 1, "k_lo": 8, "k_hi": 8, "V": 151936, "hist": 4096, "last_n": 64,
         "bias": 0, "mask": False, "lens": 9},
        # a batch: penalties over long windows, biases, and grammars on some of the rows
        {"name": "logits_batch", "op": "logits", "seqs": 64, "k_lo": 2, "k_hi": 8, "V": 151936, "hist": 8192,
         "last_n": 4096, "bias": 40, "mask": True, "lens": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attn", "attn", "attn", "fork", "release", "logits"])
    page = rng.choice([16, 32, 48, 64, 80, 128, 256])
    lens = rng.randrange(1 << 30)
    H, Hkv, D = rng.choice([(24, 4, 256), (16, 16, 64), (32, 8, 128), (6, 2, 256), (28, 4, 128), (8, 1, 64)])
    kv = rng.choice(["f16", "q8_0", "q4_0"])
    if op == "store":
        return {"op": op, "rows": _log(rng, 1, 4000), "H": H, "Hkv": Hkv, "D": D, "q": rng.choice(["f16", "f32"]),
                "page": page, "pos_hi": _log(rng, 8192, 131072)}
    if op == "attn":
        seqs = _log(rng, 1, 32)
        past_hi = _log(rng, 1, 65536 // seqs)
        new_hi = rng.choice([1, rng.randint(2, 16), _log(rng, 1, min(2000, 8192 // seqs))])
        new_hi = max(1, min(new_hi, 2 ** 38 // (seqs * past_hi * H * D)))  # no more work than the listed chunk's
        return {"op": op, "seqs": seqs, "new_lo": 1, "new_hi": new_hi, "past_lo": 0, "past_hi": past_hi, "H": H,
                "Hkv": Hkv, "D": D, "q": rng.choice(["f16", "f16", "f32"]), "page": page,
                "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "lens": lens}
    if op == "fork":
        return {"op": op, "parents": _log(rng, 1, 24), "forks": _log(rng, 1, 64), "len_lo": 0,
                "len_hi": _log(rng, 1, 900), "layers": rng.randint(1, 24), "Hkv": min(Hkv, 4), "D": D, "kv": kv,
                "page": min(page, 64), "lens": lens}
    if op == "release":
        seqs = _log(rng, 1, 1000)
        compact = rng.random() < 0.6
        len_hi = _log(rng, 16, max(16, min(4000, (60000 if compact else 2000000) // seqs)))
        return {"op": op, "seqs": seqs, "done": rng.randint(0, seqs), "len_lo": 0, "len_hi": len_hi, "page": page,
                "compact": compact, "layers": rng.randint(1, 12), "Hkv": min(Hkv, 4), "D": D, "kv": kv, "lens": lens}
    return {"op": op, "seqs": _log(rng, 1, 60), "k_lo": 0, "k_hi": rng.randrange(1, 9), "V": _log(rng, 500, 151936),
            "hist": _log(rng, 1, 8192), "last_n": rng.choice([0, 64, _log(rng, 1, 8192), -1]),
            "bias": rng.choice([0, _log(rng, 1, 300)]), "mask": rng.random() < 0.6, "lens": lens}


def _lengths(case):
    """(past, new) of each sequence: part of the case, not of its inputs."""
    rng = random.Random(case["lens"])
    past, new = [], []
    for _ in range(case["seqs"]):
        past.append(rng.randint(case["past_lo"], case["past_hi"]))
        hi, lo = case["new_hi"], case["new_lo"]
        # most sequences of a batch decode or verify, some bring a prompt
        new.append(rng.randint(lo, hi if hi <= 16 or rng.random() < 0.4 else max(lo, 16)))
    return past, new


def _branches(case):
    """Lengths of the parents; per fork its parent and the tokens that it keeps."""
    rng = random.Random(case["lens"])
    n = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["parents"])]
    who = [rng.randrange(case["parents"]) for _ in range(case["forks"])]
    # most branches start behind the parent's last token, some share a prefix only
    keep = [n[p] if rng.random() < 0.8 else rng.randint(0, n[p]) for p in who]
    return n, who, keep


def _sharing(case):
    """Pages of each sequence, how many of them it shares with the one before it, and the sequences that are done."""
    rng = random.Random(case["lens"])
    nb = [-(-rng.randint(case["len_lo"], case["len_hi"]) // case["page"]) for _ in range(case["seqs"])]
    shared = [0] + [rng.randint(0, min(a, b)) if rng.random() < 0.3 else 0 for a, b in zip(nb, nb[1:])]
    done = rng.sample(range(case["seqs"]), case["done"])
    return nb, shared, done


def _drafts(case):
    rng = random.Random(case["lens"])
    return [rng.randint(case["k_lo"], case["k_hi"]) for _ in range(case["seqs"])]


def _rules(case):
    """Tokens in each sequence's history, its biased tokens, and the token mask of each row (-1: none)."""
    rng = random.Random(case["lens"] + 1)
    ks, C = _drafts(case), case["hist"]
    nh = [rng.randint(C // 2, C) for _ in ks]
    nbias = [rng.randint(0, case["bias"]) for _ in ks]
    rows, used = [], 0
    for k in ks:  # a grammar's rows each have their set; the other sequences are free
        bound = case["mask"] and rng.random() < 0.5
        rows += list(range(used, used + k + 1)) if bound else [-1] * (k + 1)
        used += k + 1 if bound else 0
    return nh, nbias, rows


# ---- inputs --------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(n):
    at = [0]
    for k in n:
        at.append(at[-1] + k)
    return _i32(at)


ROW = {"f16": lambda D: 2 * D, "q8_0": lambda D: D // 32 * 34, "q4_0": lambda D: D // 32 * 18}


def _cache4(pages, page, Hkv, D, g):
    """A pool of pages uint8 [pages, page, Hkv, row bytes] of q4_0 blocks (the step d of either sign as f16, then 16 bytes:
    value j in the low, value j + 16 in the high half of byte j) that hold values of unit size."""
    b = torch.randint(0, 256, (pages, page, Hkv, D // 32, 18), device=DEV, generator=g, dtype=torch.uint8)
    d = torch.rand((pages, page, Hkv, D // 32, 1), device=DEV, generator=g) * 0.2 + 0.1
    d = torch.where(b[..., 2:3] < 128, d, -d).half()
    b[..., :2] = d.view(torch.uint8)
    return b.view(pages, page, Hkv, -1)


def _pools(case, pages, g):
    """K and V pools of all layers, uint8 [layers, 2, pages, page, Hkv, row bytes]: only copied here."""
    row = ROW[case["kv"]](case["D"])
    shape = (case["layers"], 2, pages, case["page"], case["Hkv"], row)
    return torch.randint(0, 256, shape, device=DEV, generator=g, dtype=torch.uint8)


def _book(parts):
    """Named int32 tensors as views of one, and a copy of it: a pass begins with the books as they were before the step."""
    flat = [p.int().reshape(-1) for p in parts.values()]
    book = torch.cat(flat)
    views, at = {}, 0
    for (name, p), f in zip(parts.items(), flat):
        views[name] = book[at:at + f.numel()].view(p.shape)
        at += f.numel()
    return book, book.clone(), views


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    op = case["op"]
    if op == "store":
        n, H, Hkv, D, P = (case[k] for k in ("rows", "H", "Hkv", "D", "page"))
        pages = -(-n // P) + 3
        st |= {"qkv": torch.randn((n, (H + 2 * Hkv) * D), device=DEV, generator=g),
               "pos": torch.randint(0, case["pos_hi"], (n,), device=DEV, generator=g).int(),
               "slots": torch.randperm(pages * P, device=DEV, generator=g)[:n].contiguous(),
               "k": _cache4(pages, P, Hkv, D, g), "v": _cache4(pages, P, Hkv, D, g),
               "q_out": torch.empty((n, H, D), device=DEV, dtype=torch.float16 if case["q"] == "f16" else torch.float32)}
    elif op == "attn":
        past, new = _lengths(case)
        H, Hkv, D, P = (case[k] for k in ("H", "Hkv", "D", "page"))
        nb = [-(-(a + b) // P) for a, b in zip(past, new)]
        pages = sum(nb) + 3
        table = torch.full((case["seqs"], max(nb)), -1, dtype=torch.int32, device=DEV)
        held = torch.arange(max(nb), device=DEV)[None, :] < _i32(nb)[:, None]
        table[held] = torch.randperm(pages, device=DEV, generator=g)[:sum(nb)].int()
        t = torch.float16 if case["q"] == "f16" else torch.float32
        T = sum(new)
        st |= {"table": table, "q_start": _starts(new), "kv_len": _i32([a + b for a, b in zip(past, new)]),
               "Lmax": max(a + b for a, b in zip(past, new)), "Nmax": max(new), "T": T,
               "q": torch.randn((T, H, D), device=DEV, generator=g).to(t), "k": _cache4(pages, P, Hkv, D, g),
               "v": _cache4(pages, P, Hkv, D, g), "out": torch.empty((T, H, D), device=DEV, dtype=t)}
    elif op == "fork":
        n, who, keep = _branches(case)
        P = case["page"]
        nb = [-(-k // P) for k in n]
        rows, cols = len(n) + len(who), max(nb) + 2
        pages = sum(nb) + len(who) + 5
        pool = torch.randperm(pages, device=DEV, generator=g).int()
        table = torch.full((rows, cols), -1, dtype=torch.int32, device=DEV)
        held = torch.arange(cols, device=DEV)[None, :] < _i32(nb + [0] * len(who))[:, None]
        table[held] = pool[:sum(nb)]
        order = torch.randperm(len(who), device=DEV, generator=g)
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        book, before, views = _book({"table": table, "refs": refs})
        pools = _pools(case, pages, g)
        st |= views | {"book": book, "before": before, "parent": _i32(who)[order].contiguous(),
                       "child": (_i32(list(range(len(who)))) + len(n))[order].contiguous(),
                       "keep": _i32(keep)[order].contiguous(), "free": pool, "head": _i32([sum(nb)]), "pools": pools,
                       "caches": list(pools.flatten(0, 1).unbind(0))}
    elif op == "release":
        nb, shared, done = _sharing(case)
        S, cols = case["seqs"], max(max(nb), 1) + 1
        fresh = [a - b for a, b in zip(nb, shared)]
        pages = sum(fresh) + 9
        pool = torch.randperm(pages, device=DEV, generator=g).int()
        table = torch.full((S, cols), -1, dtype=torch.int32)
        refs = torch.zeros(pages, dtype=torch.int32)
        names, at = pool.cpu(), 0
        for s in range(S):  # the first pages of the sequence before it, then its own
            if shared[s]:
                table[s, :shared[s]] = table[s - 1, :shared[s]]
                refs[table[s, :shared[s]].long()] += 1
            table[s, shared[s]:nb[s]] = names[at:at + fresh[s]]
            at += fresh[s]
        held = torch.tensor(nb, dtype=torch.int32)
        left = held.clone()
        left[done] = 0
        book, before, views = _book({"table": table.to(DEV), "refs": refs.to(DEV), "free": pool, "head": _i32([at])})
        pools = _pools(case, pages if case["compact"] else 1, g)
        st |= views | {"book": book, "before": before, "done_rows": _i32(done), "begin": _i32([0] * len(done)),
                       "end": held[done].to(DEV), "left": left.to(DEV), "pools": pools,
                       "caches": list(pools.flatten(0, 1).unbind(0)),
                       "src": torch.full((pages // 2 + 1,), -1, dtype=torch.int32, device=DEV),
                       "dst": torch.full((pages // 2 + 1,), -1, dtype=torch.int32, device=DEV)}
    else:
        ks = _drafts(case)
        S, T, V, C = len(ks), sum(ks) + len(ks), case["V"], case["hist"]
        lg = torch.randn((T, V), device=DEV, generator=g) * 4.0

        def words(shape):  # text repeats itself: few tokens make up most of it
            return (torch.rand(shape, device=DEV, generator=g) ** 4 * V).int().clamp(max=V - 1)

        nh, nbias, mask_row = _rules(case)
        b_ids = torch.cat([torch.randperm(V, device=DEV, generator=g)[:n] for n in nbias]).int()
        n_masks = max(1, max(mask_row) + 1)
        mask = torch.randint(-2 ** 31, 2 ** 31, (n_masks, -(-V // 32)), device=DEV, generator=g).int()
        mask &= torch.randint(-2 ** 31, 2 ** 31, mask.shape, device=DEV, generator=g).int()
        st |= {"logits": lg, "ids": words((T,)), "q_start": _starts([k + 1 for k in ks]), "history": words((S, C)),
               "n_history": _i32(nh), "last": torch.full((S,), case["last_n"], dtype=torch.int32, device=DEV),
               "repeat": 1.0 + 0.3 * torch.rand((S,), device=DEV, generator=g),
               "frequency": 0.2 * torch.rand((S,), device=DEV, generator=g),
               "presence": 0.5 * torch.rand((S,), device=DEV, generator=g),
               "bias_ids": b_ids, "bias_val": 3.0 * torch.randn((sum(nbias),), device=DEV, generator=g),
               "bias_start": _starts(nbias), "mask_bits": mask if case["mask"] else None,
               "mask_row": _i32(mask_row) if case["mask"] else None, "out": torch.empty_like(lg)}
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------
BASE = 1e6


def _turn(x, pos):
    """NeoX rotation of rows x [n, heads, D] at positions pos in 64 bits, rounded to 32."""
    half = x.shape[-1] // 2
    j = torch.arange(half, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None] * torch.exp(-math.log(BASE) * 2.0 * j / (2 * half))
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, a * s + b * c], -1).float()


def _pack_q4(x):
    """q4_0 blocks of rows x [..., D]: uint8 [..., D / 32 * 18]. The step is -1/8 of the value of largest size, so that this
    one is kept best: as number 0 of 16, which stands for -8."""
    b = x.unflatten(-1, (-1, 32))
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = big / -8.0
    q = (b * torch.where(d != 0, 1.0 / d, 0.0) + 8.5).to(torch.int32).clamp(max=15).to(torch.uint8)
    return torch.cat([d.half().view(torch.uint8), q[..., :16] | q[..., 16:] << 4], -1).flatten(-2)


def _values(c):
    """The values that q4_0 rows [..., row bytes] stand for, d * (q - 8) rounded to f16."""
    b = c.unflatten(-1, (-1, 18))
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(torch.int8) - 8
    return (d * q.float()).half().flatten(-2)


def _stored(st):
    """The values of the rows that were written."""
    return tuple(_values(st[c].flatten(0, 1)[st["slots"]]) for c in ("k", "v"))


def _store(st):
    n, H, Hkv, D = (st[k] for k in ("rows", "H", "Hkv", "D"))
    x = st["qkv"].view(n, H + 2 * Hkv, D)
    turned = _turn(x[:, :H + Hkv], st["pos"])
    st["k"].flatten(0, 1)[st["slots"]] = _pack_q4(turned[:, H:])
    st["v"].flatten(0, 1)[st["slots"]] = _pack_q4(x[:, H + Hkv:])
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
    k = _values(st["k"][pages, j % P]).float().permute(0, 2, 3, 1)
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
    v = _values(st["v"][pages, j % P]).float().permute(0, 2, 1, 3)
    v = torch.where((j[None] < kl[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(s.view(S, Hkv, G * N, L), v).view(S, Hkv, G, N, D)
    o = (o / torch.where(z > 0, z, 1.0)).permute(0, 3, 1, 2, 4).reshape(S, N, H, D)
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(qs, t, right=True) - 1
    st["out"].copy_(o[seq, t - qs[seq]])
    return st["out"]


def _fork(st):
    P, table, refs = st["page"], st["table"], st["refs"]
    parent, child, keep, free = st["parent"].long(), st["child"].long(), st["keep"].long(), st["free"]
    st["book"].copy_(st["before"])
    cols = table.shape[1]
    full, part = keep // P, (keep % P > 0).long()
    status = torch.where(full + part > cols, 1, 0)
    need = torch.where(status == 0, part, 0)
    at = st["head"].long() + need.cumsum(0)
    status = torch.where((need > 0) & (at > free.numel()), 2, status)
    ok = status == 0
    taken = torch.where(ok & (need > 0), need.cumsum(0), 0).amax()
    fresh = free[(at - 1).clamp(0, free.numel() - 1)]
    col = torch.arange(cols, device=table.device)[None, :]
    share = ok[:, None] & (col < full[:, None])
    names = table[parent]
    refs.scatter_add_(0, names.long().clamp(min=0).flatten(), share.int().flatten())
    own_page = ok & (part > 0)
    last = own_page[:, None] & (col == full[:, None])
    table[child] = torch.where(share, names, torch.where(last, fresh[:, None], table[child]))
    src = torch.where(own_page, names.gather(1, full.clamp(max=cols - 1)[:, None])[:, 0], -1)
    dst = torch.where(own_page, fresh, -1)
    a, b = src[own_page].long(), dst[own_page].long()
    st["pools"][:, :, b] = st["pools"][:, :, a]
    return table, refs, src.int(), dst.int(), status.int(), taken.int().view(1), st["pools"].view(torch.int16)


def _release(st):
    table, refs, free, head = st["table"], st["refs"], st["free"], st["head"]
    st["book"].copy_(st["before"])
    n_pages, cols = refs.numel(), table.shape[1]
    dev = table.device
    page = torch.arange(n_pages, device=dev)
    col = torch.arange(cols, device=dev)[None, :]
    rows = st["done_rows"].long()
    gone = (col >= st["begin"][:, None]) & (col < st["end"][:, None])
    names = torch.where(gone, table[rows], -1)
    drop = torch.zeros(n_pages + 1, dtype=torch.int32, device=dev)
    drop.scatter_add_(0, torch.where(names >= 0, names, n_pages).long().flatten(),
                      torch.ones_like(names).flatten())
    drop = drop[:n_pages]
    table[rows] = torch.where(gone, -1, table[rows])
    freed = drop > refs  # all of its 1 + refs holders
    refs.copy_((refs - drop).clamp(min=0))
    n_freed = freed.sum()
    rank = freed.cumsum(0) - 1
    spot = torch.where(freed, head.long() - n_freed + rank, n_pages)
    free.copy_(torch.cat([free, free[:1]]).scatter(0, spot, page.int())[:n_pages])
    head.sub_(n_freed.int())
    out = (table, refs, free, head, n_freed.int().view(1))
    if not st["compact"]:
        return out
    mine = col < st["left"][:, None]
    count = torch.zeros(n_pages + 1, dtype=torch.int32, device=dev)
    count.scatter_(0, torch.where(mine & (table >= 0), table, n_pages).long().flatten(), 1)
    used = count[:n_pages] > 0
    n_used = used.sum()
    high, hole = used & (page >= n_used), ~used & (page < n_used)
    src, dst = page[high], page[hole]
    to = page.clone()
    to[src] = dst
    table.copy_(torch.where(mine & (table >= 0), to[table.long().clamp(min=0)].int(), table))
    refs[dst] = refs[src]
    refs[src] = 0
    free.copy_(torch.where(page >= n_used, page.int(), free))
    head.copy_(n_used.int().view(1))
    st["src"][:src.numel()], st["dst"][:dst.numel()] = src.int(), dst.int()
    st["pools"][:, :, dst] = st["pools"][:, :, src]
    return out + (st["src"], st["dst"], n_used.int().view(1), high.sum().int().view(1), st["pools"].view(torch.int16))


def _logits(st):
    lg, ids, qs = st["logits"], st["ids"].long(), st["q_start"].long()
    T, V = lg.shape
    S, C = st["history"].shape
    dev = lg.device
    r = torch.arange(T, device=dev)
    seq = torch.searchsorted(qs, r, right=True) - 1
    first, nh = qs[seq], st["n_history"].long()[seq]
    total = nh + r - first + 1  # tokens ahead of the one that row r scores
    last = st["last"].long()[seq]
    begin = torch.where(last < 0, 0, (total - last).clamp(min=0))
    # the history's part of the window, then that of the step's rows
    j = torch.arange(C, device=dev)[None, :]
    count = torch.zeros((T, V), device=dev)
    inside = (j >= begin[:, None]) & (j < nh[:, None])
    count.scatter_add_(1, st["history"].long()[seq], inside.float())
    k = torch.arange(int(st["k_hi"]) + 1, device=dev)[None, :]
    inside = (first[:, None] + k <= r[:, None]) & (nh[:, None] + k >= begin[:, None])
    count.scatter_add_(1, ids[(first[:, None] + k).clamp(max=T - 1)], inside.float())
    l = lg.clone()
    if st["bias_ids"].numel():
        b = torch.zeros((S, V), device=dev)
        e = torch.arange(st["bias_ids"].numel(), device=dev)
        b[torch.searchsorted(st["bias_start"].long(), e, right=True) - 1, st["bias_ids"].long()] = st["bias_val"]
        l += b[seq]
    rep = st["repeat"][seq][:, None]
    less = torch.where(l > 0, l / rep, l * rep) - (count * st["frequency"][seq][:, None] + st["presence"][seq][:, None])
    l = torch.where(count > 0, less, l)
    if st["mask_bits"] is not None:
        x = torch.arange(V, device=dev)
        row = st["mask_row"].long()
        bits = st["mask_bits"][row.clamp(min=0)][:, x // 32] >> (x % 32).int() & 1
        l = torch.where((row[:, None] >= 0) & (bits == 0), -math.inf, l)
    st["out"].copy_(l)
    return st["out"]


# ---- the package's calls -------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if not own:
        return {"store": _store, "attn": _attn, "fork": _fork, "release": _release, "logits": _logits}[op](st)
    S, ctx = _context()
    if op == "store":
        ctx.rope_kv_paged(st["qkv"], st["pos"], st["slots"], st["k"], st["v"], S.Q4_0, st["q_out"], theta_base=BASE)
        return (st["q_out"],) + _stored(st)
    if op == "attn":
        return ctx.flash_attn_paged(st["q"], st["k"], st["v"], S.Q4_0, st["table"], st["q_start"], st["kv_len"],
                                    scale=1.0 / math.sqrt(st["D"]), window=st["window"], out=st["out"])
    kv = {"f16": S.F16, "q8_0": S.Q8_0, "q4_0": S.Q4_0}
    if op == "fork":
        st["book"].copy_(st["before"])
        f = ctx.page_fork(st["parent"], st["child"], st["keep"], st["table"], st["refs"], st["free"], st["page"],
                          free_head=st["head"])
        ctx.page_copy(st["caches"], kv[st["kv"]], f.src, f.dst)
        return st["table"], st["refs"], f.src, f.dst, f.status, f.n_taken, st["pools"].view(torch.int16)
    if op == "release":
        st["book"].copy_(st["before"])
        n_freed = ctx.page_free(st["done_rows"], st["begin"], st["end"], st["table"], st["refs"], st["free"], st["head"])
        st["head"].sub_(n_freed)
        out = (st["table"], st["refs"], st["free"], st["head"], n_freed)
        if not st["compact"]:
            return out
        c = ctx.page_compact(st["table"], st["left"], st["refs"], st["free"], out=(st["src"], st["dst"]))
        st["head"].copy_(c.n_used)
        ctx.page_copy(st["caches"], kv[st["kv"]], c.src, c.dst, n_moves=c.n_moves)
        return out + (c.src, c.dst, c.n_used, c.n_moves, st["pools"].view(torch.int16))
    bias = (st["bias_start"], st["bias_ids"], st["bias_val"]) if st["bias_ids"].numel() else None
    return ctx.adjust_logits(st["logits"], st["ids"], st["q_start"], history=st["history"], n_history=st["n_history"],
                             last_n=st["last"], repeat=st["repeat"], frequency=st["frequency"],
                             presence=st["presence"], bias=bias, mask=st["mask_bits"], mask_row=st["mask_row"],
                             out=st["out"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "store":
        n, H, Hkv, D = (case[k] for k in ("rows", "H", "Hkv", "D"))
        qb = 2 if case["q"] == "f16" else 4
        return {"bytes": n * ((H + 2 * Hkv) * D * 4 + 12 + H * D * qb + 2 * Hkv * ROW["q4_0"](D)),
                "flops": 3 * n * (H + Hkv) * D}
    if op == "attn":
        past, new = _lengths(case)
        H, Hkv, D, W = (case[k] for k in ("H", "Hkv", "D", "window"))
        seen = read = 0
        for a, b in zip(past, new):
            seen += sum(min(a + i + 1, W) if W > 0 else a + i + 1 for i in range(b))
            read += (min(a + b, W + b - 1) if W > 0 else a + b) if b else 0
        qb = 2 if case["q"] == "f16" else 4
        return {"bytes": 2 * sum(new) * H * D * qb + 2 * read * Hkv * ROW["q4_0"](D), "flops": 4 * seen * H * D}
    if op in ("fork", "release"):
        page = 2 * case["layers"] * case["page"] * case["Hkv"] * ROW[case["kv"]](case["D"])  # of all layers
    if op == "fork":
        _, _, keep = _branches(case)
        P = case["page"]
        full, part = sum(k // P for k in keep), sum(k % P > 0 for k in keep)
        # per fork three numbers in, three out; a shared page's entry is read and written and its count changed
        return {"bytes": 24 * len(keep) + 16 * full + 12 * part + 2 * part * page, "flops": 0}
    if op == "release":
        nb, shared, done = _sharing(case)
        gone = sum(nb[s] for s in done)
        b = 12 * len(done) + 20 * gone  # entry read and cleared, count changed, page written into the list
        if case["compact"]:
            gone_set = set(done)
            left = [s for s in range(len(nb)) if s not in gone_set]
            # distinct pages of the rest: a run of sequences that share their first pages counts those once
            used, named, names = 0, {}, 0
            for s in range(len(nb)):
                named[s] = (named[s - 1][:shared[s]] if shared[s] else []) + list(range(names, names + nb[s] - shared[s]))
                names += nb[s] - shared[s]
            used = len({p for s in left for p in named[s]})
            moves = used * (names + 9 - used) / (names + 9)  # used pages behind the first n_used, on average
            b += 4 * sum(nb[s] for s in left) + moves * (8 + 8 + 2 * page) + 4 * (names + 9 - used)
        return {"bytes": b, "flops": 0}
    ks = _drafts(case)
    T, V = sum(ks) + len(ks), case["V"]
    nh, nbias, rows = _rules(case)
    said = sum(n if case["last_n"] < 0 else min(case["last_n"], n) for n in nh)
    return {"bytes": 8 * T * V + sum(r >= 0 for r in rows) * (-(-V // 32) * 4) + 4 * (said + T) + 8 * sum(nbias), "flops": T * V}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op in ("fork", "release"):
        return None
    st = prepare(case, seed)
    f8 = torch.float64
    if op == "store":
        n, H, Hkv, D = (case[k] for k in ("rows", "H", "Hkv", "D"))
        x = st["qkv"].to(f8).view(n, H + 2 * Hkv, D)
        half = D // 2
        freq = torch.tensor([BASE ** (-2.0 * j / D) for j in range(half)], dtype=f8, device=DEV)
        rot = torch.polar(torch.ones((), dtype=f8, device=DEV), st["pos"].to(f8)[:, None] * freq)[:, None, :]
        z = torch.complex(x[:, :H + Hkv, :half], x[:, :H + Hkv, half:]) * rot
        turned = torch.cat([z.real, z.imag], -1)
        parts = []
        for rows in (turned[:, H:], x[:, H + Hkv:]):
            b = rows.reshape(n, Hkv, D // 32, 32)
            lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
            step = torch.where(hi > -lo, hi, lo) / -8.0
            whole = torch.floor(b / step + 8.5).clamp(max=15) - 8.0
            parts.append((step.to(torch.float16).to(f8) * whole).reshape(n, Hkv, D))
        return (turned[:, :H],) + tuple(parts)
    if op == "attn":
        past, new = _lengths(case)
        H, Hkv, D, P, W = (case[k] for k in ("H", "Hkv", "D", "page", "window"))
        G, r0 = H // Hkv, 0
        out = torch.zeros((sum(new), H, D), dtype=f8, device=DEV)

        def rows_of(pool, pages, L, h):
            b = pool[pages][:, :, h].flatten(0, 1)[:L].reshape(L, D // 32, 18)
            step = b[..., :2].contiguous().view(torch.float16).to(f8)
            num = b[..., 2:].to(torch.int32)
            whole = torch.cat([num % 16, num // 16], -1).to(f8) - 8.0
            return (step * whole).to(torch.float16).to(f8).reshape(L, D)

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
    out = st["logits"].to(f8)
    nh, start, r0 = st["n_history"].tolist(), st["bias_start"].tolist(), 0
    x = torch.arange(V, device=DEV)
    for s, k in enumerate(ks):
        said = st["history"][s, :nh[s]]
        for r in range(r0, r0 + k + 1):
            before = torch.cat([said, st["ids"][r0:r + 1]]).long()
            if case["last_n"] >= 0:
                before = before[max(0, before.numel() - case["last_n"]):]
            seen, times = torch.unique(before, return_counts=True)
            row = out[r]
            at = st["bias_ids"][start[s]:start[s + 1]].long()
            row[at] = row[at] + st["bias_val"][start[s]:start[s + 1]].to(f8)
            v = row[seen]
            v = torch.where(v > 0, v / st["repeat"][s].to(f8), v * st["repeat"][s].to(f8))
            row[seen] = v - times.to(f8) * st["frequency"][s].to(f8) - st["presence"][s].to(f8)
            if case["mask"] and int(st["mask_row"][r]) >= 0:
                word = st["mask_bits"][int(st["mask_row"][r])].to(torch.int64) & 0xffffffff
                row[(word[x // 32] >> (x % 32)) % 2 == 0] = -math.inf
        r0 += k + 1
    return out
