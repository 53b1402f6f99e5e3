"""Paged KV caches and token sampling, as timed cases.

A case is a step that a serving loop takes between two layers' products: a few
new tokens' attention over caches held in pages, the write of new rows into
their pages, forks of sequences with the copies of the pages they part at,
the compaction of a pool of pages, and the draw of the next token of every
sequence from its logits and a given random number.  ``listed`` holds sizes of
this repository's tests and benchmark, or generic ones; ``draw`` gives others
of the same ranges.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
by the framework's kernels.

Pages: a pool [(layers,) pages, 2, G, P, D] holds K and V of P rows of every
KV head a page; row n of sequence b lies in page tables[b, n // P], row n % P;
refs counts the table entries that name a page, 0: free.  New pages are the
lowest free ones, handed out in the order of the sequences.

Sampling: weights exp((logit - largest) / temperature) of the top_k largest
logits (ties: the lower token first), of these the shortest run of the largest
that holds top_p of their sum, of these the ones of at least min_p of the
largest weight; the token is the first, by number, up to which the kept
weights sum to more than u of their sum.  Temperature 0: the largest logit.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = [(9, 3, 64), (9, 3, 64), (12, 4, 64), (32, 8, 128), (8, 8, 128), (16, 2, 128)]


def listed():
    small = {"heads": 9, "kv_heads": 3, "dim": 64}
    large = {"heads": 32, "kv_heads": 8, "dim": 128}
    # 32 sequences of 4K to 131K rows, as a packed server batch holds them
    ragged = ",".join(str(4096 + (131072 - 4096) * i // 31 - (i * 37) % 64) for i in range(32))
    return [
        # a token of one short conversation with a model kept in fp32: the smallest call
        {"name": "attend_1k", "kind": "attend", "tokens": 1, "lens": "1000", "page": 16, "dtype": "fp32", **small},
        # a decode step of a continuous batch
        {"name": "attend_ragged", "kind": "attend", "tokens": 1, "lens": ragged, "page": 32, "dtype": "bf16", **small},
        # the same of a wide model, up to 42K rows
        {"name": "attend_wide", "kind": "attend", "tokens": 1,
         "lens": ",".join(str(1024 + 1777 * i) for i in range(24)), "page": 64, "dtype": "bf16", **large},
        # four drafted tokens of each of eight sequences being checked
        {"name": "attend_4_32k", "kind": "attend", "tokens": 4, "lens": ",".join(["32768"] * 8), "page": 16,
         "dtype": "fp16", "heads": 12, "kv_heads": 4, "dim": 64},
        # a decode step's new rows of a batch
        {"name": "write_32", "kind": "write", "seqs": 32, "tokens": 1, "rows": 8192, "page": 16, "dtype": "bf16",
         **small},
        # a long prompt's rows
        {"name": "write_131k", "kind": "write", "seqs": 1, "tokens": 131072, "rows": 131072, "page": 64,
         "dtype": "bf16", **large},
        # two of four beams go on as the others, a row each behind 500 shared ones, in all layers of the small model
        {"name": "fork_beams", "kind": "fork", "layers": 30, "parents": 2, "forks": 1, "rows": 500, "page": 16,
         "pages": 256, "dtype": "bf16", **small},
        # seven samples each of eight prompts of about 2000 rows part from them
        {"name": "fork_samples", "kind": "fork", "layers": 16, "parents": 8, "forks": 7, "rows": 2000, "page": 64,
         "pages": 384, "dtype": "bf16", **large},
        # the pool of a small server, half of it in use, before its end is given back
        {"name": "compact_512", "kind": "compact", "layers": 30, "pages": 512, "used": 256, "seqs": 8, "page": 16,
         "dtype": "bf16", **small},
        # a large pool, three fifths of it in use by many sequences
        {"name": "compact_4096", "kind": "compact", "layers": 8, "pages": 4096, "used": 2458, "seqs": 100, "page": 16,
         "dtype": "bf16", **large},
        # the next token of one conversation, with the usual cuts
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 49152, "dtype": "fp32", "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "spread": 2.5},
        # a large batch whose rows each ask for something else: greedy, cut by number, by share, by both, or not at all
        {"name": "sample_256", "kind": "sample", "rows": 256, "vocab": 131072, "dtype": "bf16", "temperature": -1.0,
         "top_k": -1, "top_p": -1.0, "min_p": -1.0, "spread": 2.0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng)
        if all(work(case)[k] <= most[k] for k in most):
            return case


def _draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "fork", "compact", "sample", "sample"])
    if kind == "sample":
        mixed = rng.random() < 0.4
        return {"kind": kind, "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 1000, 260_000),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "spread": round(rng.uniform(0.5, 4.0), 2),
                "temperature": -1.0 if mixed else rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                "top_k": -1 if mixed else rng.choice([0, 0, 1, 40, 1000, 20_000]),
                "top_p": -1.0 if mixed else rng.choice([1.0, 1.0, 0.1, 0.9, 0.999]),
                "min_p": -1.0 if mixed else rng.choice([0.0, 0.0, 0.05, 0.001])}
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]),
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "attend":
        n = rng.choice([1, 1, 2, 8, 24, 64])
        most = (1_200_000 if heads < 32 else 300_000) // n
        case |= {"tokens": rng.choice([1, 1, 1, 2, 4, 7]),
                 "lens": ",".join(str(_log_int(rng, 1, most)) for _ in range(n))}
    elif kind == "write":
        seqs = rng.choice([1, 1, 2, 8, 32, 100])
        tokens = rng.choice([1, 4, _log_int(rng, 1, 100_000 // seqs)])
        case |= {"seqs": seqs, "tokens": tokens, "rows": tokens + rng.randint(0, 500)}
    else:
        # pools of at most 2 GB
        layers = rng.choice([1, 4, 12, 30])
        page_bytes = layers * 2 * kv_heads * case["page"] * dim * (4 if case["dtype"] == "fp32" else 2)
        pages = _log_int(rng, 40, max(40, min(20_000, 2_000_000_000 // page_bytes)))
        case |= {"layers": layers, "pages": pages}
        if kind == "fork":
            parents, forks = rng.randint(1, 8), rng.randint(1, 7)
            rows = _log_int(rng, 1, max(1, (pages // parents - 2 * forks - 1) * case["page"]))
            if pages < parents * ((rows + 1) // case["page"] + 1 + 2 * forks):
                parents, forks, rows = 1, 1, case["page"] + 3
            case |= {"parents": parents, "forks": forks, "rows": rows}
        else:
            used = rng.randint(pages // 5, pages - 1)
            case |= {"used": used, "seqs": rng.randint(1, min(100, used))}
    return case


def _lens(text):
    return [int(x) for x in text.split(",")]


# --------------------------------------------------------------------------- inputs

def _whole(values, dtype=torch.int64):
    return torch.tensor(values, device="cuda", dtype=dtype)


def _tables(counts, pages, gen):
    """Tables int32 [n, most + 2] of sequences that hold counts[b] pages each, scattered over the pool; -1 behind."""
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    starts = _whole([sum(counts[:b]) for b in range(len(counts))])
    at = torch.arange(max(counts) + 2, device="cuda")
    there = at < _whole(counts)[:, None]
    return torch.where(there, order[torch.where(there, starts[:, None] + at, 0)], -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)

    s = {"case": case}
    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        s |= {"logits": (torch.randn(B, V, device="cuda", generator=gen) * case["spread"]).to(dtype),
              "uniforms": torch.rand(B, device="cuda", generator=gen)}
        row = torch.arange(B, device="cuda")
        mixed = {"temperature": _whole([0.0, 0.6, 1.0, 0.9, 1.3], torch.float32)[row % 5],
                 "top_k": _whole([0, 40, 0, 50, 0, 5000, 1])[row % 7],
                 "top_p": _whole([1.0, 0.9, 0.95], torch.float32)[row % 3],
                 "min_p": _whole([0.0, 0.0, 0.0, 0.02], torch.float32)[row % 4]}
        return s | {k: mixed[k] if case[k] < 0 else case[k] for k in mixed}
    G, D, P = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "attend":
        lens = _lens(case["lens"])
        counts = [-(-n // P) for n in lens]
        pages = sum(counts) + 5
        return s | {"q": normal(len(lens), case["heads"], case["tokens"], D), "pool": normal(pages, 2, G, P, D),
                    "tables": _tables(counts, pages, gen), "lens": _whole(lens), "n_keys": max(lens),
                    "scaling": D ** -0.5}
    if case["kind"] == "write":
        n, T = case["seqs"], case["tokens"]
        counts = [-(-case["rows"] // P)] * n
        first = [(seed + 13 * b) % (case["rows"] - T + 1) for b in range(n)]
        return s | {"keys": normal(n, G, T, D), "values": normal(n, G, T, D), "first_rows": _whole(first),
                    "pool": torch.zeros(sum(counts) + 5, 2, G, P, D, device="cuda", dtype=dtype),
                    "tables": _tables(counts, sum(counts) + 5, gen)}
    s["pool"] = normal(case["layers"], case["pages"], 2, G, P, D)
    if case["kind"] == "fork":
        n, f = case["parents"], case["forks"]
        lens = [max(1, case["rows"] - 7 * b) for b in range(n)]
        tables = torch.full((n * (1 + f), -(-(case["rows"] + 1) // P) + 1), -1, device="cuda", dtype=torch.int32)
        held = _tables([-(-r // P) for r in lens], case["pages"], gen)[:, :tables.shape[1]]
        tables[:n, :held.shape[1]] = held
        sources = list(range(n)) + [b for b in range(n) for _ in range(f)]
        s |= {"lens": _whole(lens + [0] * (n * f)), "sources": _whole(sources), "counts": _whole([0] * n + [1] * (n * f))}
    else:
        n = case["seqs"]
        counts = [case["used"] * (b + 1) // n - case["used"] * b // n for b in range(n)]
        tables = _tables(counts, case["pages"], gen)
        s["lens"] = _whole([c * P for c in counts]) - _whole([(3 * b) % P for b in range(n)])
    s |= {"tables": tables.contiguous(), "refs": torch.zeros(case["pages"], device="cuda", dtype=torch.int32)}
    s["refs"].index_add_(0, tables.clamp_min(0).flatten().long(), (tables >= 0).int().flatten())
    return s


# --------------------------------------------------------------------------- the plain forms

def _attend(q, k, v, allowed, scaling):
    """softmax attention in fp32: q [n, H, Q, D] over k, v [n, G, N, D]; allowed [n, 1, Q, N]."""
    H, Q, D = q.shape[-3:]
    G = k.shape[-3]
    rows = q.float().reshape(q.shape[0], G, H // G * Q, D)
    s = torch.matmul(rows, k.transpose(-1, -2)).reshape(*q.shape[:-1], -1) * scaling
    s = s.masked_fill(~allowed, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z == 0, torch.ones_like(z), z)).reshape(q.shape[0], G, H // G * Q, -1)
    return torch.matmul(p, v).reshape(q.shape)


def _pages_of(lens, P):
    return (lens + P - 1) // P


def _count(refs, pages, by):
    """refs + by for every page of `pages` (of the same shape; by 0: nothing)."""
    refs.index_add_(0, pages.clamp_min(0).flatten().long(), by.int().flatten())


def _plain_fork(tables, lens, refs, sources, P):
    at, row = torch.arange(tables.shape[1], device="cuda"), torch.arange(tables.shape[0], device="cuda")
    moved = sources != row
    _count(refs, tables, -(moved[:, None] & (at < _pages_of(lens, P)[:, None])).int())
    new_lens = torch.where(moved, torch.where(sources >= 0, lens[sources.clamp_min(0)], 0), lens)
    there = at < _pages_of(new_lens, P)[:, None]
    new = torch.where(there, tables[sources.clamp_min(0)], -1)
    tables.copy_(torch.where(moved[:, None], new, tables))
    lens.copy_(new_lens)
    _count(refs, tables, moved[:, None] & there)


def _plain_reserve(tables, lens, refs, counts, P):
    at = torch.arange(tables.shape[1], device="cuda")
    old, new_lens = _pages_of(lens, P), lens + counts
    fits = (counts >= 0) & (new_lens <= tables.shape[1] * P)
    last = tables.gather(1, (lens // P).clamp_max(tables.shape[1] - 1)[:, None])[:, 0]
    shared = fits & (counts > 0) & (lens % P != 0) & (last >= 0) & (refs[last.clamp_min(0).long()] > 1)
    need = torch.where(fits, _pages_of(new_lens, P) - old + shared.long(), 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= (refs == 0).sum()))
    free = torch.argsort((refs != 0).int(), stable=True).int()
    begin = old - shared.long()
    taken = granted[:, None] & (at >= begin[:, None]) & (at < (begin + need)[:, None])
    slot = ((upto - need - begin)[:, None] + at).clamp(0, free.shape[0] - 1)
    parts = shared & granted
    src = torch.where(parts, last, -1)
    tables.copy_(torch.where(taken, free[slot], tables))
    dst = torch.where(parts, tables.gather(1, (lens // P).clamp_max(tables.shape[1] - 1)[:, None])[:, 0], -1)
    _count(refs, src, -parts.int())
    _count(refs, tables, taken)
    first = torch.where(granted, lens, -1)
    lens.copy_(torch.where(granted, new_lens, lens))
    return first, src, dst


def _plain_compact(tables, refs):
    n = refs.shape[0]
    at, used = torch.arange(n, device="cuda"), refs > 0
    count = used.sum()
    moved, hole = used & (at >= count), ~used & (at < count)
    holes = torch.argsort((~hole).int(), stable=True)
    to = torch.where(moved, holes[(moved.long().cumsum(0) - 1).clamp_min(0)], at)
    tables.copy_(torch.where(tables >= 0, to[tables.clamp_min(0).long()].int(), tables))
    refs.copy_(torch.zeros_like(refs).index_add_(0, to, torch.where(used, refs, 0)))
    there = at[:n // 2] < moved.sum()
    src = torch.where(there, torch.argsort((~moved).int(), stable=True)[:n // 2], -1).int()
    dst = torch.where(there, holes[:n // 2], -1).int()
    return src, dst, count.int()[None]


def _plain_copy(pool, src, dst):
    pairs = src >= 0
    pool[:, dst[pairs].long()] = pool[:, src[pairs].long()]


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    row = {k: (s[k] if torch.is_tensor(s[k]) else torch.full((B,), s[k], device="cuda", dtype=torch.float32)).double()[:, None]
           for k in ("temperature", "top_k", "top_p", "min_p")}
    value, token = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = row["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(row["temperature"]), row["temperature"])
    w = torch.exp((value - value[:, :1]) / t)
    rank = torch.arange(V, device="cuda")
    keep = (rank < row["top_k"]) | (row["top_k"] <= 0)
    w = torch.where(keep, w, 0.0)
    upto = w.cumsum(-1)
    keep &= (upto - w < row["top_p"] * upto[:, -1:]) | (row["top_p"] >= 1)
    keep &= w >= row["min_p"]
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, token, torch.where(keep, w, 0.0))
    upto = kept.cumsum(-1)
    there = torch.where(kept > 0, rank, 0).amax(-1)
    drawn = (upto <= s["uniforms"].double()[:, None] * upto[:, -1:]).sum(-1)
    return torch.where(greedy[:, 0], token[:, 0], torch.minimum(drawn, there))


def _plain(s):
    case = s["case"]
    if case["kind"] == "sample":
        return _plain_sample(s)
    P = case["page"]
    if case["kind"] == "attend":
        at = torch.arange(s["n_keys"], device="cuda")
        there = at < s["lens"][:, None]
        pages = torch.where(there, s["tables"].long()[:, at // P], 0)
        kv = s["pool"][pages, :, :, at % P].float()  # [n, N, 2, G, D]
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        last = torch.arange(case["tokens"], device="cuda") + (s["lens"] - case["tokens"])[:, None]
        allowed = (at <= last[..., None]) & there[:, None]
        return _attend(s["q"], k, v, allowed[:, None], s["scaling"]).to(s["q"].dtype)
    if case["kind"] == "write":
        at = s["first_rows"][:, None] + torch.arange(case["tokens"], device="cuda")
        pages = s["tables"].gather(1, at // P).long()
        s["pool"][pages, :, :, at % P] = torch.stack([s["keys"], s["values"]], 1).permute(0, 3, 1, 2, 4)
        return s["pool"]
    if case["kind"] == "fork":
        _plain_fork(s["tables"], s["lens"], s["refs"], s["sources"], P)
        first, src, dst = _plain_reserve(s["tables"], s["lens"], s["refs"], s["counts"], P)
        _plain_copy(s["pool"], src, dst)
        return {"tables": s["tables"], "lens": s["lens"], "refs": s["refs"], "first_rows": first, "src": src, "dst": dst,
                "pool": s["pool"]}
    tables, refs = s["tables"].clone(), s["refs"].clone()  # (the program keeps the old ones until the copies are done)
    src, dst, used = _plain_compact(tables, refs)
    _plain_copy(s["pool"], src, dst)
    return {"tables": tables, "refs": refs, "src": src, "dst": dst, "used": used, "pool": s["pool"]}


def _own(s):
    from sva_amd import kernels

    case = s["case"]
    if case["kind"] == "sample":
        return kernels.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"])
    if case["kind"] == "attend":
        return kernels.paged_attention(s["q"], s["pool"], s["tables"], s["lens"], s["scaling"], n_keys=s["n_keys"])
    if case["kind"] == "write":
        kernels.paged_write(s["keys"], s["values"], s["pool"], s["tables"], s["first_rows"])
        return s["pool"]
    if case["kind"] == "fork":
        kernels.pages_fork(s["tables"], s["lens"], s["refs"], s["sources"], case["page"])
        first, src, dst = kernels.pages_reserve(s["tables"], s["lens"], s["refs"], s["counts"], case["page"])
        kernels.pages_copy(s["pool"], src, dst)
        return {"tables": s["tables"], "lens": s["lens"], "refs": s["refs"], "first_rows": first, "src": src, "dst": dst,
                "pool": s["pool"]}
    tables, refs = s["tables"].clone(), s["refs"].clone()
    src, dst, used = kernels.pages_compact(tables, refs)
    kernels.pages_copy(s["pool"], src, dst)
    return {"tables": tables, "refs": refs, "src": src, "dst": dst, "used": used, "pool": s["pool"]}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + 12 * case["rows"], "flops": 2 * n}
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    row = 2 * G * D * e  # K and V of a row
    if case["kind"] == "attend":
        lens, T = _lens(case["lens"]), case["tokens"]
        pairs = sum(max(0, k - T + 1 + t) for k in lens for t in range(T))
        return {"bytes": 2 * e * D * H * T * len(lens) + sum(lens) * row + 4 * sum(-(-k // P) for k in lens),
                "flops": 4 * D * H * pairs}
    if case["kind"] == "write":
        return {"bytes": 2 * case["seqs"] * case["tokens"] * row, "flops": 0}
    page = case["layers"] * P * row
    if case["kind"] == "fork":
        lens = [max(1, case["rows"] - 7 * b) for b in range(case["parents"])]
        parted = case["forks"] * sum(n % P != 0 for n in lens)
        return {"bytes": 2 * parted * page + 4 * (1 + 2 * case["forks"]) * sum(-(-n // P) for n in lens) + 4 * case["pages"],
                "flops": 0}
    moved = case["used"] * (case["pages"] - case["used"]) // case["pages"]  # as many as lie behind the others on average
    return {"bytes": 2 * moved * page + 8 * case["pages"] + 8 * case["used"], "flops": 0}


# --------------------------------------------------------------------------- the definition in 64 bits

def _fork_by_hand(s, P):
    """Tables, lengths, counts, first rows and pairs of the fork case, sequence by sequence."""
    tables, lens, refs, sources, counts = (s[k].cpu().tolist() for k in ("tables", "lens", "refs", "sources", "counts"))
    held = [t[:-(-n // P)] for t, n in zip(tables, lens)]
    before = [list(h) for h in held], list(lens)
    for i, src in enumerate(sources):
        if src == i:
            continue
        for p in held[i]:
            refs[p] -= 1
        held[i], lens[i] = (list(before[0][src]), before[1][src]) if src >= 0 else ([], 0)
        for p in held[i]:
            refs[p] += 1
    free = [p for p, r in enumerate(refs) if r == 0]
    shares = [r > 1 for r in refs]
    first, pairs, gone = [], [], []
    for i, c in enumerate(counts):
        first.append(lens[i])
        pairs.append((-1, -1))
        if c and lens[i] % P and shares[held[i][-1]]:
            pairs[-1] = (held[i][-1], free[0])
            gone.append(held[i][-1])
            held[i][-1] = free.pop(0)
            refs[held[i][-1]] = 1
        lens[i] += c
        while len(held[i]) * P < lens[i]:
            held[i].append(free.pop(0))
            refs[held[i][-1]] = 1
    for p in gone:
        refs[p] -= 1
    width = len(tables[0])
    return [h + [-1] * (width - len(h)) for h in held], lens, refs, first, pairs


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        out = []
        for b in range(case["rows"]):
            T, k, p, m = (float(s[n][b] if torch.is_tensor(s[n]) else torch.tensor(float(s[n])))  # (fp32, as given)
                          for n in ("temperature", "top_k", "top_p", "min_p"))
            x = s["logits"][b].double()
            if T <= 0:
                out.append(int((x == x.max()).nonzero()[0]))
                continue
            w = torch.exp((x - x.max()) / T)
            order = torch.argsort(x, descending=True, stable=True)[:int(k) if k > 0 else None]
            if p < 1:
                share = torch.cumsum(w[order], 0)
                order = order[:int((share < p * share[-1]).sum()) + 1]
            order = order[w[order] >= m].sort().values
            share = torch.cumsum(w[order], 0)
            at = int(torch.searchsorted(share, float(s["uniforms"][b]) * share[-1:], right=True))
            out.append(int(order[min(at, len(order) - 1)]))
        return _whole(out)
    P = case["page"]
    if case["kind"] == "attend":
        q, T = s["q"].double(), case["tokens"]
        out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
        grp = case["heads"] // case["kv_heads"]
        for b, n in enumerate(_lens(case["lens"])):
            pages = s["tables"][b, :-(-n // P)].long()
            for g in range(case["kv_heads"]):
                K, V = (s["pool"][pages, i, g].double().flatten(0, 1)[:n] for i in (0, 1))
                for t in range(T):
                    end = n - T + 1 + t
                    if end > 0:
                        w = torch.softmax(q[b, g * grp:(g + 1) * grp, t] @ K[:end].T * s["scaling"], -1)
                        out[b, g * grp:(g + 1) * grp, t] = w @ V[:end]
        return out
    if case["kind"] == "write":
        pool = s["pool"].double()
        for b, first in enumerate(s["first_rows"].tolist()):
            for page in range(first // P, (first + case["tokens"] - 1) // P + 1):
                a, z = max(first, page * P), min(first + case["tokens"], (page + 1) * P)
                to = pool[int(s["tables"][b, page])]
                to[0, :, a - page * P:z - page * P] = s["keys"][b, :, a - first:z - first].double()
                to[1, :, a - page * P:z - page * P] = s["values"][b, :, a - first:z - first].double()
        return pool
    if case["kind"] == "fork":
        tables, lens, refs, first, pairs = _fork_by_hand(s, P)
        src, dst = zip(*pairs)
        out = {"tables": _whole(tables, torch.int32), "lens": _whole(lens), "refs": _whole(refs, torch.int32),
               "first_rows": _whole(first), "src": _whole(src, torch.int32), "dst": _whole(dst, torch.int32)}
    else:
        refs = s["refs"].tolist()
        used = sum(r > 0 for r in refs)
        pairs = list(zip([p for p in range(used, len(refs)) if refs[p] > 0], [p for p in range(used) if refs[p] == 0]))
        to = dict(pairs)
        for a, b in pairs:
            refs[a], refs[b] = 0, refs[a]
        tables = [[to.get(p, p) for p in t] for t in s["tables"].tolist()]
        src, dst = zip(*(pairs + [(-1, -1)] * (len(refs) // 2 - len(pairs))))
        out = {"tables": _whole(tables, torch.int32), "refs": _whole(refs, torch.int32), "src": _whole(src, torch.int32),
               "dst": _whole(dst, torch.int32), "used": _whole([used], torch.int32)}
    out["pool"] = s["pool"].double()
    for a, b in pairs:
        if a >= 0:
            out["pool"][:, b] = s["pool"][:, a].double()
    return out
