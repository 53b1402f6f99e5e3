"""Attention over whole prompts and over a cache held in 4 bits, as timed cases.

A case is one public call (for the cache's write: the write and the read of
the written rows) at one size: a prompt's dense attention, packed prompts of
different lengths with and without cached prefixes, a chunk of a prompt over
a long cache, one token over long caches, the write of a prompt's or a
token's rows into the 4-bit cache, attention of a few tokens over all of it,
and the exact verifier over chosen rows of it.  ``listed`` holds sizes of
this repository's tests and benchmark; ``draw`` gives others of the same
ranges.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
by the framework's kernels.

The 4-bit format: 32 consecutive elements of a K or V row share a scale 2^e,
e = floor(log2(largest magnitude)) - 2, kept as the byte e + 127 (at least 1);
an element is the sign and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the
scale (ties to the even code).  Row r of KV head g holds its K half, then its
V half: data [G, rows, 2, D / 2] (two codes a byte, the first in the low bits)
and scales [G, rows, 2, D / 32].
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
    # 32 sequences of 4K to 131K keys, as a packed server batch holds them
    ragged = ",".join(str(4096 + (131072 - 4096) * i // 31 - (i * 37) % 64) for i in range(32))
    return [
        # a whole prompt through one layer of the small model
        {"name": "prompt_8k", "kind": "prompt", "q_lens": "8192", "k_lens": "8192", "dtype": "bf16", **small},
        # prompts of a server's batch, packed without padding: one of one token, odd ones, two that go on after a
        # cached prefix
        {"name": "prompt_packed", "kind": "prompt", "q_lens": "1,17,333,1024,2047,2500,4096,777",
         "k_lens": "1,17,333,1024,2047,3524,4096,2777", "dtype": "bf16", **large},
        # an odd prompt of a model kept in fp32
        {"name": "prompt_fp32", "kind": "prompt", "q_lens": "1001", "k_lens": "1001", "dtype": "fp32", "heads": 12,
         "kv_heads": 4, "dim": 64},
        # the next chunk of eight long prompts, over what is cached of each
        {"name": "prompt_chunk_32k", "kind": "prompt", "q_lens": ",".join(["512"] * 8),
         "k_lens": ",".join(["32768"] * 8), "dtype": "fp16", **small},
        # one token of each of 32 sequences over all of its keys
        {"name": "token_ragged", "kind": "prompt", "q_lens": ",".join(["1"] * 32), "k_lens": ragged, "dtype": "bf16",
         **small},
        # a decode step's new rows of a batch: the smallest call
        {"name": "append_8", "kind": "write", "seqs": 8, "tokens": 1, "rows": 32768, "dtype": "bf16", **small},
        # a long prompt's rows
        {"name": "write_131k", "kind": "write", "seqs": 1, "tokens": 131072, "rows": 131072, "dtype": "bf16",
         **large},
        # one token over a million keys in 4 bits
        {"name": "attend_1m", "kind": "attend", "tokens": 1, "k_lens": "1048576", "dtype": "bf16", **small},
        # a decode step of a packed batch of the wide model; the largest cache
        {"name": "attend_ragged", "kind": "attend", "tokens": 1,
         "k_lens": ",".join(str(1024 + 1777 * i) for i in range(24)), "dtype": "bf16", **large},
        # drafted tokens being checked against one short cache
        {"name": "attend_4_8k", "kind": "attend", "tokens": 4, "k_lens": "8192", "dtype": "fp16", **small},
        # the verifier of a decode lookup over a million keys
        {"name": "verify_1m", "kind": "verify", "tokens": 1, "k_lens": "1048576", "budget": 512, "dtype": "bf16",
         **small},
        # the verifier of the late-layer socket's batch
        {"name": "verify_8_32k", "kind": "verify", "tokens": 1, "k_lens": ",".join(["32768"] * 8), "budget": 2048,
         "dtype": "bf16", **small},
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
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": rng.choice(["prompt", "prompt", "prompt", "write", "attend", "attend", "verify"]),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if case["kind"] == "prompt":
        form = rng.choice(["whole", "packed", "chunk", "token"])
        n = {"whole": 1, "packed": rng.randint(2, 8), "chunk": rng.randint(1, 8), "token": rng.randint(1, 32)}[form]
        if form == "token":
            k_lens = [_log_int(rng, 1, 100_000) for _ in range(n)]
            q_lens = [1] * n
        elif form == "chunk":
            k_lens = [_log_int(rng, 512, 20_000) for _ in range(n)]
            q_lens = [min(k, _log_int(rng, 2, 512)) for k in k_lens]
        else:
            q_lens = [_log_int(rng, 1, 7000 if form == "whole" and heads < 32 else 3000) for _ in range(n)]
            k_lens = [q + rng.choice([0, 0, 0, rng.randint(1, 1000)]) for q in q_lens]
        case |= {"q_lens": ",".join(map(str, q_lens)), "k_lens": ",".join(map(str, k_lens))}
    elif case["kind"] == "write":
        seqs = rng.choice([1, 1, 2, 8, 32])
        tokens = rng.choice([1, 4, _log_int(rng, 1, 100_000 // seqs)])
        case |= {"seqs": seqs, "tokens": tokens, "rows": tokens + rng.randint(0, 500)}
    else:
        n = rng.choice([1, 1, 2, 8, 24])
        most = 900_000 // n if heads < 32 else 300_000 // n
        k_lens = [_log_int(rng, 1, most) for _ in range(n)]
        case |= {"tokens": rng.choice([1, 1, 1, 2, 4, 7]), "k_lens": ",".join(map(str, k_lens))}
        if case["kind"] == "verify":
            case["budget"] = rng.choice([64, 128, 512, 1000, 2048])
    return case


def _lens(text):
    return [int(x) for x in text.split(",")]


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# --------------------------------------------------------------------------- the 4-bit format, plainly

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _scale(byte):
    """2^(byte - 127) in fp32 (NaN for 255)."""
    scale = (byte.int() << 23).view(torch.float32)
    return torch.where(byte == 255, torch.full_like(scale, float("nan")), scale)


def _to_4_bits(x):
    """(codes, scale bytes) of the rows x [..., D]: uint8 [..., D / 2] and [..., D / 32]."""
    x = x.float()
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = blocks.abs().amax(-1)
    _, exponent = torch.frexp(amax)  # amax = m 2^exponent, 0.5 <= m < 1
    byte = torch.where(amax > 0, exponent - 3 + 127, torch.ones_like(exponent)).clamp(1, 254)
    byte = torch.where(torch.isfinite(amax), byte, torch.full_like(byte, 255))
    a = blocks.abs() / _scale(byte)[..., None]  # exact: a power of two
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(blocks)).to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), byte.to(torch.uint8)


def _from_4_bits(codes, scales):
    """fp32 rows [..., D] of codes [..., D / 2] and scale bytes [..., D / 32]."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    values = table[nibbles.long()]
    return (values.unflatten(-1, (-1, 32)) * _scale(scales)[..., None]).flatten(-2)


# --------------------------------------------------------------------------- inputs

def _cache(case, rows, gen):
    """A 4-bit cache of K and V rows drawn from normal values, made a head at a time."""
    data = torch.empty(case["kv_heads"], rows, 2, case["dim"] // 2, device="cuda", dtype=torch.uint8)
    scales = torch.empty(case["kv_heads"], rows, 2, case["dim"] // 32, device="cuda", dtype=torch.uint8)
    for g in range(case["kv_heads"]):
        for a in range(0, rows, 1 << 18):
            b = min(rows, a + (1 << 18))
            kv = torch.randn(b - a, 2, case["dim"], device="cuda", generator=gen)
            data[g, a:b], scales[g, a:b] = _to_4_bits(kv)
    return data, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    def whole(values):
        return torch.tensor(values, device="cuda", dtype=torch.int64)

    s = {"case": case, "scaling": D ** -0.5}
    if case["kind"] == "write":
        n, T = case["seqs"], case["tokens"]
        first = [b * case["rows"] + (seed + 13 * b) % (case["rows"] - T + 1) for b in range(n)]
        s |= {"keys": normal(n, G, T, D), "values": normal(n, G, T, D), "first_rows": whole(first),
              "data": torch.zeros(G, n * case["rows"], 2, D // 2, device="cuda", dtype=torch.uint8),
              "scales": torch.zeros(G, n * case["rows"], 2, D // 32, device="cuda", dtype=torch.uint8)}
        return s
    k_lens = _lens(case["k_lens"])
    n, rows = len(k_lens), sum(k_lens)
    s |= {"n": n, "n_keys": max(k_lens), "seq_lens": whole(k_lens), "seq_offsets": whole(_starts(k_lens)[:-1])}
    if case["kind"] == "prompt":
        q_lens = _lens(case["q_lens"])
        s |= {"q": normal(H, sum(q_lens), D), "keys": normal(G, rows, D), "values": normal(G, rows, D),
              "q_lens": whole(q_lens), "q_offsets": whole(_starts(q_lens)[:-1]), "max_q": max(q_lens)}
        return s
    s["q"] = normal(n, H, case["tokens"], D)
    s["data"], s["scales"] = _cache(case, rows, gen)
    if case["kind"] == "verify":
        # each item's budget list: distinct rows of its sequence, ascending, -1 behind the last
        B, T = case["budget"], case["tokens"]
        idx = torch.full((n * H * T, B), -1, device="cuda", dtype=torch.int32)
        for b, length in enumerate(k_lens):
            m = min(B, length)
            at = torch.arange(m, device="cuda") * length // m
            width = (torch.arange(1, m + 1, device="cuda") * length // m) - at
            pick = at + (torch.rand(H * T, m, device="cuda", generator=gen) * width).long().clamp_max(width - 1)
            idx[b * H * T:(b + 1) * H * T, :m] = pick.int()
        counts = torch.tensor(k_lens, device="cuda").clamp_max(B).repeat_interleave(H * T)
        s |= {"fin_idx": idx, "fin_count": counts.int()}
    return s


# --------------------------------------------------------------------------- the plain forms

def _attend(q, k, v, allowed, scaling):
    """softmax attention in fp32: q [..., H, Q, D] over k, v [..., G, N, D]; allowed [..., 1, Q, N]."""
    H, Q, D = q.shape[-3:]
    G = k.shape[-3]
    rows = q.float().reshape(*q.shape[:-3], G, H // G * Q, D)
    s = torch.matmul(rows, k.transpose(-1, -2)).reshape(*q.shape[:-1], -1) * scaling
    s = s.masked_fill(~allowed, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z == 0, torch.ones_like(z), z)).reshape(*q.shape[:-3], G, H // G * Q, -1)
    return torch.matmul(p, v).reshape(q.shape)


def _padded(offsets, lens, most):
    """Row numbers [n, most] of packed sequences, and which of them are there."""
    at = torch.arange(most, device=lens.device)
    there = at < lens[:, None]
    return torch.where(there, offsets[:, None] + at, torch.zeros_like(offsets)[:, None]), there


def _plain(s):
    case = s["case"]
    if case["kind"] == "write":
        T = case["tokens"]
        at = (s["first_rows"][:, None] + torch.arange(T, device="cuda")).flatten()
        kv = torch.stack([s["keys"], s["values"]], 3).transpose(0, 1).flatten(1, 2)  # [G, n T, 2, D]
        s["data"][:, at], s["scales"][:, at] = _to_4_bits(kv)
        back = _from_4_bits(s["data"][:, at], s["scales"][:, at]).to(s["keys"].dtype)
        back = back.unflatten(1, (-1, T)).transpose(0, 1)
        return {"keys": back[..., 0, :], "values": back[..., 1, :]}
    k_at, k_there = _padded(s["seq_offsets"], s["seq_lens"], s["n_keys"])
    if case["kind"] == "prompt":
        q_at, q_there = _padded(s["q_offsets"], s["q_lens"], s["max_q"])
        q = s["q"][:, q_at].transpose(0, 1)  # [n, H, max_q, D]
        k = s["keys"].float()[:, k_at].transpose(0, 1)
        v = s["values"].float()[:, k_at].transpose(0, 1)
        last = torch.arange(s["max_q"], device="cuda") + (s["seq_lens"] - s["q_lens"])[:, None]
        allowed = (torch.arange(s["n_keys"], device="cuda") <= last[..., None]) & k_there[:, None]
        out = _attend(q, k, v, allowed[:, None], s["scaling"])
        return out.transpose(1, 2)[q_there].transpose(0, 1).to(s["q"].dtype)
    if case["kind"] == "attend":
        T = case["tokens"]
        kv = _from_4_bits(s["data"], s["scales"])[:, k_at].transpose(0, 1)  # [n, G, N, 2, D]
        last = torch.arange(T, device="cuda") + (s["seq_lens"] - T)[:, None]
        allowed = (torch.arange(s["n_keys"], device="cuda") <= last[..., None]) & k_there[:, None]
        return _attend(s["q"], kv[..., 0, :], kv[..., 1, :], allowed[:, None], s["scaling"]).to(s["q"].dtype)
    n, H, T, D = s["q"].shape
    there = torch.arange(case["budget"], device="cuda") < s["fin_count"][:, None]
    local = torch.where(there, s["fin_idx"], torch.zeros_like(s["fin_idx"]))
    at = s["seq_offsets"].repeat_interleave(H * T)[:, None] + local
    g = (torch.arange(H, device="cuda") // (H // case["kv_heads"])).repeat_interleave(T).repeat(n)[:, None]
    kv = _from_4_bits(s["data"][g, at], s["scales"][g, at])  # [n H T, B, 2, D]
    out = _attend(s["q"].reshape(-1, 1, 1, D), kv[:, None, :, 0], kv[:, None, :, 1], there[:, None, None], s["scaling"])
    return out.reshape(s["q"].shape).to(s["q"].dtype)


def _own(s):
    from sva_amd import kernels

    case = s["case"]
    if case["kind"] == "write":
        kernels.cache4_write(s["keys"], s["values"], s["data"], s["scales"], s["first_rows"])
        keys, values = kernels.cache4_read(s["data"], s["scales"], s["first_rows"], case["tokens"], s["keys"].dtype)
        return {"keys": keys, "values": values}
    where = {"seq_offsets": s["seq_offsets"], "seq_lens": s["seq_lens"]}
    if case["kind"] == "prompt":
        return kernels.prompt_attention(s["q"], s["keys"], s["values"], s["n_keys"], s["scaling"],
                                        q_offsets=s["q_offsets"], q_lens=s["q_lens"], max_q=s["max_q"], **where)
    if case["kind"] == "attend":
        return kernels.cache4_attention(s["q"], s["data"], s["scales"], s["n_keys"], s["scaling"], **where)
    return kernels.cache4_verify(s["q"], s["data"], s["scales"], s["fin_idx"], s["fin_count"], s["n_keys"],
                                 s["scaling"], **where)


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    e = 4 if case["dtype"] == "fp32" else 2
    row4 = D + D // 16  # K and V codes and scales of a row
    if case["kind"] == "write":
        rows = case["seqs"] * case["tokens"] * G
        return {"bytes": rows * (2 * (2 * D * e) + 2 * row4), "flops": 0}
    k_lens = _lens(case["k_lens"])
    if case["kind"] == "prompt":
        q_lens = _lens(case["q_lens"])
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(q_lens, k_lens))
        return {"bytes": e * D * (2 * H * sum(q_lens) + 2 * G * sum(k_lens)), "flops": 4 * D * H * pairs}
    T = case["tokens"]
    out = 2 * e * D * H * T * len(k_lens)
    if case["kind"] == "attend":
        pairs = sum(max(0, k - T + 1 + t) for k in k_lens for t in range(T))
        return {"bytes": out + G * sum(k_lens) * row4, "flops": 4 * D * H * pairs}
    chosen = [min(case["budget"], k) for k in k_lens]
    lists = H // G * T
    rows = sum(k * (1 - (1 - m / k) ** lists) for m, k in zip(chosen, k_lens))  # rows that any list of a group holds
    return {"bytes": int(out + G * rows * row4 + 4 * H * T * sum(chosen)), "flops": 4 * D * H * T * sum(chosen)}


# --------------------------------------------------------------------------- the definition in 64 bits

def _value64(data, scales):
    """Rows in 64 bits, code by code: sign, then 0 and 0.5 below code 2, 2^(c / 2 - 1) and half as much again above."""
    c = torch.stack([data.long() % 16, data.long() // 16], -1).flatten(-2)
    m = c % 8
    low = m.double() / 2
    high = torch.exp2((m // 2 - 1).double()) * (1 + (m % 2).double() / 2)
    size = torch.where(m < 2, low, high) * torch.where(c < 8, 1.0, -1.0).double()
    e = torch.exp2(scales.double() - 127)
    return (size.unflatten(-1, (-1, 32)) * e[..., None]).flatten(-2)


def _round64(x):
    """The nearest values of the format to x [..., D], in 64 bits."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -124))) - 2)
    a = (x / e).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    near = (torch.round(a / step) * step).clamp_max(6)  # round: ties to even
    return (near * torch.sign(x) * e).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    H, G = case["heads"], case["kv_heads"]
    if case["kind"] == "write":
        return {"keys": _round64(s["keys"]), "values": _round64(s["values"])}
    k_lens = _lens(case["k_lens"])
    starts = _starts(k_lens)
    if case["kind"] == "prompt":
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        q_lens = _lens(case["q_lens"])
        for h in range(H):
            for k0, N, q0, Q in zip(starts, k_lens, _starts(q_lens), q_lens):
                K, V = (s[x][h // (H // G), k0:k0 + N].double() for x in ("keys", "values"))
                w = s["q"][h, q0:q0 + Q].double() @ K.T * s["scaling"]
                w = w + torch.full_like(w, float("-inf")).triu(N - Q + 1)
                out[h, q0:q0 + Q] = torch.softmax(w, -1) @ V
        return out
    n, _, T, D = s["q"].shape
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b in range(n):
        for g in range(G):
            rows = slice(starts[b], starts[b + 1])
            kv = None
            if case["kind"] == "attend":
                kv = _value64(s["data"][g, rows], s["scales"][g, rows])
            for h in range(g * (H // G), (g + 1) * (H // G)):
                for t in range(T):
                    q = s["q"][b, h, t].double()
                    if case["kind"] == "attend":
                        end = k_lens[b] - T + 1 + t
                        if end <= 0:
                            continue
                        K, V = kv[:end, 0], kv[:end, 1]
                    else:
                        i = (b * H + h) * T + t
                        at = s["fin_idx"][i, :min(case["budget"], k_lens[b])].long() + starts[b]
                        K, V = _value64(s["data"][g, at], s["scales"][g, at]).unbind(1)
                    out[b, h, t] = torch.softmax(K @ q * s["scaling"], 0) @ V
    return out
