"""Dense prompt attention on the GPU against softmax attention in 64 bits: whole, packed and ragged prompts, chunks
over cached prefixes, single tokens, explicit masks, values that are not finite where they are masked."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .cache4_reference import attend

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# weights are rounded to the inputs' type for the second product (fp32: not), each within half a step, and a weight
# under fp16's normal range (2^-14 of a maximum kept at 2^8) within 2^-25 of 2^8
WEIGHTS = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def normal(rng, shape, dtype, device):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(device, dtype)


def check(got, q, keys, values, allowed, scaling):
    """got / q [R, D] of one head over its keys / values [N, D], allowed [R, N]."""
    K, V, x = (t.double().cpu().numpy() for t in (keys, values, q))
    ref, bound = attend(x, K, V, allowed, scaling)
    size, _ = attend(x, K, np.abs(V), allowed, scaling)
    g = got.double().cpu().numpy()
    extra = WEIGHTS[q.dtype] * size + (2.0 ** -33 * len(K) * np.abs(V).max() if q.dtype == torch.float16 and len(K)
                                       else 0.0)
    over = np.abs(g - ref) - bound - extra - HALF_STEP[got.dtype] * np.abs(ref)
    assert (over <= 1e-30).all(), f"over the bound by {np.nanmax(over)}"


def causal(q_len, n):
    return np.arange(n) <= n - q_len + np.arange(q_len)[:, None]


@pytest.mark.parametrize("n,Q,H,G,D,dtype", [
    (1, 1, 1, 1, 64, torch.float32), (1, 1, 3, 1, 64, torch.bfloat16), (31, 31, 2, 2, 64, torch.float16),
    (65, 65, 9, 3, 64, torch.bfloat16), (300, 300, 9, 3, 64, torch.float32), (257, 257, 8, 1, 128, torch.bfloat16),
    (130, 130, 4, 4, 128, torch.float16), (100, 100, 4, 2, 128, torch.float32), (140, 140, 2, 1, 256, torch.bfloat16),
    (90, 90, 2, 1, 256, torch.float32), (77, 77, 2, 1, 256, torch.float16), (200, 200, 4, 2, 8, torch.float32),
    (70, 70, 3, 1, 80, torch.bfloat16), (70, 70, 3, 1, 17, torch.float16), (66, 66, 2, 1, 200, torch.float32),
    (1000, 70, 9, 3, 64, torch.bfloat16), (2500, 33, 4, 1, 128, torch.float16), (3000, 1, 9, 3, 64, torch.bfloat16),
    (5000, 1, 4, 2, 128, torch.float32), (2000, 2, 64, 2, 64, torch.float16), (5, 9, 2, 1, 64, torch.float32)])
def test_one_sequence(device, n, Q, H, G, D, dtype):
    from sva_amd import kernels

    rng = np.random.default_rng(n + Q + D)
    q, k, v = (normal(rng, s, dtype, device) for s in ((1, H, Q, D), (G, n, D), (G, n, D)))
    for out_dtype in {dtype, torch.float32}:
        got = kernels.prompt_attention(q, k, v, n, D ** -0.5, out_dtype=out_dtype)
        assert got.shape == q.shape and got.dtype == out_dtype
        for h in range(H):
            check(got[0, h], q[0, h], k[h // (H // G)], v[h // (H // G)], causal(Q, n), D ** -0.5)


@pytest.mark.parametrize("q_lens,k_lens,H,G,D,dtype", [
    ([1, 17, 200, 64], [1, 17, 200, 64], 9, 3, 64, torch.bfloat16), ([5, 0, 130], [400, 9, 131], 4, 2, 128, torch.float16),
    ([1, 1, 1], [700, 1, 2000], 9, 3, 64, torch.bfloat16), ([3, 40], [2, 0], 2, 1, 64, torch.float32),
    ([33, 1], [33, 1500], 8, 8, 64, torch.float32)])
def test_packed(device, q_lens, k_lens, H, G, D, dtype):
    """Packed tokens, gaps between sequences: rows of no sequence stay as they were."""
    from sva_amd import kernels

    rng = np.random.default_rng(sum(k_lens))
    q_at = np.concatenate([[0], np.cumsum([n + 2 for n in q_lens])])[:-1] + 1
    k_at = np.concatenate([[0], np.cumsum([n + 3 for n in k_lens])])[:-1]
    T, rows = int(q_at[-1]) + q_lens[-1] + 4, int(k_at[-1]) + k_lens[-1] + 1
    q, k, v = (normal(rng, s, dtype, device) for s in ((H, T, D), (G, rows, D), (G, rows, D)))
    for b, n in enumerate(k_lens):  # what lies between the sequences is never used
        k[:, k_at[b] + n:k_at[b] + n + 1] = float("nan")
        v[:, k_at[b] + n:k_at[b] + n + 1] = float("inf")
    dev = lambda x: torch.tensor(list(x), device=device)  # noqa: E731
    out = torch.full((H, T, D), 7.0, device=device, dtype=dtype)
    got = kernels.prompt_attention(q, k, v, max(k_lens), D ** -0.5, seq_offsets=dev(k_at), seq_lens=dev(k_lens),
                                   q_offsets=dev(q_at), q_lens=dev(q_lens), max_q=max(q_lens) + 5, out=out)
    assert got is out
    inside = np.zeros(T, bool)
    for b in range(len(q_lens)):
        t, n = slice(q_at[b], q_at[b] + q_lens[b]), slice(k_at[b], k_at[b] + k_lens[b])
        inside[t] = True
        for h in range(H):
            g = h // (H // G)
            check(got[h, t], q[h, t], k[g, n], v[g, n], causal(q_lens[b], k_lens[b]), D ** -0.5)
    assert (got[:, torch.from_numpy(~inside).to(device)] == 7).all()


def test_batch_with_ragged_lengths(device):
    from sva_amd import kernels

    rng = np.random.default_rng(8)
    lens, H, G, Q, D = [90, 40, 33], 6, 2, 33, 64
    q, k, v = (normal(rng, s, torch.bfloat16, device) for s in ((3, H, Q, D), (G, 300, D), (G, 300, D)))
    off, ln = torch.tensor([0, 100, 200], device=device), torch.tensor(lens, device=device)
    got = kernels.prompt_attention(q, k, v, 90, 0.2, seq_offsets=off, seq_lens=ln)
    for b in range(3):
        for h in range(H):
            n = slice(100 * b, 100 * b + lens[b])
            check(got[b, h], q[b, h], k[h // 3, n], v[h // 3, n], causal(Q, lens[b]), 0.2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["bool", "float32", "dtype"])
def test_masks(device, dtype, kind):
    """Random, empty and left-padded rows; the type's lowest value, -inf and NaN mask; other values are not added."""
    from sva_amd import kernels

    rng = np.random.default_rng(5)
    n_seq, H, G, Q, N, D = 2, 4, 2, 70, 130, 64
    q, k, v = (normal(rng, s, dtype, device) for s in ((n_seq, H, Q, D), (G, n_seq * N, D), (G, n_seq * N, D)))
    allowed = rng.random((n_seq, Q, N)) < 0.3
    allowed[0, 5] = False
    allowed[1, :, :40] = False
    allowed[1, 6] = True
    if kind == "bool":
        mask = torch.from_numpy(allowed).to(device)[:, None]
    else:
        mt = torch.float32 if kind == "float32" else dtype
        low = torch.tensor([torch.finfo(mt).min, float("-inf"), float("nan")])[rng.integers(0, 3, allowed.shape)]
        high = torch.tensor([0.0, 1.0, -3.0])[rng.integers(0, 3, allowed.shape)]
        mask = torch.where(torch.from_numpy(allowed), high, low).to(device, mt)[:, None]
    off, ln = torch.tensor([0, N], device=device), torch.tensor([N, N], device=device)
    got = kernels.prompt_attention(q, k, v, N, 0.125, mask=mask, seq_offsets=off, seq_lens=ln)
    for b in range(n_seq):
        for h in range(H):
            at = slice(b * N, (b + 1) * N)
            check(got[b, h], q[b, h], k[h // 2, at], v[h // 2, at], allowed[b], 0.125)
    assert (got[0, :, 5] == 0).all()
    one = kernels.prompt_attention(q, k, v, N, 0.125, mask=mask[:1], seq_offsets=off, seq_lens=ln)
    assert torch.equal(one[0], got[0])
    wide = torch.cat([mask, mask], -1)  # a mask of a longer cache, not contiguous
    assert torch.equal(kernels.prompt_attention(q, k, v, N, 0.125, mask=wide, seq_offsets=off, seq_lens=ln), got)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("n,Q", [(200, 200), (1500, 3)])
def test_values_not_finite(device, dtype, D, n, Q):
    """NaN and infinities in K and V reach the tokens that see them, and no others."""
    from sva_amd import kernels

    rng = np.random.default_rng(n)
    q, k, v = (normal(rng, s, dtype, device) for s in ((1, 2, Q, D), (1, n, D), (1, n, D)))
    clean = kernels.prompt_attention(q, k, v, n, 0.125).float()
    at = n - 2  # the last two tokens see it
    v[0, at, 3], v[0, at, 5], v[0, n - 1, 5] = float("nan"), float("inf"), float("-inf")
    got = kernels.prompt_attention(q, k, v, n, 0.125).float()
    # rows done again keep their weights in fp32: each weight of the first pass and each output is within half a step,
    # of values up to 4.5 (fp32: sums of n terms, n 2^-24 of them)
    tol = 4.5 * (3 * HALF_STEP[dtype] if dtype != torch.float32 else 2 * (n + 80) * 2.0 ** -24)
    assert torch.isnan(got[0, :, -2:, 3]).all()
    assert (got[0, :, -2, 5] == float("inf")).all() and torch.isnan(got[0, :, -1, 5]).all()
    rest = torch.ones(D, dtype=torch.bool, device=device)
    rest[[3, 5]] = False
    assert (got[0, :, -2:, rest] - clean[0, :, -2:, rest]).abs().max() <= tol
    assert (got[0, :, :-2] - clean[0, :, :-2]).abs().max() <= tol if Q > 2 else True
    k[0, n - 1, 0] = float("nan")  # the last token alone sees it
    again = kernels.prompt_attention(q, k, v, n, 0.125).float()
    assert torch.isnan(again[0, :, -1]).all()
    assert torch.equal(torch.nan_to_num(again[0, :, :-1]), torch.nan_to_num(got[0, :, :-1]))
    mask = torch.ones(Q, n, dtype=torch.bool, device=device).tril(n - Q)
    mask[:, at:] = False  # masked for everyone
    k[0, at:], v[0, at:] = float("nan"), float("inf")
    hidden = kernels.prompt_attention(q, k, v, n, 0.125, mask=mask).float()
    assert torch.isfinite(hidden).all()
    ref = kernels.prompt_attention(q, k[:, :at], v[:, :at], at, 0.125, mask=mask[:, :at]).float()
    assert (hidden - ref).abs().max() <= tol


def test_scores_far_apart_and_negative_scale(device):
    """A maximum that keeps rising, scores of +-1e4, scales below and at 0."""
    from sva_amd import kernels

    rng = np.random.default_rng(2)
    n, D = 300, 64
    q, k, v = (normal(rng, s, torch.float32, device) for s in ((1, 2, n, D), (1, n, D), (1, n, D)))
    k = k * torch.linspace(0.1, 30, n, device=device)[:, None]
    for scaling in (1.0, -1.0, 10.0, 0.0, 1e-6):
        got = kernels.prompt_attention(q, k, v, n, scaling)
        for h in range(2):
            sign = -1 if scaling < 0 else 1
            check(got[0, h], sign * q[0, h], k[0], v[0], causal(n, n), sign * scaling)


def test_strides_alignment_and_output(device):
    from sva_amd import kernels

    rng = np.random.default_rng(4)
    n, H, G, D = 150, 4, 2, 64
    base = normal(rng, (1, n, H + 2 * G, D), torch.bfloat16, device)  # a fused projection's output
    q, k, v = base[:, :, :H].transpose(1, 2), base[0, :, H:H + G].transpose(0, 1), base[0, :, H + G:].transpose(0, 1)
    want = kernels.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), n, 0.125)
    assert want.transpose(1, 2).is_contiguous()  # what the output projection takes
    assert torch.equal(kernels.prompt_attention(q, k, v, n, 0.125), want)
    assert torch.equal(kernels.prompt_attention(q[0], k, v, n, 0.125), want[0])
    odd = torch.empty(1 + k.numel(), device=device, dtype=k.dtype)[1:].view(G, n, D).copy_(k)
    assert torch.equal(kernels.prompt_attention(q, odd, v.contiguous(), n, 0.125), want)
    out = torch.empty(1, H, n, D, device=device)
    assert kernels.prompt_attention(q, k, v, n, 0.125, out=out) is out
    assert torch.equal(out.bfloat16(), want)
    cols = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(kernels.prompt_attention(cols, k, v, n, 0.125), want)


def test_streams_and_graphs(device):
    from sva_amd import kernels

    rng = np.random.default_rng(6)
    q, k, v = (normal(rng, s, torch.bfloat16, device) for s in ((1, 9, 5, 64), (3, 9000, 64), (3, 9000, 64)))
    q2 = q.flip(1).contiguous()
    call = lambda x: kernels.prompt_attention(x, k, v, 9000, 0.125)  # noqa: E731  (split over the keys: a workspace)
    want, want2 = call(q), call(q2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a = call(q)
        b = call(q2)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want2)
    static = q.clone()
    with torch.cuda.stream(side):
        call(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(static)
    for x, w in ((q2, want2), (q, want), (q2, want2)):
        static.copy_(x)
        graph.replay()
        assert torch.equal(call(q), want)
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_empty(device):
    from sva_amd import kernels

    z = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    assert kernels.prompt_attention(z(1, 2, 0, 64), z(1, 5, 64), z(1, 5, 64), 5, 1.0).shape == (1, 2, 0, 64)
    got = kernels.prompt_attention(z(1, 2, 3, 64) + 1, z(1, 5, 64), z(1, 5, 64), 0, 1.0)
    assert (got == 0).all()
    zero = torch.zeros(1, dtype=torch.int64, device=device)
    got = kernels.prompt_attention(z(2, 4, 64) + 1, z(1, 0, 64), z(1, 0, 64), 0, 1.0, seq_offsets=zero, seq_lens=zero,
                                   q_offsets=zero, q_lens=zero + 4, max_q=4, out=z(2, 4, 64) + 5)
    assert (got == 0).all()


def test_offsets_past_32_bits(device):
    from sva_amd import kernels

    rows, D = 12_000_000, 128  # 3 GB a KV head
    k = torch.zeros(2, rows, D, device=device, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    g = torch.Generator(device=device).manual_seed(0)
    k[:, -300:].normal_(generator=g)
    v[:, -300:].normal_(generator=g)
    q = torch.randn(1, 4, 40, D, device=device, generator=g).bfloat16()
    off, ln = torch.tensor([rows - 300], device=device), torch.tensor([300], device=device)
    got = kernels.prompt_attention(q, k, v, 300, 0.1, seq_offsets=off, seq_lens=ln)
    want = kernels.prompt_attention(q, k[:, -300:].contiguous(), v[:, -300:].contiguous(), 300, 0.1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_far_apart_in_16_bits(device, dtype, rising):
    """The reference moves often, or stays far above later scores; over several ranges of keys too."""
    from sva_amd import kernels

    rng = np.random.default_rng(12)
    for n, Q in ((500, 500), (3000, 5)):
        q, k, v = (normal(rng, s, torch.float32, device) for s in ((1, 3, Q, 64), (1, n, 64), (1, n, 64)))
        size = torch.linspace(0.1, 12, n, device=device)[:, None]
        k = k * (size if rising else size.flip(0))
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        got = kernels.prompt_attention(q, k, v, n, 1.0)
        for h in range(3):
            check(got[0, h], q[0, h], k[0], v[0], causal(Q, n), 1.0)


def test_a_mask_of_the_causal_rule_equals_it(device):
    from sva_amd import kernels

    rng = np.random.default_rng(13)
    for n, Q in ((333, 333), (1200, 70)):
        q, k, v = (normal(rng, s, torch.bfloat16, device) for s in ((1, 6, Q, 64), (2, n, 64), (2, n, 64)))
        mask = torch.ones(Q, n + 3, dtype=torch.bool, device=device).tril(n - Q)[:, :n]  # rows at odd addresses
        want = kernels.prompt_attention(q, k, v, n, 0.125).float()
        got = kernels.prompt_attention(q, k, v, n, 0.125, mask=mask).float()
        # other ranges of keys: weights within half a step each, of values up to 4.5, and half a step of the outputs
        assert (got - want).abs().max() <= 4.5 * 4 * HALF_STEP[torch.bfloat16]


def test_packed_prompts_in_a_graph(device):
    from sva_amd import kernels

    rng = np.random.default_rng(14)
    lens = [100, 1, 60]
    q, k, v = (normal(rng, s, torch.float16, device) for s in ((9, 161, 64), (3, 161, 64), (3, 161, 64)))
    off, ln = torch.tensor([0, 100, 101], device=device), torch.tensor(lens, device=device)
    out = torch.zeros(9, 161, 64, device=device, dtype=torch.float16)

    def call():
        return kernels.prompt_attention(q, k, v, 100, 0.125, seq_offsets=off, seq_lens=ln, q_offsets=off, q_lens=ln,
                                        max_q=100, out=out)

    want = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([100, 1, 60], [50, 1, 10], [100, 1, 60]):  # lengths are read when it runs
        ln.copy_(torch.tensor(lens, device=device))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call())
        if lens[0] == 100:
            assert torch.equal(got, want)
        else:
            assert (got[:, 50:100] == 0).all() and got[:, :50].abs().max() > 0
