"""The next token of a row of logits against the definition in 64 bits, at ties, cuts and values where it can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .paged_reference import sample

pytestmark = pytest.mark.gpu

# The kernel's shares of the sum are off by its weights' rounding: exp in 64 bits (a polynomial of degree 4 on 2^-7.5 of a
# binade, 4e-14, and a table, 2^-53) and half of 2^-45 of the largest weight a token (2^-42 for 2^20 tokens), of at most
# 2^20 tokens and a sum of at least 1 such weight.  A row whose border lies nearer than this to its random number or cut
# has two answers; the rows below are none of these (asserted).
def border(vocab):
    point = min(46, 62 - max(0, (vocab - 1).bit_length()))
    return 1e-13 + vocab * 2.0 ** -(point + 1)


def compare(device, logits, u, dtype, near=None, **params):
    """logits float32 [B, V]; params: numbers, or arrays [B]; near: the border's width."""
    from sva_amd import kernels

    x = torch.as_tensor(np.asarray(logits, np.float32)).to(device, dtype)
    un = torch.as_tensor(np.asarray(u, np.float32)).to(device)
    types = {"temperature": torch.float32, "top_k": torch.int64, "top_p": torch.float32, "min_p": torch.float32}
    given = {k: torch.as_tensor(v).to(device, types[k]) if isinstance(v, np.ndarray) else v for k, v in params.items()}
    got = kernels.sample_tokens(x, un, **given).tolist()
    ref = x.double().cpu().numpy()
    known = 0
    for b in range(len(ref)):
        p = {k: float(np.float32(v[b] if isinstance(v, np.ndarray) else v)) if k != "top_k" else
             int(v[b] if isinstance(v, np.ndarray) else v) for k, v in params.items()}
        want = sample(ref[b], float(un[b]), border=border(ref.shape[1]) if near is None else near, **p)
        known += want is not None
        assert want is None or got[b] == want, (b, got[b], want, p, float(un[b]))
    assert known > len(ref) // 2
    return got


def normal(rng, B, V, spread=2.0):
    return (rng.standard_normal((B, V)) * spread).astype(np.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 8191, 8192, 8193, 50001, 131072])
def test_vocabularies(device, V, dtype):
    rng = np.random.default_rng(V)
    B = 12
    compare(device, normal(rng, B, V), rng.random(B), dtype)
    compare(device, normal(rng, B, V), rng.random(B), dtype, temperature=0.7, top_k=min(V, 50), top_p=0.9)
    compare(device, normal(rng, B, V), rng.random(B), dtype, temperature=1.4, top_p=0.95, min_p=0.002)
    compare(device, normal(rng, B, V), rng.random(B), dtype, temperature=0.0, top_k=7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_row_its_own(device, dtype):
    rng = np.random.default_rng(1)
    B, V = 300, 3001
    compare(device, normal(rng, B, V, 3.0), rng.random(B), dtype,
            temperature=rng.choice([0.0, 0.2, 0.7, 1.0, 2.0], B).astype(np.float32),
            top_k=rng.choice([0, 1, 2, 50, 2000, 3000, 3001, 10 ** 12, -4], B),
            top_p=rng.choice([1.0, 0.9, 0.5, 0.01, 0.0, 0.9999], B).astype(np.float32),
            min_p=rng.choice([0.0, 0.0, 0.1, 0.001, 1.0], B).astype(np.float32))


@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (5000, 1.0), (0, 0.5), (7000, 0.3), (3, 0.5), (0, 0.00001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_ties(device, top_k, top_p, dtype):
    """All logits equal, or of four values: cuts fall among more ties than are sorted; the lowest tokens stay."""
    rng = np.random.default_rng(7)
    V = 20000
    for x in (np.full((6, V), -3.5, np.float32), rng.choice([0.0, -0.0, 1.0, -2.0], (6, V)).astype(np.float32)):
        u = np.array([0.0, 0.25 + 1e-5, 0.5, 0.7, 0.9, 1 - 2.0 ** -24], np.float32)
        # (equal logits weigh 1 each: their sums, and a sum of 15 bits times a number of 24, are exact, at a border too)
        compare(device, x, u, dtype, near=0.0 if x.min() == x.max() else None, top_k=top_k, top_p=top_p)


@pytest.mark.parametrize("top_k,top_p,min_p", [(5000, 1.0, 0.0), (0, 0.5, 0.0), (7000, 0.3, 0.0), (12500, 1.0, 0.0),
                                               (12500, 0.8, 0.1), (0, 0.9, 0.3), (19990, 0.99999, 0.0), (300, 0.5, 0.0)])
@pytest.mark.parametrize("V", [20000, 100003])
def test_few_values(device, V, top_k, top_p, min_p):
    """bf16 rows of a few values, -0 beside 0: the cut falls among thousands of equal logits."""
    rng = np.random.default_rng(V + top_k)
    values = [[0.0, -0.0, 1.0, -2.0], [0.0, -0.0], [-0.0, -1.0, -3.0], [2.0, 3.0, 3.015625], [-5.0, -5.03125, -100.0]]
    x = np.stack([rng.choice(np.array(v, np.float32), V) for v in values for _ in range(3)])
    # (the 300 largest are equal in every row: they weigh 1 each, half of their sum is 150 exactly, and 300 times a number
    # of 24 bits is exact in 64: no border is unclear)
    compare(device, x, rng.random(len(x)), torch.bfloat16, near=0.0 if top_k == 300 else None, top_k=top_k, top_p=top_p,
            min_p=min_p)


@pytest.mark.parametrize("T", [0.05, 1.0, 12.0, 500.0])
def test_values_at_the_ends_of_bf16(device, T):
    """bf16 logits of 510 and more, of less than 2^-55, of -510 and less that weigh something, and far below."""
    rng = np.random.default_rng(5)
    V = 30001
    x = normal(rng, 14, V)
    x[0] += 507.0
    x[1, 20] = 1e30
    x[2, ::3] *= 1e-20
    x[3, ::2] = 0.0
    x[4, ::2] *= 2.0 ** -54
    x[5] -= 508.0
    x[6] -= 511.0
    x[7, ::2] = -509.0
    x[8, ::2] = -512.0
    x[9, 1:] = -np.inf
    x[10, ::2] = np.nan
    x[11, 5::7] = -np.nan
    x[12, 9000] = np.inf
    x[13] *= 1e4
    u = rng.random(14)
    for params in ({"top_p": 0.9}, {"top_k": 6000}, {"top_k": 14000, "top_p": 0.99}, {"top_p": 0.7, "min_p": 0.01}):
        compare(device, x, u, torch.bfloat16, temperature=T, **params)


@pytest.mark.parametrize("mask", [-np.inf, float(np.finfo(np.float32).min) * 0.99, -1e4])
@pytest.mark.parametrize("V,kept", [(40000, 900), (130001, 9000)])
def test_masked_bf16(device, V, kept, mask):
    rng = np.random.default_rng(V + kept)
    x = normal(rng, 6, V)
    for b in range(6):
        x[b, rng.permutation(V)[:V - kept]] = mask
        x[b, :V // 2 if b % 2 else 0] = mask
    u = rng.random(6)
    for params in ({"top_p": 0.9}, {"top_k": 300}, {"top_k": 8000}, {"top_k": 8000, "top_p": 0.8},
                   {"top_k": 10000, "top_p": 0.999, "temperature": 0.4}, {"top_p": 0.9, "temperature": 20.0}):
        compare(device, x, u, torch.bfloat16, **params)


@pytest.mark.parametrize("top_k,top_p,T", [(5000, 1.0, 1.0), (0, 0.7, 1.0), (9000, 0.9, 1.0), (3000, 0.5, 0.01), (0, 0.999, 30.0)])
def test_cuts_far_below_the_largest(device, top_k, top_p, T):
    """One logit far above the others, so that a cut lies where the first bins say nothing; and logits far apart."""
    rng = np.random.default_rng(3)
    V = 30000
    x = normal(rng, 8, V)
    x[:4, 77] = 300.0
    x[4:] *= 1e4
    compare(device, x, rng.random(8), torch.float32, top_k=top_k, top_p=top_p, temperature=T)


@pytest.mark.parametrize("mask", [-np.inf, float(np.finfo(np.float32).min), -1e9])
@pytest.mark.parametrize("V,kept", [(3000, 40), (40000, 900), (40000, 9000)])
def test_masked_vocabularies(device, V, kept, mask):
    """Most tokens masked, the first ones of the row among them; top_k of more tokens than are left."""
    rng = np.random.default_rng(V + kept)
    x = normal(rng, 6, V)
    for b in range(6):
        x[b, rng.permutation(V)[:V - kept]] = mask
        x[b, :V // 2 if b % 2 else 0] = mask
    u = rng.random(6)
    for params in ({}, {"top_p": 0.9}, {"top_k": 300}, {"top_k": 8000}, {"top_k": 8000, "top_p": 0.8}, {"min_p": 0.01},
                   {"top_k": 10000, "top_p": 0.999, "temperature": 0.4}, {"top_k": 20, "top_p": 0.7}):
        compare(device, x, u, torch.float32, **params)


@pytest.mark.parametrize("T", [0.1, 1.0, 8.0])
@pytest.mark.parametrize("V", [16384, 16385, 60000])
def test_the_largest_come_last(device, V, T):
    """Rows whose first thousands of logits are far below the others, or rise to the end."""
    rng = np.random.default_rng(V)
    x = normal(rng, 8, V)
    x[:4, :15000] -= 60.0
    x[4:6].sort(axis=1)
    x[6:, -5:] += 40.0
    for dtype in (torch.float32, torch.bfloat16):
        for params in ({"top_p": 0.9}, {"top_k": 700}, {"top_k": 700, "top_p": 0.6}, {"top_k": 7000, "min_p": 0.001}, {}):
            compare(device, x, rng.random(8), dtype, temperature=T, **params)


def test_values_that_are_not_finite(device):
    rng = np.random.default_rng(5)
    V = 9000
    x = normal(rng, 8, V)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan                 # as -inf
    x[3, 5:] = -np.inf                 # five tokens
    x[4, [17, 4000, 8999]] = np.inf    # share all of the weight
    x[5, :8990] = np.finfo(np.float32).min
    x[6] = -np.inf
    x[6, 8999] = -3e38
    u = np.array([0.5, 0.5, 0.3, 0.6, 0.5, 0.5, 0.99, 0.8])
    for params in ({}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0}, {"top_k": 8000, "top_p": 0.5}):
        got = compare(device, x, u, torch.float32, **params)
        assert got[0] == got[1] == -1 and got[6] == 8999 and got[4] in (17, 4000)


def test_numbers_at_the_ends(device):
    """0: the first kept token with any weight; just under 1, and 1 and above: the last; below 0 and NaN: as 0."""
    from sva_amd import kernels

    x = torch.tensor([[-200.0, 1.0, 3.0, 2.0, -200.0]], device=device).repeat(6, 1)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")], device=device)
    assert kernels.sample_tokens(x, u).tolist() == [1, 3, 3, 3, 1, 1]
    assert kernels.sample_tokens(x, u, top_k=2).tolist() == [2, 3, 3, 3, 2, 2]
    odd = torch.tensor([float("nan")] * 6, device=device)
    assert kernels.sample_tokens(x, u, top_p=odd).tolist() == [2] * 6        # one at least
    assert kernels.sample_tokens(x, u, temperature=odd).tolist() == [2] * 6  # no weight at all: the largest
    wide = torch.tensor([float("inf")] * 6, device=device)
    assert kernels.sample_tokens(x, u, temperature=wide).tolist() == [0, 4, 4, 4, 0, 0]


def test_strides_and_the_largest_vocabulary(device):
    from sva_amd import kernels

    rng = np.random.default_rng(9)
    V = 5003
    x = torch.as_tensor(normal(rng, 6, V)).to(device)
    u = torch.as_tensor(rng.random(6).astype(np.float32)).to(device)
    want = kernels.sample_tokens(x, u, top_p=0.9)
    padded = torch.full((6, 2, V + 5), 100.0, device=device)[:, 1]
    padded[:, 1:V + 1] = x
    assert torch.equal(kernels.sample_tokens(padded[:, 1:V + 1], u, top_p=0.9), want)
    aligned = torch.full((6, 8192), 100.0, device=device)
    aligned[:, :V] = x
    assert torch.equal(kernels.sample_tokens(aligned[:, :V], u, top_p=0.9), want)
    assert torch.equal(kernels.sample_tokens(x.T.contiguous().T, u, top_p=0.9), want)
    assert torch.equal(kernels.sample_tokens(x[:1].expand(6, V), u, top_p=0.9)[:1], want[:1])
    assert kernels.sample_tokens(x[:0], u[:0]).shape == (0,)
    big = normal(rng, 3, 1 << 20)
    compare(device, big, [0.1, 0.5, 0.9], torch.bfloat16)
    compare(device, big, [0.1, 0.5, 0.9], torch.bfloat16, top_p=0.8, top_k=100000)


def test_shares(device):
    """Numbers spread evenly over [0, 1) give every token its share of them, within one."""
    from sva_amd import kernels

    rng = np.random.default_rng(4)
    n, V = 20000, 40
    x = normal(rng, 1, V)
    u = torch.as_tensor(((np.arange(n) + 0.5) / n).astype(np.float32)).to(device)
    got = kernels.sample_tokens(torch.as_tensor(x).to(device).expand(n, V), u, temperature=0.9, top_k=20, top_p=0.95)
    w = np.exp(x[0].astype(np.float64) / float(np.float32(0.9)))
    order = np.argsort(-w)[:20]
    share = np.cumsum(w[order]) / w[order].sum()
    order = order[:int((share < float(np.float32(0.95))).sum()) + 1]
    want = np.zeros(V)
    want[order] = w[order] / w[order].sum() * n
    assert (np.abs(np.bincount(got.cpu().numpy(), minlength=V) - want) <= 1.01 + n * 2.0 ** -23).all()


def test_in_a_graph_and_on_another_stream(device):
    from sva_amd import kernels

    rng = np.random.default_rng(6)
    x = torch.as_tensor(normal(rng, 5, 40000)).to(device)
    u = torch.zeros(5, device=device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kernels.sample_tokens(x, u, top_p=0.9, top_k=10000)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.sample_tokens(x, u, top_p=0.9, top_k=10000)
    for i in range(10):
        u.copy_(torch.as_tensor(rng.random(5).astype(np.float32)))
        x.mul_(1.01)
        graph.replay()
        assert torch.equal(out, kernels.sample_tokens(x, u, top_p=0.9, top_k=10000)), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [0.05, 0.1, 0.2, 0.7])
@pytest.mark.parametrize("V", [3, 3000, 20000])
def test_only_what_weighs_as_much_as_the_largest(device, V, T, dtype):
    """min_p = 1 with tied largest logits, of any size against the temperature: all of them are kept, and nothing else."""
    rng = np.random.default_rng(V)
    B = 48
    x = np.minimum(normal(rng, B, V), 4.0)
    top = 5.0 + np.concatenate([np.arange(B - 4) * 1.375, [12.875, 13.75, 25.5, 45.0]]).astype(np.float32)  # 17.875, 18.75, 30.5, 50
    for b in range(B):
        x[b, rng.permutation(V)[:2 if V == 3 else 2 + 5 * b]] = top[b]
    u = rng.random(B)
    for params in ({}, {"top_p": 0.9}, {"top_k": max(1, V // 2)}, {"top_k": 40}, {"top_k": 600, "top_p": 0.47}):
        got = compare(device, x, u, dtype, temperature=T, min_p=1.0, **params)
        assert all(x[b, g] == top[b] for b, g in enumerate(got))
    odd = np.where(np.arange(B) % 2, np.float32(1e-32), np.float32(T))  # too cold for the usual weights
    compare(device, x, u, dtype, temperature=odd, min_p=1.0)


def test_masked_and_absent_logits_take_no_longer(device):
    """A share of the sum (top_p) at temperatures whose reciprocal fp32 rounds up, or down: rows that do not fill their
    last step, and rows masked with -inf or the lowest number, are cut in the same number of passes.  (A row that is done
    over again takes several times as long; the factor leaves room for the cards' noise alone.)"""
    from sva_amd import kernels

    gen = torch.Generator(device=device).manual_seed(2)

    def time(x, T):
        u = torch.rand(x.shape[0], device=device, generator=gen)
        kernels.sample_tokens(x, u, temperature=T, top_p=0.9)
        best = float("inf")
        for _ in range(15):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                kernels.sample_tokens(x, u, temperature=T, top_p=0.9)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    for V, mask in ((50001, None), (49152, -float("inf")), (49152, torch.finfo(torch.float32).min)):
        x = torch.randn(64, V, device=device, generator=gen) * 2.0
        if mask is not None:
            x[:, torch.randperm(V, device=device, generator=gen)[:V // 2]] = mask
        want = time(x, 1.0)
        for T in (0.7, 0.8, 0.9):
            assert time(x, T) < 2.0 * want, (V, mask, T)


@pytest.mark.parametrize("T", [1e-39, 1e-44, 1e-36, 1e-31])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cuts_of_ties_at_any_temperature(device, T, dtype):
    """top_k among equal largest logits where 1 / temperature is past fp32."""
    V = 30000
    x = np.full((6, V), -2.0, np.float32)
    x[3:] = 0.5
    x[3:, ::3] = 1.25
    u = np.array([0.0, 0.3, 0.77, 0.1, 0.5, 0.99], np.float32)
    # (equal weights of 2^45 each: sums and borders are exact)
    for params in ({"top_k": 300}, {"top_k": 5000}, {"top_k": 5000, "top_p": 0.5}, {"top_k": 40}):
        compare(device, x, u, dtype, temperature=T, near=0.0, **params)
