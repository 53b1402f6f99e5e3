"""Attention over a cache in pages, and the write and read of its rows, against softmax attention in 64 bits and the rows
themselves."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .paged_reference import check_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(gen, shape, dtype, device):
    return torch.randn(*shape, generator=gen).to(device, dtype)


def make(device, lens, G, D, P, dtype, seed=0, spare=3, layers=0):
    """(pool, tables, lens, keys, values): pages of the sequences scattered over a pool whose other rows are NaN."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // P) for n in lens]
    pages = sum(counts) + spare
    pool = torch.full((pages, max(1, layers), 2, G, P, D), float("nan"), dtype=dtype)[:, layers // 2]
    tables = torch.full((len(lens), max(counts) + 2), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=gen).int()
    kv, at = [], 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        tables[b, :c] = order[at:at + c]
        rows = torch.randn(2, G, n, D, generator=gen).to(dtype)
        for i in range(c):
            part = rows[:, :, i * P:(i + 1) * P]
            pool[order[at + i], :, :, :part.shape[2]] = part
        kv.append(rows.to(device))
        at += c
    whole = torch.empty((pages, max(1, layers), 2, G, P, D), dtype=dtype, device=device)
    whole[:, layers // 2] = pool.to(device)
    return whole[:, layers // 2], tables.to(device), torch.tensor(lens, device=device), kv, gen


def check(got, q, kv, lens, scaling):
    n_seq, H, Q, D = q.shape
    for b, n in enumerate(lens):
        G = kv[b].shape[1]
        for h in range(H):
            allowed = np.arange(n) <= n - Q + np.arange(Q)[:, None]
            check_attention(got[b, h], q[b, h], kv[b][0, h // (H // G)], kv[b][1, h // (H // G)], allowed, scaling)


@pytest.mark.parametrize("lens,Q,H,G,D,P,dtype", [
    ([1], 1, 1, 1, 64, 16, F32), ([15], 1, 9, 3, 64, 16, BF16), ([16], 1, 9, 3, 64, 16, F16), ([17], 1, 4, 4, 128, 16, F32),
    ([0, 33, 1], 1, 8, 2, 128, 32, BF16), ([255, 256, 257, 0], 1, 9, 3, 64, 16, BF16), ([700, 31], 1, 12, 4, 64, 64, F32),
    ([3000], 1, 9, 3, 64, 16, F32), ([5000, 4097], 1, 32, 8, 128, 128, BF16), ([20000], 1, 9, 3, 64, 1024, F16),
    ([2500, 3, 77, 1025], 4, 12, 4, 64, 16, F16), ([40], 40, 9, 3, 64, 16, BF16), ([600, 5], 9, 16, 2, 128, 32, F32),
    ([900], 7, 16, 2, 64, 16, BF16), ([300, 40], 2, 4, 1, 256, 16, BF16), ([300, 40], 1, 4, 1, 256, 64, F32),
    ([515], 3, 2, 1, 256, 16, F16), ([130, 9], 1, 3, 1, 8, 16, BF16), ([130], 2, 2, 2, 40, 32, F16),
    ([333], 1, 3, 3, 72, 16, F32), ([515], 2, 4, 2, 96, 16, BF16), ([600], 1, 2, 1, 200, 16, F16), ([600], 1, 2, 1, 136, 16, F32),
    ([90, 200], 1, 64, 2, 64, 16, BF16), ([5, 2], 7, 6, 2, 64, 16, F32)])
def test_against_64_bits(device, lens, Q, H, G, D, P, dtype):
    from sva_amd import kernels

    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype, seed=sum(lens) + D)
    q = normal(gen, (len(lens), H, Q, D), dtype, device)
    for out_dtype in {dtype, F32}:
        got = kernels.paged_attention(q, pool, tables, seq_lens, D ** -0.5, n_keys=max(1, max(lens)), out_dtype=out_dtype)
        assert got.shape == q.shape and got.dtype == out_dtype
        check(got, q, kv, lens, D ** -0.5)
    # the bound that the tables give, and a negative scale
    check(kernels.paged_attention(q, pool, tables, seq_lens, D ** -0.5), q, kv, lens, D ** -0.5)
    check(kernels.paged_attention(-q, pool, tables, seq_lens, -(D ** -0.5)), q, kv, lens, D ** -0.5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strides(device, dtype):
    """A layer of a pool that holds several, tokens before heads, rows at odd addresses, columns of a wider table."""
    from sva_amd import kernels

    lens, H, G, D, P = [100, 37, 260], 6, 2, 64, 16
    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype, layers=3)
    assert not pool.is_contiguous()
    q = normal(gen, (3, 2, H, D), dtype, device).transpose(1, 2)
    odd = torch.empty(3, H, 2, D + 3, device=device, dtype=dtype)[..., 1:1 + D]
    odd.copy_(q)
    wide = torch.full((3, 50), 1 << 30, device=device, dtype=torch.int32)
    wide[:, 5:5 + tables.shape[1]] = tables
    cut = wide[:, 5:5 + tables.shape[1]]
    want = kernels.paged_attention(q.contiguous(), pool.contiguous(), tables, seq_lens, 0.2)
    check(want, q, kv, lens, 0.2)
    for x, t in ((q, tables), (odd, cut), (q.expand(3, H, 2, D), cut)):
        assert torch.equal(kernels.paged_attention(x, pool, t, seq_lens, 0.2), want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_without_a_page(device, dtype):
    """Entries outside the pool: their rows are not seen, by attention, write and read."""
    from sva_amd import kernels

    lens, H, G, D, P = [200, 90], 4, 2, 64, 16
    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype)
    gone = {0: [0, 3, 12], 1: [5]}
    for (b, pages), bad in zip(gone.items(), (pool.shape[0], -7)):
        tables[b, pages] = bad
    tables[0, 3] = 2 ** 31 - 1
    q = normal(gen, (2, H, 2, D), dtype, device)
    got = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
    for b, n in enumerate(lens):
        there = ~np.isin(np.arange(n) // P, gone[b])
        for h in range(H):
            allowed = (np.arange(n) <= n - 2 + np.arange(2)[:, None]) & there
            check_attention(got[b, h], q[b, h], kv[b][0, h // 2], kv[b][1, h // 2], allowed, 0.3)
    keys, values = kernels.paged_read(pool, tables, [0, 0], 90)
    for b in range(2):
        there = torch.from_numpy(~np.isin(np.arange(90) // P, gone[b])).to(device)
        for x, want in ((keys[b], kv[b][0]), (values[b], kv[b][1])):
            assert torch.equal(x[:, there], want[:, :90][:, there]) and (x[:, ~there] == 0).all()
    before = pool.clone()
    kernels.paged_write(keys + 1, values, pool, torch.full_like(tables, -1), [0, 5])
    kernels.paged_write(keys + 1, values, pool, tables, [-1000, 10 ** 9])
    assert torch.equal(pool.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_what_is_not_seen_reaches_nothing(device, dtype):
    """Rows behind a token, of K and V, that are infinite or NaN (the rest of the pool is NaN as it is)."""
    from sva_amd import kernels

    lens, H, G, D, P = [70, 33], 4, 2, 64, 16
    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype)
    q = normal(gen, (2, H, 5, D), dtype, device)
    want = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
    check(want, q, kv, lens, 0.3)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for b, n in enumerate(lens):  # the last two rows: seen by tokens 3 and 4, or by 4 alone
            page, row = int(tables[b, (n - 2) // P]), (n - 2) % P
            pool[page, 1, :, row] = bad
            page, row = int(tables[b, (n - 1) // P]), (n - 1) % P
            pool[page, 0, :, row] = bad
        got = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
        assert torch.isfinite(got[:, :, :3]).all()
        for b, n in enumerate(lens):
            for h in range(H):
                allowed = np.arange(n) <= n - 5 + np.arange(3)[:, None]
                check_attention(got[b, h, :3], q[b, h, :3], kv[b][0, h // 2], kv[b][1, h // 2], allowed, 0.3)
        assert not torch.isfinite(got[:, :, 3]).any()
        if bad == bad:  # an infinite element of V is one of the output
            assert (got[:, :, 3].float() == bad).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_range_done_again_joins_the_others(device, dtype):
    """Several ranges, of which one holds what takes its sums out of the finite numbers: its share stays as large as it is."""
    from sva_amd import kernels

    lens, H, G, D, P = [3000, 2100], 4, 2, 64, 16
    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype)
    q = normal(gen, (2, H, 5, D), dtype, device)
    clean, want = pool.clone(), kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
    check(want, q, kv, lens, 0.3)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for b, n in enumerate(lens):  # the last row: seen by token 4 alone
            pool[int(tables[b, (n - 1) // P]), :, :, (n - 1) % P] = bad
        got = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
        for b, n in enumerate(lens):
            for h in range(H):
                allowed = np.arange(n) <= n - 5 + np.arange(4)[:, None]
                check_attention(got[b, h, :4], q[b, h, :4], kv[b][0, h // 2], kv[b][1, h // 2], allowed, 0.3)
    # an infinite element of V is one of the output; the others are as they were
    pool.copy_(clean)
    pool[int(tables[0, 1500 // P]), 1, :, 1500 % P, 7] = float("inf")
    got = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
    assert torch.isinf(got[0, :, :, 7]).all()
    rest = torch.arange(D, device=device) != 7
    for h in range(H):
        allowed = np.arange(3000) <= 2995 + np.arange(5)[:, None]
        whole = torch.where(rest, got[0, h], want[0, h])
        check_attention(whole, q[0, h], kv[0][0, h // 2], kv[0][1, h // 2], allowed, 0.3)
    # rows without a page, page 0 (which is read in their place) of NaN
    pool.copy_(clean)
    tables[0, 60] = -1
    zero = (tables == 0).nonzero()
    for b, at in zero.tolist():
        tables[b, at] = -1
    pool[0] = float("nan")
    gone = {0: [60], 1: []}
    for b, at in zero.tolist():
        gone[b].append(at)
    got = kernels.paged_attention(q, pool, tables, seq_lens, 0.3)
    for b, n in enumerate(lens):
        there = ~np.isin(np.arange(n) // P, gone[b])
        for h in range(H):
            allowed = (np.arange(n) <= n - 5 + np.arange(5)[:, None]) & there
            check_attention(got[b, h], q[b, h], kv[b][0, h // 2], kv[b][1, h // 2], allowed, 0.3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,cut", [(100, 50), (100, 97), (3000, 2600), (3000, 2998)])
def test_sequences_longer_than_what_is_read(device, n, cut, dtype):
    """Rows behind n_keys, or behind the table, are not read; a token still sees every row up to its own place before."""
    from sva_amd import kernels

    H, G, D, P, Q = 4, 2, 64, 16, 5
    pool, tables, seq_lens, kv, gen = make(device, [n], G, D, P, dtype)
    q = normal(gen, (1, H, Q, D), dtype, device)
    short = tables[:, :cut // P]
    for got, rows in ((kernels.paged_attention(q, pool, tables, seq_lens, 0.2, n_keys=cut), cut),
                      (kernels.paged_attention(q, pool, short, seq_lens, 0.2), cut // P * P)):
        for h in range(H):
            allowed = np.arange(rows) <= n - Q + np.arange(Q)[:, None]
            check_attention(got[0, h], q[0, h], kv[0][0, h // 2, :rows], kv[0][1, h // 2, :rows], allowed, 0.2)
    # lengths past any table, and none
    far = kernels.paged_attention(q, pool, tables, torch.tensor([2 ** 62], device=device), 0.2, n_keys=cut)
    for h in range(H):
        check_attention(far[0, h], q[0, h], kv[0][0, h // 2, :cut], kv[0][1, h // 2, :cut], np.ones((Q, cut), bool), 0.2)
    assert (kernels.paged_attention(q, pool, tables, torch.tensor([-2 ** 63], device=device), 0.2, n_keys=cut) == 0).all()


def test_an_infinite_key_takes_or_leaves_all(device):
    """Scores of -inf weigh nothing, of one +inf make the row NaN, as in softmax."""
    from sva_amd import kernels

    pool, tables, seq_lens, kv, gen = make(device, [50], 1, 64, 16, F32)
    q = torch.ones(1, 1, 1, 64, device=device)
    pool[tables[0, 1], 0, 0, 3, 7] = -float("inf")
    kv[0][0, 0, 19, 7] = -1e30
    got = kernels.paged_attention(q, pool, tables, seq_lens, 0.1)
    check_attention(got[0, 0], q[0, 0], kv[0][0, 0], kv[0][1, 0], np.arange(50)[None] != 19, 0.1)
    pool[tables[0, 1], 0, 0, 3, 7] = float("inf")
    assert torch.isnan(kernels.paged_attention(q, pool, tables, seq_lens, 0.1)).all()


@pytest.mark.parametrize("dtype,large", [(F32, 3e38), (BF16, 3e38), (F16, 60000.0)])
@pytest.mark.parametrize("n", [40, 3000])
def test_values_near_the_largest(device, dtype, large, n):
    """V near the type's largest number: the outputs are finite, within a thousandth (fp32 sums of 2^-60 of them)."""
    from sva_amd import kernels

    pool, tables, seq_lens, kv, gen = make(device, [n], 1, 64, 16, dtype)
    sign = torch.where(torch.rand(n, 1, generator=gen) < 0.9, 1.0, -1.0).to(device)
    for i in range(-(-n // 16)):
        part = (sign[16 * i:16 * i + 16] * large).to(dtype).expand(-1, 64)
        pool[tables[0, i], 1, 0, :part.shape[0]] = part
    q = normal(gen, (1, 2, 1, 64), dtype, device)
    got = kernels.paged_attention(q, pool, tables, seq_lens, 0.1, out_dtype=F32)
    K, V = kv[0][0, 0].double(), (sign * large).to(dtype).double().expand(-1, 64)
    w = torch.softmax(q[0, :, 0].double() @ K.T * 0.1, -1)
    assert ((got[0, :, 0].double() - w @ V).abs() <= 1e-3 * large).all()


@pytest.mark.parametrize("dtype,size", [(F32, 2.0 ** 20), (BF16, 2.0 ** 20), (F16, 2.0 ** 7)])
def test_large_scores(device, dtype, size):
    """Scores up to 2^40: the largest takes all; equal ones share (differences are exact before the scale)."""
    from sva_amd import kernels

    n, D = 600, 64
    pool, tables, seq_lens, kv, gen = make(device, [n], 1, D, 16, dtype)
    q = torch.zeros(1, 1, 1, D, device=device, dtype=dtype)
    q[..., 0] = size
    keys = torch.zeros(n, D, device=device, dtype=dtype)
    keys[:, 0] = -size
    keys[[7, 300, 599], 0] = size
    kernels.paged_write(keys[None, None], kv[0][1][None].contiguous(), pool, tables, [0])
    got = kernels.paged_attention(q, pool, tables, seq_lens, 1.0, out_dtype=F32)
    want = kv[0][1, 0][[7, 300, 599]].double().mean(0)
    assert ((got[0, 0, 0].double() - want).abs() <= 2.0 ** -15 * 4).all()  # two terms of weights that are equal


@pytest.mark.parametrize("G,D,P,dtype,T", [(3, 64, 16, BF16, 1), (3, 64, 16, F32, 37), (2, 128, 64, F16, 130), (1, 8, 16, BF16, 50),
                                           (2, 72, 32, F32, 33), (1, 256, 1024, F16, 1500)])
def test_write_and_read(device, G, D, P, dtype, T):
    from sva_amd import kernels

    lens = [T + 40, T + 7, T]
    pool, tables, seq_lens, kv, gen = make(device, lens, G, D, P, dtype)
    first = torch.tensor([29, 0, 0], device=device)
    rows = normal(gen, (2, 3, T, G, D), dtype, device).transpose(2, 3)  # tokens before heads
    kernels.paged_write(rows[0], rows[1], pool, tables, first)
    keys, values = kernels.paged_read(pool, tables, [0, 0, 0], T + 40)
    for b, a in enumerate(first.tolist()):
        kv[b][:, :, a:a + T] = rows[:, b]
        assert torch.equal(keys[b, :, :lens[b]], kv[b][0]) and torch.equal(values[b, :, :lens[b]], kv[b][1])
    # rows at odd addresses
    odd = torch.empty(2, 3, G, T, D + 1, device=device, dtype=dtype)[..., 1:]
    odd.copy_(rows)
    again = pool.clone()
    for b, a in enumerate(first.tolist()):  # one sequence at a time, by an int
        kernels.paged_write(odd[0, b], odd[1, b], again, tables[b:b + 1], a)
    assert torch.equal(again.view(torch.uint8), pool.view(torch.uint8))


def test_many_sequences(device):
    """More (sequence, head) pairs than a grid's second dimension holds."""
    from sva_amd import kernels

    n, G, D, P = 20000, 4, 8, 16
    gen = torch.Generator(device=device).manual_seed(2)
    pool = kernels.pages_alloc(n, G, P, D, device, F32)
    tables = torch.randperm(n, device=device, generator=gen).int()[:, None]
    lens = torch.arange(n, device=device) % P + 1
    keys, values = (torch.randn(n, G, P, D, device=device, generator=gen) for _ in range(2))
    kernels.paged_write(keys, values, pool, tables, torch.zeros(n, device=device, dtype=torch.int64))
    back = kernels.paged_read(pool, tables, torch.zeros(n, device=device, dtype=torch.int64), P)
    assert torch.equal(back[0], keys) and torch.equal(back[1], values)
    q = torch.randn(n, G, 1, D, device=device, generator=gen)
    got = kernels.paged_attention(q, pool, tables, lens, 0.3)
    s = (q.double() @ keys.double().transpose(-1, -2) * 0.3).masked_fill(torch.arange(P, device=device) >= lens[:, None, None, None],
                                                                        -float("inf"))
    want = torch.softmax(s, -1) @ values.double()
    # scores of 8 products and 16 weights and sums: (2 (8 + 4) + 16 + 16) 2^-24 of at most 16 values' size, scores under 30
    assert (got.double() - want).abs().max() <= 30 * 56 * 2.0 ** -24 * values.abs().max()


def test_beyond_32_bits(device):
    """Pages, and elements between pages, past 2^32."""
    from sva_amd import kernels

    G, D, P, n = 2, 64, 16, 40
    pages = 2 ** 33 // (2 * G * P * D * 2) + 2  # 8 GiB
    pool = kernels.pages_alloc(pages, G, P, D, device)
    gen = torch.Generator().manual_seed(1)
    tables = torch.tensor([[pages - 1, 0, pages - 2], [1, pages // 2 + 1, 2]], device=device, dtype=torch.int32)
    kv = [normal(gen, (2, G, n, D), BF16, device) for _ in range(2)]
    kernels.paged_write(torch.stack([x[0] for x in kv]), torch.stack([x[1] for x in kv]), pool, tables, [0, 0])
    keys, values = kernels.paged_read(pool, tables, [0, 0], n)
    assert all(torch.equal(keys[b], kv[b][0]) and torch.equal(values[b], kv[b][1]) for b in range(2))
    q = normal(gen, (2, 4, 1, D), BF16, device)
    check(kernels.paged_attention(q, pool, tables, torch.tensor([n, n], device=device), 0.2), q, kv, [n, n], 0.2)
    kernels.pages_copy(pool, torch.tensor([pages - 1], device=device, dtype=torch.int32),
                       torch.tensor([7], device=device, dtype=torch.int32))
    assert torch.equal(pool[7], pool[pages - 1])


def test_shared_pages_and_another_stream(device):
    """Two sequences that name the same pages; calls on two streams at once."""
    from sva_amd import kernels

    pool, tables, seq_lens, kv, gen = make(device, [1500, 1200], 3, 64, 16, BF16)
    tables[1] = tables[0]
    q = normal(gen, (2, 9, 1, 64), BF16, device)
    want = kernels.paged_attention(q, pool, tables, seq_lens, 0.125)
    check(want, q, [kv[0], kv[0][:, :, :1200]], [1500, 1200], 0.125)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(kernels.paged_attention(q, pool, tables, seq_lens, 0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in outs)


def test_empty_calls(device):
    from sva_amd import kernels

    pool, tables, seq_lens, kv, gen = make(device, [20, 30], 2, 64, 16, F32)
    q = normal(gen, (2, 4, 1, 64), F32, device)
    assert kernels.paged_attention(q[:0], pool, tables[:0], seq_lens[:0], 1.0).shape == (0, 4, 1, 64)
    assert kernels.paged_attention(q[:, :, :0], pool, tables, seq_lens, 1.0).shape == (2, 4, 0, 64)
    assert (kernels.paged_attention(q, pool, tables, seq_lens, 1.0, n_keys=0) == 0).all()
    assert (kernels.paged_attention(q, pool[:0], tables, seq_lens, 1.0) == 0).all()
    assert (kernels.paged_attention(q, pool, tables[:, :0], seq_lens, 1.0) == 0).all()
    assert (kernels.paged_attention(q, pool, tables, torch.tensor([-3, 0], device=device), 1.0) == 0).all()
    kernels.paged_write(q[:, :2, :0], q[:, :2, :0], pool, tables, [0, 0])
    assert kernels.paged_read(pool, tables, [0, 0], 0)[0].shape == (2, 2, 0, 64)
    assert (kernels.paged_read(pool[:0], tables, [0, 0], 3)[1] == 0).all()
