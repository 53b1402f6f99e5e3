"""Subspaces of any width, also ones that are no whole number of 16-byte words: the query's table, the rows' codes and
the lookup over them against the plain computation, twice with other work in between."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,sub,C", [(2, 2, 8), (4, 1, 16), (4, 3, 8), (2, 6, 64), (8, 2, 256), (2, 10, 32), (2, 4, 8)])
@pytest.mark.parametrize("Q", [1, 9])
def test_tables_and_codes(device, S, sub, C, Q):
    from sva_amd import kernels

    g = torch.Generator(device=device).manual_seed(S + sub)
    H, G, D, R, n = 4, 2, 32, S * sub, 300
    q_proj, k_proj = (torch.randn(H, D, R, device=device, generator=g) for _ in range(2))
    books = torch.randn(H, S, C, sub, device=device, generator=g)
    scale = torch.rand(H, device=device, generator=g) + 0.5
    q, keys = torch.randn(1, H, Q, D, device=device, generator=g), torch.randn(G, n, D, device=device, generator=g)
    k_low = torch.empty(H, n, R, device=device)
    codes = torch.empty(H, n, S, device=device, dtype=torch.uint8)
    kernels.write_encode(keys, k_proj, books, k_low, codes)
    want_low = torch.matmul(keys.repeat_interleave(H // G, 0).double(), k_proj.double())
    assert (k_low.double() - want_low).abs().max() <= 2.0 ** -23 * D * 2 * want_low.abs().max()
    parts = k_low.double().view(H, n, S, 1, sub)
    distance = ((parts - books.double()[:, None]) ** 2).sum(-1)  # [H, n, S, C]
    best = distance.min(-1).values
    taken = distance.gather(-1, codes.long()[..., None])[..., 0]
    # fp32 scores of sub products decide: within 8 (sub + 2) 2^-24 of the terms' size
    assert (taken - best <= 8 * (sub + 2) * 2.0 ** -24 * (distance.max() + 1)).all()
    x = torch.matmul(q.double(), q_proj.double()) * scale.double()[:, None, None]
    for sampled in (False, True):
        extra = (codes, n, 12) if sampled else ()
        q_low, lut, _ = kernels.query_lut(q, q_proj, scale, books, *extra)
        assert (q_low.double() - x).abs().max() <= 2.0 ** -23 * (D + 1) * 4 * x.abs().max()
        table = (q_low.double().view(1, H, Q, S, 1, sub) * books.double()[None, :, None]).sum(-1)
        size = (q_low.double().abs().view(1, H, Q, S, 1, sub) * books.double().abs()[None, :, None]).sum(-1)
        assert ((lut.double() - table).abs() <= sub * 2.0 ** -23 * size + 1e-30).all()
        torch.randn(1 << 20, device=device).softmax(0)  # (another kernel's shared memory)
        again = kernels.query_lut(q, q_proj, scale, books, *extra)
        assert torch.equal(again[0], q_low) and torch.equal(again[1], lut)
