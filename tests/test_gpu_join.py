"""Attention over several ranges of keys: what is not finite reaches every token that sees it, in whichever range it
lies and however far the range's scores lie below the others, as in one range."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

N, D = 2048, 64  # eight ranges of 256 keys and more


def rows(device, far, Q, H, G, seed=0):
    """q, keys, values: scores of about 1, those of keys 512 .. 767 by `far` lower (in units of log 2 1.44)."""
    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn(1, H, Q, D, device=device, generator=g) * 0.1
    q[..., 0] = 8.0
    k = torch.randn(G, N, D, device=device, generator=g)
    k[..., 0] = 0.0
    k[:, 512:768, 0] = -far
    return q, k, torch.randn(G, N, D, device=device, generator=g)


# 4 items: each takes a part of a workgroup's join; 1200: a wave each
@pytest.mark.parametrize("Q", [1, 300])
def test_cache4_whole_range_of_nan_keys(device, Q):
    from sva_amd import kernels

    q, k, v = rows(device, 0.0, Q, 4, 2)
    k[1, 512:768, 40] = float("nan")
    data, scales = kernels.cache4_alloc(2, N, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    got = kernels.cache4_attention(q, data, scales, N, 1.0)
    assert torch.isfinite(got[:, :2]).all()
    assert torch.isnan(got[:, 2:]).all()


@pytest.mark.parametrize("Q", [1, 300])
def test_cache4_nan_value_in_a_far_range(device, Q):
    from sva_amd import kernels

    q, k, v = rows(device, 48.0, Q, 4, 2)  # scores of -384: weights of 2^-554
    data, scales = kernels.cache4_alloc(2, N, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    clean = kernels.cache4_attention(q, data, scales, N, 1.0)
    v[1, 600, 40] = float("nan")
    kernels.cache4_write(k, v, data, scales, 0)
    got = kernels.cache4_attention(q, data, scales, N, 1.0)
    assert torch.isnan(got[:, 2:, :, 32:]).all()
    assert torch.equal(got[:, :2], clean[:, :2]) and torch.equal(got[:, 2:, :, :32], clean[:, 2:, :, :32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Q", [1, 300])
def test_prompt_values_not_finite_in_a_far_range(device, Q, dtype):
    from sva_amd import kernels

    q, k, v = (x.to(dtype) for x in rows(device, 48.0, Q, 4, 2))
    clean = kernels.prompt_attention(q, k, v, N, 1.0).float()
    v[1, 600, 40], v[1, 601, 41] = float("nan"), float("inf")
    k[0, 700, 3] = float("nan")
    got = kernels.prompt_attention(q, k, v, N, 1.0).float()
    assert torch.isnan(got[:, :2]).all()  # a score that is NaN
    # (a weight of 2^-554 is 0 in 32 bits: 0 times an infinity is NaN)
    assert not torch.isfinite(got[:, 2:, :, 40:42]).any()
    rest = torch.ones(D, dtype=torch.bool, device=device)
    rest[40:42] = False
    # the range done again has weights of 0 all the same: the other elements are the same sums
    assert torch.equal(got[:, 2:][..., rest], clean[:, 2:][..., rest])


def test_a_range_without_a_key_for_a_row_stays_out(device):
    """A masked range holding NaN and infinities, and ranges that no token sees."""
    from sva_amd import kernels

    q, k, v = rows(device, 0.0, 300, 4, 2)
    mask = torch.ones(300, N, dtype=torch.bool, device=device)
    mask[:, 512:768] = False
    mask[7] = False
    clean = kernels.prompt_attention(q, k, v, N, 1.0, mask=mask)
    k[:, 512:768], v[:, 512:768] = float("nan"), float("inf")
    got = kernels.prompt_attention(q, k, v, N, 1.0, mask=mask)
    assert torch.isfinite(got).all() and (got[:, :, 7] == 0).all()
    # (rows done again: sums of 2048 terms in another order, values up to 4.5)
    assert (got - clean).abs().max() <= 4.5 * 2 * (N + 80) * 2.0 ** -24
