"""Scores so large that their last bit is far more than one: attention is finite wherever softmax attention is, within
the same bounds as for ordinary ones."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_cache4 import WEIGHTS

pytestmark = pytest.mark.gpu

D = 64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", [-2.22e38, -3e12, 1e11, 2.22e38])  # times log2 e: up to 3.2e38
@pytest.mark.parametrize("Q,n", [(2, 1500), (150, 150), (1, 1)])
def test_large_scores(device, Q, n, score, dtype):
    """Scores whose last bit is far more than one, all alike: the mean of the values that a token sees."""
    from sva_amd import kernels

    q = torch.zeros(1, 2, Q, D, device=device)
    k = torch.zeros(1, n, D, device=device)
    k[..., 0] = 6.0 * 2.0 ** 60  # (a value of the 4-bit format)
    q[..., 0] = score / (6.0 * 2.0 ** 60)
    q, k = q.to(dtype), k.to(dtype)
    g = torch.Generator(device=device).manual_seed(0)
    v = torch.randn(1, n, D, device=device, generator=g).to(dtype)
    got = kernels.prompt_attention(q, k, v, n, 1.0, out_dtype=torch.float32)
    for t in range(Q):
        want = v[0, :n - Q + 1 + t].double().mean(0)
        assert (got[0, :, t].double() - want).abs().max() <= 4.5 * (n + 16) * 2.0 ** -23, t
    data, scales = kernels.cache4_alloc(1, n, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    _, back = kernels.cache4_read(data, scales, 0, n, torch.float32)
    idx = torch.arange(n, device=device, dtype=torch.int32).expand(2 * Q, n).contiguous()
    count = (n - Q + 1 + torch.arange(Q, device=device, dtype=torch.int32)).repeat(2)
    for got in (kernels.cache4_attention(q, data, scales, n, 1.0, torch.float32),
                kernels.cache4_verify(q, data, scales, idx, count, n, 1.0, torch.float32)):
        for t in range(Q):
            want = back[0, 0, :n - Q + 1 + t].double().mean(0)
            assert (got[0, :, t].double() - want).abs().max() <= 6.0 * ((n + 16) * 2.0 ** -23 + WEIGHTS), t


@pytest.mark.parametrize("times,apart", [(0.0, 0.75), (1.25, 0.75), (1.375, 0.75), (-1.625, 0.75), (3.5, 0.75), (2048.0, 4.0), (-2048.0, 4.0)])
@pytest.mark.parametrize("Q,n,far", [(2, 3000, 1024), (70, 3000, 1024), (2, 200, 100)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_close_scores_of_any_size_keep_their_distance(device, Q, n, far, times, apart, sign):
    """Two kinds of keys whose scores of 24576 `times` lie `apart` (the last bit of 5e7 is 4), each kind in ranges of
    its own, V 1 and 0: the output is the first kind's share of the weights, as of scores near 0.  Scores, their
    difference and V are exact."""
    from sva_amd import kernels

    q = torch.zeros(1, 2, Q, D, device=device)
    q[..., 0], q[..., 32] = sign * times, sign * apart / 4
    k = torch.zeros(1, n, D, device=device)
    k[..., 0] = 24576.0  # (values of the 4-bit format, in blocks of their own)
    k[:, :far, 32] = 4.0
    v = torch.zeros(1, n, D, device=device)
    v[:, :far] = 1.0
    data, scales = kernels.cache4_alloc(1, n, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    back = kernels.cache4_read(data, scales, 0, n, torch.float32)
    assert torch.equal(back[0][0], k) and torch.equal(back[1][0], v)
    got = [kernels.prompt_attention(q, k, v, n, sign), kernels.cache4_attention(q, data, scales, n, sign)]
    seen = (n - Q + 1 + torch.arange(Q, device=device, dtype=torch.float64))[:, None]
    weight = torch.tensor(apart, device=device, dtype=torch.float64).exp()
    want = far * weight / (far * weight + seen - far)
    for x in got:
        # sums of n weights, two exponentials and a quotient, and (4 bits) weights of two terms
        assert (x[0].double() - want).abs().max() <= (n + 16) * 2.0 ** -24 + WEIGHTS
