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
