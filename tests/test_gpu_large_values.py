"""Attention of values near the type's largest: finite wherever softmax attention is, within the same bounds as
ordinary values."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .cache4_reference import attend
from .test_gpu_cache4 import close, decoded

pytestmark = pytest.mark.gpu

N, D = 1500, 64


def inputs(device, kind, size, Q=2, H=3, n=N):
    """Rising scores (the reference moves late: weights of up to 2^16 of the first ones), or all alike; V of one sign,
    up to `size` ("late": in the last rows alone), small beside it in the second half of the elements."""
    rng = np.random.default_rng(17)
    q = rng.standard_normal((1, H, Q, D)) * 0.05
    k = rng.standard_normal((1, n, D)) * 0.05
    q[..., 0], k[..., 0] = 1.0, np.linspace(0, 40, n) if kind == "rising" else 0.0
    v = np.abs(rng.uniform(0.5, 1, (1, n, D))) * size
    if kind == "late":
        v[:, :-n // 4] /= size
    v[..., 32:] = rng.standard_normal((1, n, 32))
    return [torch.from_numpy(x.astype(np.float32)).to(device) for x in (q, k, v)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [200, N, 6000])  # one range, six, 24
@pytest.mark.parametrize("kind,size", [("rising", 1e36), ("rising", 3e38), ("alike", 3e38), ("late", 3e38),
                                       ("alike", 1e-36)])
def test_cache4_attention(device, kind, size, dtype, n):
    from sva_amd import kernels

    q, k, v = inputs(device, kind, size, n=n)
    q = q.to(dtype)
    data, scales = kernels.cache4_alloc(1, n, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    K, V = decoded(data, scales)
    got = kernels.cache4_attention(q, data, scales, n, 1.0, torch.float32)
    allowed = np.arange(n) <= n - 2 + np.arange(2)[:, None]
    for h in range(3):
        x = q[0, h].double().cpu().numpy()
        ref, bound = attend(x, K[0], V[0], allowed, 1.0)
        scale, _ = attend(x, K[0], np.abs(V[0]), allowed, 1.0)
        # (1e-36: products below the smallest normal number, each off by at most that)
        close(got[0, h], ref, bound + n * 2.0 ** -126, scale=scale)


@pytest.mark.parametrize("kind,size", [("rising", 3e38), ("alike", 3e38), ("late", 3e38), ("alike", 1e36)])
def test_cache4_verify(device, kind, size):
    from sva_amd import kernels

    q, k, v = inputs(device, kind, size, Q=1)
    data, scales = kernels.cache4_alloc(1, N, D, device)
    kernels.cache4_write(k, v, data, scales, 0)
    K, V = decoded(data, scales)
    idx = torch.arange(N, device=device, dtype=torch.int32).expand(3, N).contiguous()
    got = kernels.cache4_verify(q, data, scales, idx, torch.full((3,), N, device=device, dtype=torch.int32), N, 1.0)
    for h in range(3):
        ref, bound = attend(q[0, h].double().cpu().numpy(), K[0], V[0], np.ones((1, N), bool), 1.0)
        close(got[0, h], ref, 2 * bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Q,n", [(2, N), (2, 200), (150, 150)])
@pytest.mark.parametrize("kind,size", [("rising", 1e36), ("rising", 3e38), ("alike", 3e38), ("late", 3e38)])
def test_prompt_attention(device, kind, size, Q, n, dtype):
    from sva_amd import kernels

    q, k, v = (x.to(dtype) for x in inputs(device, kind, size, Q=Q, n=n))
    got = kernels.prompt_attention(q, k, v, n, 1.0, out_dtype=torch.float32)
    allowed = np.arange(n) <= n - Q + np.arange(Q)[:, None]
    for h in range(3):
        x, K, V = (t.double().cpu().numpy() for t in (q[0, h], k[0], v[0]))
        ref, bound = attend(x, K, V, allowed, 1.0)
        scale, _ = attend(x, K, np.abs(V), allowed, 1.0)
        weights = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22
        close(got[0, h], ref, bound, weights=weights, scale=scale)
