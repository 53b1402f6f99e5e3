"""Prompt attention: the accuracy of few rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .cache4_reference import attend
from .test_gpu_cache4 import close
from .test_gpu_prompt_attention import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,H,G,Q,D,masked,odd", [
    ([3000, 1, 700], 9, 3, 1, 64, False, False), ([5000], 4, 2, 1, 128, False, False),
    ([900], 8, 1, 2, 256, False, False), ([1300], 16, 2, 2, 64, True, False), ([400], 3, 1, 1, 80, True, False),
    ([700], 4, 2, 1, 128, False, True)])
def test_weights_of_few_rows_keep_their_bits(device, dtype, lens, H, G, Q, D, masked, odd):
    """At most 16 rows (token x head of a KV group) a sequence: outputs in fp32 are within 2^-17 of the weights' sums,
    as the 4-bit cache's attention, where one 16-bit term a weight leaves 2^-9 (fp16: 2^-12)."""
    from sva_amd import kernels

    rng = np.random.default_rng(sum(lens) + D)
    n, rows = len(lens), sum(lens)
    q, k, v = (normal(rng, s, dtype, device) for s in ((n, H, Q, D), (G, rows, D), (G, rows, D)))
    if odd:
        k = torch.empty(1 + k.numel(), device=device, dtype=dtype)[1:].view(k.shape).copy_(k)
        v = v.clone()
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)])[:-1], device=device)
    allowed = rng.random((n, Q, max(lens))) < 0.5 if masked else None
    mask = torch.from_numpy(allowed).to(device) if masked else None
    got = kernels.prompt_attention(q, k, v, max(lens), D ** -0.5, mask=mask, seq_offsets=off,
                                   seq_lens=torch.tensor(lens, device=device), out_dtype=torch.float32)
    for b, m in enumerate(lens):
        see = allowed[b, :, :m] if masked else np.arange(m) <= m - Q + np.arange(Q)[:, None]
        for h in range(H):
            g, at = h // (H // G), slice(int(off[b]), int(off[b]) + m)
            x, K, V = (t.double().cpu().numpy() for t in (q[b, h], k[g, at], v[g, at]))
            ref, bound = attend(x, K, V, see, D ** -0.5)
            size, _ = attend(x, K, np.abs(V), see, D ** -0.5)
            # (fp16: the second term of a weight below 2^-2 of a reference kept at 2^8 is subnormal: 2^-25 of 2^8)
            close(got[b, h], ref, bound + (m * 2.0 ** -33 * np.abs(V).max() if dtype == torch.float16 else 0.0),
                  scale=size)
