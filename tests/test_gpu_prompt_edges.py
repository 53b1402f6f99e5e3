"""Prompt attention: empty caches, masks at every width and alignment, and the accuracy of few rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .cache4_reference import attend
from .test_gpu_cache4 import close
from .test_gpu_prompt_attention import check, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Q", [1, 4])
def test_packed_tokens_over_no_key_are_zero(device, Q):
    """n_keys 0: nothing is seen, whatever the cache's rows and the given lengths hold."""
    from sva_amd import kernels

    ones = lambda *s: torch.ones(*s, device=device)  # noqa: E731
    zero = torch.zeros(1, dtype=torch.int64, device=device)
    for where in ({}, {"seq_offsets": zero, "seq_lens": zero}, {"seq_offsets": zero, "seq_lens": zero + 5}):
        got = kernels.prompt_attention(ones(2, Q + 2, 64), ones(1, 9, 64), ones(1, 9, 64), 0, 1.0, q_offsets=zero + 1,
                                       q_lens=zero + Q, max_q=Q, out=ones(2, Q + 2, 64) * 5, **where)
        assert (got[:, 1:Q + 1] == 0).all() and (got[:, 0] == 5).all() and (got[:, -1] == 5).all()
    two = torch.zeros(2, dtype=torch.int64, device=device)
    got = kernels.prompt_attention(ones(2, 4, 64), ones(1, 0, 64), ones(1, 0, 64), 0, 1.0, seq_offsets=two,
                                   seq_lens=two, q_offsets=torch.tensor([0, 3], device=device), q_lens=two + 1,
                                   max_q=1, out=ones(2, 4, 64) * 5)
    assert (got[:, [0, 3]] == 0).all() and (got[:, [1, 2]] == 5).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.float32, 128),
                                     (torch.bfloat16, 256), (torch.float16, 256), (torch.float32, 256),
                                     (torch.bfloat16, 80), (torch.float16, 17), (torch.float32, 200),
                                     (torch.bfloat16, 64)])
@pytest.mark.parametrize("odd", [False, True])  # rows at odd addresses
@pytest.mark.parametrize("Q,N", [(1, 300), (67, 130), (9, 1200)])
def test_masks_at_every_width(device, dtype, D, odd, Q, N):
    from sva_amd import kernels

    rng = np.random.default_rng(D + Q)
    H, G = 4, 2
    q, k, v = (normal(rng, s, dtype, device) for s in ((1, H, Q, D), (G, N, D), (G, N, D)))
    if odd:
        q, k, v = (torch.empty(1 + x.numel(), device=device, dtype=dtype)[1:].view(x.shape).copy_(x)
                   for x in (q, k, v))
    allowed = rng.random((Q, N)) < 0.4
    if Q > 5:
        allowed[5] = False
        allowed[4] = True
    mask = torch.from_numpy(allowed).to(device)
    low = torch.zeros(Q, N, device=device).masked_fill(~mask, torch.finfo(torch.float32).min)
    for m in (mask, low, low.to(dtype if dtype != torch.float32 else torch.bfloat16)):
        got = kernels.prompt_attention(q, k, v, N, D ** -0.5, mask=m)
        for h in range(H):
            check(got[0, h], q[0, h], k[h // 2], v[h // 2], allowed, D ** -0.5)
        if Q > 5:
            assert (got[0, :, 5] == 0).all()


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
