"""The 4-bit cache's entry points refuse what they cannot take, before any device work; the tests' reference of the
format against itself."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from .cache4_reference import CODES, decode, encode


def _kernels():
    from sva_amd import kernels

    return kernels


def test_reference_format():
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.99] + [4.0] * 24])
    codes, scales = encode(x)
    assert scales.tolist() == [[127]]
    assert decode(codes, scales)[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    every = np.concatenate([CODES, -CODES, CODES, -CODES])[None]
    assert np.array_equal(decode(*encode(every)), every)


@pytest.mark.parametrize("heads,rows,dim", [(0, 4, 64), (1, 0, 64), (1, 4, 48), (1, 4, 0), (1, 4, 288)])
def test_alloc_refuses(heads, rows, dim):
    with pytest.raises(ValueError):
        _kernels().cache4_alloc(heads, rows, dim, "cpu")


def test_wrappers_refuse():
    k = _kernels()
    data, scales = k.cache4_alloc(2, 8, 64, "cpu")
    kv = torch.zeros(1, 2, 3, 64)
    q = torch.zeros(1, 4, 1, 64)
    idx, cnt = torch.zeros(4, 5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    two = torch.zeros(2, dtype=torch.int64)
    bad = [
        lambda: k.cache4_write(kv[..., :32], kv[..., :32], data, scales, 0),          # another width
        lambda: k.cache4_write(kv, kv.half(), data, scales, 0),
        lambda: k.cache4_write(kv[:, :1], kv[:, :1], data, scales, 0),                # another number of heads
        lambda: k.cache4_write(kv, kv, data[:, :, :1], scales, 0),
        lambda: k.cache4_write(kv, kv, data, scales[:, :4], 0),
        lambda: k.cache4_write(kv, kv, data.float(), scales, 0),
        lambda: k.cache4_read(data, scales[..., :1], 0, 4),
        lambda: k.cache4_attention(q[..., :32], data, scales, 8, 1.0),
        lambda: k.cache4_attention(torch.zeros(1, 3, 1, 64), data, scales, 8, 1.0),   # 3 heads over 2
        lambda: k.cache4_attention(q, data, scales, 9, 1.0),                          # more keys than rows
        lambda: k.cache4_attention(q.expand(2, 4, 1, 64), data, scales, 8, 1.0),      # two sequences, no offsets
        lambda: k.cache4_attention(q, data, scales, 8, 1.0, seq_offsets=two[:1]),
        lambda: k.cache4_attention(q, data, scales, 8, 1.0, None, two, two),
        lambda: k.cache4_attention(q, data, scales, 8, 1.0, None, two[:1].int(), two[:1].int()),
        lambda: k.cache4_attention(q[0, 0], data, scales, 8, 1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: k.cache4_write(kv, kv, data, scales, 0), lambda: k.cache4_read(data, scales, 0, 4),
                 lambda: k.cache4_attention(q, data, scales, 8, 1.0),
                 lambda: k.cache4_verify(q, data, scales, idx, cnt, 8, 1.0)):
        with pytest.raises(RuntimeError, match="ROCm"):  # well formed, but on the CPU
            call()


def test_c_entry_points_refuse():
    from sva_amd import _lib

    lib = _lib.lib()
    p, one = ctypes.c_void_p(256), ctypes.c_float(1.0)  # never dereferenced: the arguments are refused first

    def attention(ws=p, ws_bytes=1 << 30, D=64, H=4, G=2, q=p, off=None, ln=None, n_seq=1, data=p, Q=1, dt=1):
        return lib.sva_cache4_attention(q, dt, 0, 0, 0, data, p, 100, off, ln, 100, n_seq, H, G, Q, D, one, p, 1, 0, 0,
                                        0, ws, ws_bytes, None)

    def verify(D=64, B=4, idx=p, n_seq=1, dt=1):
        return lib.sva_cache4_verify(p, dt, 0, 0, 0, p, p, 100, None, None, 100, idx, p, n_seq, 4, 2, 1, D, B, one, p,
                                     1, 0, 0, 0, None)

    def write(D=64, n=3, dt=1, data=p, first=p, n_seq=1):
        return lib.sva_cache4_write(p, p, dt, 0, 0, 0, n_seq, n, 2, D, first, 0, data, p, 100, None)

    def read(D=64, n=3, dt=1, first=p, n_seq=1):
        return lib.sva_cache4_read(p, p, 100, first, 0, n_seq, n, 2, D, p, p, dt, 0, 0, 0, None)

    calls = [attention(q=None), attention(D=48), attention(D=288), attention(H=3), attention(off=p), attention(n_seq=2),
             attention(ws=None), attention(dt=3), attention(data=ctypes.c_void_p(264)), verify(D=40),
             verify(B=0), verify(idx=None), verify(n_seq=2), verify(dt=-1), write(D=33), write(n=0), write(dt=7),
             write(data=None), write(first=None, n_seq=2), read(D=0), read(n=-1), read(dt=3), read(first=None, n_seq=2)]
    assert calls == [1] * len(calls), calls
    assert attention(Q=1 << 20) == 3  # SVA_ERR_UNSUPPORTED
    big = lib.sva_cache4_attention_workspace_bytes(1, 9, 3, 1, 64, 1 << 20)
    assert big > 256 and attention(ws_bytes=16) == 1
    assert "workspace" in lib.sva_last_error().decode()
    assert lib.sva_cache4_attention_workspace_bytes(1, 9, 2, 1, 64, 100) == 0
