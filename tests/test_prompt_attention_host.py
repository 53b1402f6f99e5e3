"""Dense prompt attention refuses what it cannot take, before any device work."""

from __future__ import annotations

import ctypes

import pytest
import torch


def _kernels():
    from sva_amd import kernels

    return kernels


def test_wrapper_refuses():
    k = _kernels()
    q, kv = torch.zeros(1, 4, 3, 64), torch.zeros(2, 8, 64)
    two, packed = torch.zeros(2, dtype=torch.int64), torch.zeros(4, 10, 64)
    call = lambda q=q, keys=kv, values=kv, n=8, **kw: k.prompt_attention(q, keys, values, n, 1.0, **kw)  # noqa: E731
    bad = [
        dict(q=q[0, 0]), dict(q=torch.zeros(1, 3, 3, 64)), dict(q=q.half()), dict(keys=kv[..., :32], values=kv[..., :32]),
        dict(values=kv[:, :4]), dict(values=kv.half()), dict(n=9), dict(q=q.expand(2, 4, 3, 64)),
        dict(q=torch.zeros(1, 4, 3, 264), keys=torch.zeros(2, 8, 264), values=torch.zeros(2, 8, 264)),
        dict(seq_lens=two[:1]), dict(q_lens=two[:1]), dict(out=torch.zeros(1, 4, 3, 32)),
        dict(q=q[0], out=torch.zeros(1, 4, 3, 64)),
        dict(q=packed, q_offsets=two, q_lens=two, max_q=0, seq_offsets=two, seq_lens=two),
        dict(q=packed[None], q_offsets=two, q_lens=two, max_q=3, seq_offsets=two, seq_lens=two),
        dict(q=packed, q_offsets=two, q_lens=two, max_q=3),                       # two sequences of keys, not told apart
        dict(q=packed, q_offsets=two, q_lens=two, max_q=3, seq_offsets=two, seq_lens=two, mask=torch.zeros(3, 8)),
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
            pytest.fail(f"taken: { {a: tuple(b.shape) if isinstance(b, torch.Tensor) else b for a, b in kw.items()} }")
    with pytest.raises(RuntimeError, match="ROCm"):
        call()
    for mask in (torch.zeros(2, 8), torch.zeros(3, 7), torch.zeros(2, 1, 3, 8), torch.zeros(1, 4, 3, 8), torch.zeros(8)):
        with pytest.raises(ValueError):
            k._prompt_mask(mask, 1, 3, 8)
    with pytest.raises(TypeError):
        k._prompt_mask(torch.zeros(3, 8, dtype=torch.int32), 1, 3, 8)
    m, kind, seq, tok = k._prompt_mask(torch.zeros(1, 1, 5, 9).expand(1, 4, 5, 9), 3, 3, 8)
    assert tuple(m.shape) == (1, 3, 8) and (kind, seq, tok) == (1, 0, 9)


def test_c_entry_point_refuses():
    from sva_amd import _lib

    lib = _lib.lib()
    p, one = ctypes.c_void_p(256), ctypes.c_float(1.0)  # never dereferenced: the arguments are refused first

    def call(q=p, dt=1, qo=None, ql=None, q_rows=0, so=None, sl=None, n_keys=100, n_seq=1, H=4, G=2, Q=8, D=64, mask=None,
             mt=0, ws=p, ws_bytes=1 << 30, odt=1, kv_rows=100):
        return lib.sva_prompt_attention(q, dt, 0, 0, 0, qo, ql, q_rows, p, p, 0, 0, kv_rows, so, sl, n_keys, n_seq, H, G,
                                        Q, D, one, mask, mt, 0, 0, p, odt, 0, 0, 0, ws, ws_bytes, None)

    bad = [dict(q=None), dict(dt=3), dict(odt=-1), dict(qo=p), dict(so=p), dict(n_seq=2), dict(H=5), dict(D=0),
           dict(D=257), dict(Q=0), dict(n_keys=0), dict(n_keys=1 << 31), dict(mask=p), dict(mt=1), dict(mask=p, mt=5),
           dict(qo=p, ql=p, q_rows=9, mask=p, mt=1), dict(qo=p, ql=p, q_rows=0), dict(ws=None), dict(kv_rows=0),
           dict(Q=1 << 30), dict(Q=1, n_keys=1 << 20, ws_bytes=256)]
    got = [call(**kw) for kw in bad]
    assert got == [1] * len(bad), got
    assert "workspace" in lib.sva_last_error().decode()
    size = lib.sva_prompt_attention_workspace_bytes
    assert size(1, 9, 3, 8192, 64, 8192) == 256 and size(1, 9, 3, 1, 64, 1 << 20) > 256 and size(1, 9, 2, 1, 64, 9) == 0


def test_gradients_are_refused():
    k = _kernels()
    q = torch.zeros(1, 4, 3, 64, requires_grad=True)
    with pytest.raises(RuntimeError, match="inference only"):
        k._inference_only("prompt_attention", q)
    with torch.no_grad():
        k._inference_only("prompt_attention", q)
