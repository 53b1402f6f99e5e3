"""The paged cache's and the sampler's entry points refuse what they cannot take, before any device work; the tests'
references against themselves."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from .paged_reference import Holder, sample


def _kernels():
    from sva_amd import kernels

    return kernels


def test_reference_holder():
    h = Holder(3, 4, 6, 16)
    assert h.reserve([20, 0, 0]) == ([0, 0, 0], [(-1, -1)] * 3) and h.held[0] == [0, 1]
    h.fork([0, 0, 0])
    assert h.refs() == [3, 3, 0, 0, 0, 0]
    assert h.reserve([1, 0, 1]) == ([20, 20, 20], [(1, 2), (-1, -1), (1, 3)])
    assert h.held == [[0, 2], [0, 1], [0, 3]] and h.refs() == [3, 1, 1, 1, 0, 0]
    assert h.reserve([60, 1, 1]) == ([-1, 20, 21], [(-1, -1)] * 3)  # the table, not the pool, is too short
    assert h.reserve([0, 27, 1]) == ([21, 21, 22], [(-1, -1)] * 3) and h.held[1] == [0, 1, 4]
    h.fork([-1, 1, 7])
    assert h.lens[0] == 0


def test_reference_sampler():
    x = np.log(np.array([0.1, 0.4, 0.1, 0.3, 0.1]))
    assert [sample(x, u) for u in (0.0, 0.05, 0.15, 0.55, 0.65, 0.95)] == [0, 0, 1, 2, 3, 4]
    assert [sample(x, u, top_k=3) for u in (0.0, 0.2, 0.9)] == [0, 1, 3]          # the lowest of three ties
    assert [sample(x, u, top_p=0.5) for u in (0.0, 0.9)] == [1, 3]
    assert [sample(x, u, min_p=0.5) for u in (0.5, 0.6)] == [1, 3]
    assert sample(x, 0.9, temperature=0.0) == 1 and sample(np.full(3, -np.inf), 0.5) == -1


def _bad(calls):
    for i, call in enumerate(calls):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")


def test_pages_refuse():
    k = _kernels()
    pool = k.pages_alloc(4, 2, 16, 64, "cpu", torch.float32)
    kv, q = torch.zeros(1, 2, 3, 64), torch.zeros(1, 4, 1, 64)
    tables, lens, refs = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    pair = torch.zeros(3, dtype=torch.int32)
    _bad([
        lambda: k.pages_alloc(0, 2, 16, 64, "cpu"), lambda: k.pages_alloc(4, 2, 8, 64, "cpu"),
        lambda: k.pages_alloc(4, 2, 24, 64, "cpu"), lambda: k.pages_alloc(4, 2, 2048, 64, "cpu"),
        lambda: k.pages_alloc(4, 2, 16, 60, "cpu"), lambda: k.pages_alloc(4, 2, 16, 264, "cpu"),
        lambda: k.pages_alloc(4, 2, 16, 64, "cpu", layers=0), lambda: k.pages_alloc(4, 2, 16, 64, "cpu", torch.float64),
        lambda: k.paged_write(kv[..., :32], kv[..., :32], pool, tables, 0),
        lambda: k.paged_write(kv.half(), kv.half(), pool, tables, 0),
        lambda: k.paged_write(kv, kv[:, :1], pool, tables, 0),
        lambda: k.paged_write(kv, kv, pool[:, :1], tables, 0),
        lambda: k.paged_write(kv, kv, pool.transpose(2, 3), tables, 0),
        lambda: k.paged_write(kv, kv, pool[..., :32], tables, 0),
        lambda: k.paged_write(kv, kv, pool, tables.long(), 0),
        lambda: k.paged_write(kv, kv, pool, tables.repeat(2, 1), 0),
        lambda: k.paged_write(kv, kv, pool, tables, [0, 1]),
        lambda: k.paged_write(kv, kv, pool, tables, lens.int()),
        lambda: k.paged_read(pool, tables, 0, -1),
        lambda: k.paged_read(pool[0], tables, 0, 3),
        lambda: k.paged_attention(q[..., :32], pool, tables, lens, 1.0),
        lambda: k.paged_attention(q.half(), pool, tables, lens, 1.0),
        lambda: k.paged_attention(torch.zeros(1, 3, 1, 64), pool, tables, lens, 1.0),
        lambda: k.paged_attention(q, pool, tables, lens.int(), 1.0),
        lambda: k.paged_attention(q, pool, tables, lens.repeat(2), 1.0),
        lambda: k.paged_attention(q.repeat(2, 1, 1, 1), pool, tables, lens, 1.0),
        lambda: k.paged_attention(q, pool, tables.t(), lens, 1.0),
        lambda: k.pages_reserve(tables, lens, refs.long(), 1, 16), lambda: k.pages_reserve(tables, lens, refs, 1, 10),
        lambda: k.pages_reserve(tables, lens, refs, lens.int(), 16), lambda: k.pages_reserve(tables[0], lens, refs, 1, 16),
        lambda: k.pages_reserve(tables.expand(2, 4), lens.repeat(2), refs, 1, 16),
        lambda: k.pages_fork(tables, lens, refs, lens.int(), 16), lambda: k.pages_fork(tables, lens, refs, lens.repeat(2), 16),
        lambda: k.pages_fork(tables, lens, refs[::2], lens, 16), lambda: k.pages_compact(tables, refs[None]),
        lambda: k.pages_copy(pool[0], pair, pair), lambda: k.pages_copy(pool, pair, pair[:2]),
        lambda: k.pages_copy(pool, pair.long(), pair.long()), lambda: k.pages_copy(pool[None][:0], pair, pair),
    ])
    for call in (lambda: k.paged_write(kv, kv, pool, tables, lens), lambda: k.paged_read(pool, tables, lens, 3),
                 lambda: k.paged_attention(q, pool, tables, lens, 1.0), lambda: k.pages_reserve(tables, lens, refs, 1, 16),
                 lambda: k.pages_fork(tables, lens, refs, lens, 16), lambda: k.pages_compact(tables, refs),
                 lambda: k.pages_copy(pool, pair, pair)):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()
    grad = torch.zeros(1, 4, 1, 64, requires_grad=True)
    for call in (lambda: k.paged_attention(grad, pool, tables, lens, 1.0),
                 lambda: k.paged_write(grad[:, :2], grad[:, :2], pool, tables, lens)):
        with pytest.raises(RuntimeError, match="inference only"):
            call()


def test_sampler_refuses():
    k = _kernels()
    x, u = torch.zeros(3, 10), torch.zeros(3)
    _bad([
        lambda: k.sample_tokens(x[0], u), lambda: k.sample_tokens(x, u[:2]), lambda: k.sample_tokens(x, u.double()),
        lambda: k.sample_tokens(x.double(), u), lambda: k.sample_tokens(x[:, :0], u),
        lambda: k.sample_tokens(torch.zeros(1, 1).expand(3, (1 << 20) + 1), u),
        lambda: k.sample_tokens(x, u, temperature=-0.1), lambda: k.sample_tokens(x, u, top_k=-1),
        lambda: k.sample_tokens(x, u, top_p=1.1), lambda: k.sample_tokens(x, u, top_p=-0.1),
        lambda: k.sample_tokens(x, u, min_p=1.5), lambda: k.sample_tokens(x, u, temperature=float("nan")),
        lambda: k.sample_tokens(x, u, top_k=u), lambda: k.sample_tokens(x, u, top_p=u.double()),
        lambda: k.sample_tokens(x, u, min_p=u[:1]),
    ])
    with pytest.raises(RuntimeError, match="ROCm"):
        k.sample_tokens(x, u)
    with pytest.raises(RuntimeError, match="inference only"):
        k.sample_tokens(x.clone().requires_grad_(), u)


def test_c_entries_refuse():
    from sva_amd import _lib

    lib = _lib.lib()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)  # never dereferenced: the arguments are refused first
    one = ctypes.c_float(1.0)

    def refused(name, args, text, status=1):
        rc = getattr(lib, name)(*args)
        assert rc == status and text in lib.sva_last_error().decode(), (name, rc, lib.sva_last_error())

    def with_(args, changes):
        args = list(args)
        for at, v in changes.items():
            args[at] = v
        return args

    write = [p, p, 1, 64, 64, 64, 1, 1, 1, 64, p, p, 4, 2 * 16 * 64, 16, p, 4, 4, None]
    for changes, text in (({0: None}, "null"), ({10: None}, "null"), ({2: 3}, "dtype"), ({9: 60}, "head_dim"),
                          ({9: 264}, "head_dim"), ({14: 24}, "rows a page"), ({14: 8}, "rows a page"), ({11: odd}, "16-byte"),
                          ({13: 2 * 16 * 64 - 8}, "16-byte"), ({12: 0}, "sizes"), ({6: 0}, "sizes")):
        refused("sva_paged_write", with_(write, changes), text)
    refused("sva_paged_write", with_(write, {6: 1 << 30, 8: 4, 12: 4, 13: 2 * 4 * 16 * 64}), "sequences", 3)
    read = [p, 4, 2 * 16 * 64, 16, p, 4, 4, p, 1, 1, 1, 64, p, p, 1, 64, 64, 64, None]
    refused("sva_paged_read", with_(read, {12: odd}), "16-byte")
    attend = [p, 1, 64, 64, 64, p, 4, 2 * 16 * 64, 16, p, 4, 4000, p, 64000, 1, 1, 1, 1, 64, one, p, 1, 64, 64, 64, p, 1 << 20, None]
    for changes, text in (({0: None}, "null"), ({12: None}, "null"), ({1: 5}, "dtype"), ({21: -1}, "dtype"), ({15: 3, 16: 2}, "sizes"),
                          ({18: 4}, "head_dim"), ({8: 17}, "rows a page"), ({5: odd}, "16-byte"), ({25: None}, "workspace"),
                          ({26: 10}, "workspace"), ({17: 0}, "sizes"), ({11: 1 << 30, 13: 1 << 40}, "too many")):
        refused("sva_paged_attention", with_(attend, changes), text)
    reserve = [p, 4, 4, p, 1, p, 40000, 16, None, 1, p, p, p, p, 1 << 20, None]
    for changes, text in (({0: None}, "null"), ({2: 0}, "sizes"), ({7: 0}, "rows a page"), ({13: odd}, "workspace"), ({14: 8}, "workspace")):
        refused("sva_pages_reserve", with_(reserve, changes), text)
    fork = [p, 40000, 40000, p, 1, p, 4, 16, p, p, 1 << 20, None]
    for changes, text in (({8: None}, "null"), ({4: 0}, "sizes"), ({7: 100}, "rows a page"), ({10: 8}, "workspace")):
        refused("sva_pages_fork", with_(fork, changes), text)
    compact = [p, 4, 4, 1, p, 4, p, p, p, p, 1 << 20, None]
    for changes, text in (({8: None}, "null"), ({5: 0}, "sizes"), ({10: 8}, "workspace")):
        refused("sva_pages_compact", with_(compact, changes), text)
    copy = [p, 4, 4096, 1, 0, 4096, p, p, 1, None]
    for changes, text in (({6: None}, "null"), ({0: odd}, "16-byte"), ({5: 4100}, "16-byte"), ({2: 2048}, "16-byte"), ({8: 0}, "sizes")):
        refused("sva_pages_copy", with_(copy, changes), text)
    draw = [p, 0, 10, 1, 10, p, None, one, None, 0, None, one, None, one, p, None]
    for changes, text in (({0: None}, "null"), ({5: None}, "null"), ({1: 3}, "dtype"), ({4: 0}, "sizes"), ({3: 0}, "sizes")):
        refused("sva_sample_tokens", with_(draw, changes), text)
    refused("sva_sample_tokens", with_(draw, {4: (1 << 20) + 1}), "tokens", 3)


def test_workspaces():
    lib = _kernels().lib()
    size = lib.sva_paged_attention_workspace_bytes
    assert size(0, 9, 3, 1, 64, 1, 100000) == size(1, 9, 2, 1, 64, 1, 100000) == size(1, 9, 3, 1, 64, 1, 256) == 0
    assert 256 < size(1, 9, 3, 1, 64, 0, 100000) < 1 << 24
    assert lib.sva_pages_reserve_workspace_bytes(3, 10) == 0 and lib.sva_pages_reserve_workspace_bytes(3, 10000) >= 3 * 16 + 40000
    assert lib.sva_pages_reserve_workspace_bytes(2000, 10) >= 2000 * 16 + 40 and lib.sva_pages_fork_workspace_bytes(3, 10) == 0
    assert lib.sva_pages_fork_workspace_bytes(3, 10000) >= 3 * 8 + 120000 and lib.sva_pages_compact_workspace_bytes(7) >= 28


@pytest.mark.parametrize("keep,refs,lens", [(40, [1, 2, 2, 0], [40, 0, 40]), (33, [1, 2, 2, 0], [33, 0, 33]),
                                            (32, [1, 2, 0, 0], [32, 0, 32]), (20, [1, 2, 0, 0], [20, 0, 20]), (0, [0, 0, 0, 0], [0, 0, 0])])
def test_crop_of_a_batch_with_a_freed_sequence(keep, refs, lens):
    """A sequence that kernels.pages_fork freed names no page: a crop counts none for it and leaves its length."""
    from transformers import LlamaConfig

    from sva_amd import PagedCache

    cache = PagedCache(LlamaConfig(hidden_size=64, num_attention_heads=1, num_key_value_heads=1, num_hidden_layers=1))
    cache._begin(3, torch.zeros(3, 1, 45, 64))
    cache.pool = torch.zeros(1, 4, 2, 1, 16, 64)
    cache.tables = torch.tensor([[0, 1, 2, -1], [-1, -1, -1, -1], [0, 1, 2, -1]], dtype=torch.int32)
    cache.tables[2, 0] = 2 ** 31 - 1  # (an entry outside the pool names no page either)
    cache.refs = torch.tensor([1, 2, 2, 0], dtype=torch.int32)
    cache.lens = torch.tensor([45, 0, 45])
    cache.length = cache.layers[0].length = 45
    cache.crop(keep - 45)
    assert cache.refs.tolist() == refs and cache.lens.tolist() == lens and cache.get_seq_length() == keep
    held = -(-keep // 16)
    assert (cache.tables[:, held:] == -1).all() and (held == 0 or cache.tables[0, :held].tolist() == [0, 1, 2][:held])


def test_crop_of_a_cache_without_pages():
    from transformers import LlamaConfig

    from sva_amd import PagedCache

    cache = PagedCache(LlamaConfig(hidden_size=64, num_attention_heads=1, num_key_value_heads=1, num_hidden_layers=1))
    cache._begin(1, torch.zeros(1, 1, 20, 64))
    cache.tables = torch.full((1, 2), -1, dtype=torch.int32)
    cache.length = cache.layers[0].length = 20
    cache.crop(-20)
    assert cache.length == 0 and cache.lens.tolist() == [0]
