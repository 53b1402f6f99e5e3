"""The key catalog of a 4-bit cache belongs to that cache: caches that are decoded in turn, cut, emptied or copied go on
exactly as one that is decoded alone (the shortlist and the budget are far below the length, so a row of another
cache's catalog would choose other keys)."""

from __future__ import annotations

import copy

import pytest
import torch

from sva import patch_llama_attention

from .test_gpu_llama import make_tiny_bundle, make_tiny_model

pytestmark = pytest.mark.gpu

N = 70  # a prompt's tokens


def setup(device):
    model = make_tiny_model(device, hidden=128, heads=4, kv_heads=2, seed=3)
    return model, make_tiny_bundle(heads=4, head_dim=32, shortlist=12, budget=4)


def tokens(device, seed):
    return torch.randint(0, 64, (1, 100), generator=torch.Generator().manual_seed(seed)).to(device)


@torch.no_grad()
def feed(model, cache, ids, a, b):
    """Logits of tokens a .. b - 1 of ids in one call over what the cache holds."""
    return model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True,
                 position_ids=torch.arange(a, b, device=ids.device)[None]).logits


def alone(model, ids, steps=8):
    from sva_amd import FourBitCache

    cache = FourBitCache()
    return cache, [feed(model, cache, ids, 0, N)] + [feed(model, cache, ids, N + i, N + i + 1) for i in range(steps)]


@pytest.mark.parametrize("prompt", ["dense", "summon"])
def test_caches_of_one_length_decoded_in_turn(device, prompt):
    from sva_amd import FourBitCache

    model, bundle = setup(device)
    a, b = tokens(device, 1), tokens(device, 2)
    with patch_llama_attention(model, bundle, prompt_attention=prompt):
        want_a, want_b = alone(model, a)[1], alone(model, b)[1]
        assert not torch.equal(want_a[1], want_b[1])
        ca, cb = FourBitCache(), FourBitCache()
        assert torch.equal(feed(model, ca, a, 0, N), want_a[0])
        assert torch.equal(feed(model, cb, b, 0, N), want_b[0])
        for i in range(8):
            assert torch.equal(feed(model, ca, a, N + i, N + i + 1), want_a[1 + i]), i
            if i != 3:  # (and of lengths that differ)
                assert torch.equal(feed(model, cb, b, N + i - (i > 3), N + i + 1 - (i > 3)), want_b[1 + i - (i > 3)]), i


def test_a_cut_cache_goes_on_from_the_rows_that_are_left(device):
    model, bundle = setup(device)
    a, b = tokens(device, 1), tokens(device, 2)
    with patch_llama_attention(model, bundle):
        cache, want = alone(model, a)
        for layer in cache.layers:
            layer.crop(-6)
        for i in range(2, 8):
            assert torch.equal(feed(model, cache, a, N + i, N + i + 1), want[1 + i]), i
        # other tokens behind the cut, then the first ones again
        cache.crop(-8)
        feed(model, cache, b, N, N + 8)
        cache.crop(-8)
        for i in range(8):
            assert torch.equal(feed(model, cache, a, N + i, N + i + 1), want[1 + i]), i
        cache.reset()
        assert torch.equal(feed(model, cache, a, 0, N), want[0])
        assert torch.equal(feed(model, cache, a, N, N + 1), want[1])


def test_a_copied_cache_and_a_catalog_that_starts_over(device):
    model, bundle = setup(device)
    a, b = tokens(device, 1), tokens(device, 2)
    with patch_llama_attention(model, bundle) as handle:
        cache, want = alone(model, a, steps=1)
        twin = copy.deepcopy(cache)
        feed(model, cache, b, N + 1, N + 2)
        assert torch.equal(feed(model, twin, a, N + 1, N + 2), alone(model, a, steps=2)[1][2])
        # a 16-bit cache in between does not touch the catalog, nor the other way round
        cache, want = alone(model, a)
        cache.crop(-1)
        with torch.no_grad():
            plain = model(input_ids=b[:, :N], use_cache=True)
        first = model.model.layers[0].self_attn
        assert first._cached_key_len == N
        assert torch.equal(feed(model, cache, a, N + 7, N + 8), want[8])
        assert first._cached_key_len == N
        go = feed(model, plain.past_key_values, b, N, N + 1)
        with torch.no_grad():
            again = model(input_ids=b[:, :N], use_cache=True)
        assert torch.equal(feed(model, again.past_key_values, b, N, N + 1), go)
        # the catalog made again is that of the rows as they are held
        cache.crop(-1)
        handle.reset_catalogs()
        once = feed(model, cache, a, N + 7, N + 8)
        cache.crop(-1)
        handle.reset_catalogs()
        assert torch.equal(feed(model, cache, a, N + 7, N + 8), once) and torch.isfinite(once).all()


def test_rows_that_came_in_without_the_layer_enter_its_catalog(device):
    """They are encoded as they are held; the rows before them stay as they were made from the keys."""
    from sva_amd import kernels

    model, bundle = setup(device)
    a = tokens(device, 1)
    with patch_llama_attention(model, bundle):
        cache, _ = alone(model, a)
        before = [(x.catalog.k_low[:, :N + 8].clone(), x.catalog.codes[:, :N + 8].clone()) for x in cache.layers]
        g = torch.Generator(device=device).manual_seed(0)
        for layer in cache.layers:
            layer.append(*(torch.randn(1, 2, 300, 32, device=device, generator=g) for _ in range(2)))  # (it grows)
        out = feed(model, cache, a, N + 8, N + 9)
        assert torch.isfinite(out).all() and cache.get_seq_length() == N + 309
        for layer, (k_low, codes), block in zip(cache.layers, before, model.model.layers):
            at, c = slice(N + 8, N + 308), layer.catalog
            assert c.rows == N + 309
            assert torch.equal(c.k_low[:, :N + 8], k_low) and torch.equal(c.codes[:, :N + 8], codes)
            want = torch.empty_like(c.k_low[:, at]).contiguous(), torch.empty_like(c.codes[:, at]).contiguous()
            kernels.write_encode(layer.read()[0][0][:, at].contiguous(), block.self_attn.sva_k_proj,
                                 block.self_attn.sva_coarse_codebooks, *want)
            assert torch.equal(c.k_low[:, at], want[0]) and torch.equal(c.codes[:, at], want[1])
