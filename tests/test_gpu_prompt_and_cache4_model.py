"""Dense prompts and the 4-bit cache in a patched model: prompt, cached decode and chunks together, against the same
model unpatched.  A shortlist and budget of every key make the lookup exact, so the logits may differ by fp32 rounding
alone (1e-4 of their largest; sums of at most 200 keys and 64 elements, twice 264 2^-24 each, over two layers and an
output layer of gain under ten)."""

from __future__ import annotations

import pytest
import torch

from sva import patch_llama_attention

from .test_gpu_llama import make_tiny_bundle, make_tiny_model

pytestmark = pytest.mark.gpu


def setup(device, heads=4, kv_heads=2, head_dim=32, seed=3):
    model = make_tiny_model(device, hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, seed=seed)
    return model, make_tiny_bundle(heads=heads, head_dim=head_dim, shortlist=256, budget=256)


def tokens(device, batch, n, seed=0):
    return torch.randint(0, 64, (batch, n), generator=torch.Generator().manual_seed(seed)).to(device)


def near(a, b):
    assert (a - b).abs().max() <= 1e-4 * b.abs().max()


@torch.no_grad()
def run(model, ids, cuts, cache=None, mask=None):
    """Logits of ids fed in pieces that end at `cuts`."""
    out, a = [], 0
    for b in cuts:
        r = model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True,
                  attention_mask=None if mask is None else mask[:, :b])
        cache, a = r.past_key_values, b
        out.append(r.logits)
    return torch.cat(out, 1)


@pytest.mark.parametrize("mode", ["scan", "inverted_static"])
def test_dense_prompt_equals_the_model(device, mode):
    model, bundle = setup(device)
    ids = tokens(device, 1, 90)
    cuts = [70, 71, 72, 88, 89, 90]  # a prompt, two tokens, a chunk over what is cached, two tokens
    want = run(model, ids, cuts)
    with patch_llama_attention(model, bundle, prompt_attention="dense", summon_mode=mode,
                               inverted_cells_per_subspace=8) as handle:
        got = run(model, ids, cuts)
        assert handle.stats.summary()["queries"] == 2 * 4 * 4  # layers x heads x single tokens
        first = model.model.layers[0].self_attn
        assert first._cached_key_len == 90
    near(got[:, :70], want[:, :70])
    if mode == "scan":  # (a static index looks up a part of the keys)
        near(got, want)


def test_dense_prompt_of_a_batch_and_of_a_padded_one(device):
    model, bundle = setup(device)
    ids = tokens(device, 3, 40)
    want = run(model, ids, [40])
    mask = torch.ones(3, 40, dtype=torch.long, device=device)
    mask[1, :7] = 0
    mask[2, :25] = 0
    padded = run(model, ids, [40], mask=mask)
    with patch_llama_attention(model, bundle, prompt_attention="dense"):
        near(run(model, ids, [40]), want)
        got = run(model, ids, [40], mask=mask)
    for b, pad in enumerate((0, 7, 25)):
        near(got[b, pad:], padded[b, pad:])


def test_prompt_modes_are_checked(device):
    model, bundle = setup(device)
    with pytest.raises(ValueError, match="prompt_attention"):
        patch_llama_attention(model, bundle, prompt_attention="sparse")


@pytest.mark.parametrize("prompt", ["dense", "summon"])
def test_four_bit_cache_with_its_reader_equals_a_read_back_cache(device, prompt):
    """Patched layers read the 4-bit rows in place; unpatched ones get the same rows back in fp32."""
    from sva_amd import FourBitCache

    model, bundle = setup(device)
    ids = tokens(device, 1, 190)
    cuts = [150, 151, 152, 153, 160, 161, 162]
    want = run(model, ids, cuts, cache=FourBitCache())
    exact = run(model, ids, cuts)
    assert (want[:, 151:] - exact[:, 151:]).abs().max() > 1e-3 * exact.abs().max()  # 4 bits do show
    with patch_llama_attention(model, bundle, prompt_attention=prompt):
        cache = FourBitCache()
        got = run(model, ids, cuts, cache=cache)
        if prompt == "dense":  # (a summoned prompt is verified on the rows as held, a dense one uses them as made)
            near(got, want)
        assert cache.get_seq_length() == 162
        layer = cache.layers[0]
        assert layer.data.dtype == torch.uint8 and layer.data.shape[1] == 256
        text = model.generate(ids[:, :20], past_key_values=FourBitCache(), max_new_tokens=4, do_sample=False)
        assert text.shape == (1, 24) and torch.equal(text[:, :20], ids[:, :20])
        again = run(model, ids, cuts, cache=FourBitCache())  # a new cache: the catalogs start over
        assert torch.equal(again, got)
        # a cropped cache goes on from where it was cut
        cache.layers[0].crop(-10), cache.layers[1].crop(-10)
        with torch.no_grad():
            more = model(input_ids=ids[:, 152:153], past_key_values=cache, use_cache=True,
                         position_ids=torch.tensor([[152]], device=device)).logits
        # (its catalog is made again from the rows as held: the lookup still covers every key)
        near(more[0, 0], got[0, 152])


def test_four_bit_cache_grows_and_serves_a_partly_patched_model(device):
    from sva_amd import FourBitCache

    model, bundle = setup(device)
    ids = tokens(device, 1, 300)
    cuts = [200, 250, 255, 256, 257, 258, 300]  # past the first capacity of 256 rows
    want = run(model, ids, cuts, cache=FourBitCache())
    bundle_all = make_tiny_bundle(heads=4, head_dim=32, shortlist=512, budget=512)
    for layers in ([0], [0, 1]):
        with patch_llama_attention(model, bundle_all, prompt_attention="dense", layers=layers):
            near(run(model, ids, cuts, cache=FourBitCache()), want)


def test_four_bit_cache_refusals(device):
    from sva_amd import FourBitCache

    model, bundle = setup(device)
    with patch_llama_attention(model, bundle):
        with pytest.raises(ValueError, match="one sequence"):
            run(model, tokens(device, 2, 5), [5], cache=FourBitCache())
    with patch_llama_attention(model, bundle, summon_mode="inverted"):
        with pytest.raises(ValueError, match="scan"):
            run(model, tokens(device, 1, 5), [5], cache=FourBitCache())
    small = make_tiny_model(device)  # head_dim 8
    with pytest.raises(ValueError, match="multiple of 32"):
        run(small, tokens(device, 1, 5), [5], cache=FourBitCache())


def test_operators_together(device):
    """Packed prompts, their rows into a 4-bit cache, tokens over it: all keys, chosen keys, and the read-back."""
    from sva_amd import kernels

    g = torch.Generator(device=device).manual_seed(5)
    H, G, D, lens, room = 9, 3, 64, [120, 1, 77], 140
    T = sum(lens)
    starts = torch.tensor([0, 120, 121], device=device)
    ln = torch.tensor(lens, device=device)
    q, k, v = (torch.randn(h, T, D, device=device, generator=g) for h in (H, G, G))
    out = kernels.prompt_attention(q, k, v, 120, 0.125, seq_offsets=starts, seq_lens=ln, q_offsets=starts, q_lens=ln,
                                   max_q=120)
    data, scales = kernels.cache4_alloc(G, 3 * room, D, device)
    first = torch.arange(3, device=device) * room
    for b, n in enumerate(lens):
        s = slice(int(starts[b]), int(starts[b]) + n)
        kernels.cache4_write(k[:, s], v[:, s], data, scales, first[b:b + 1])
    q1, k1, v1 = (torch.randn(3, h, 1, D, device=device, generator=g) for h in (H, G, G))
    kernels.cache4_write(k1, v1, data, scales, first + ln)
    got = kernels.cache4_attention(q1, data, scales, room, 0.125, seq_offsets=first, seq_lens=ln + 1)
    keys, values = kernels.cache4_read(data, scales, first, room, torch.float32)  # [3, G, room, D]
    rows = keys.transpose(0, 1).reshape(G, 3 * room, D), values.transpose(0, 1).reshape(G, 3 * room, D)
    dense = kernels.prompt_attention(q1, *rows, room, 0.125, seq_offsets=first, seq_lens=ln + 1)
    assert (got - dense).abs().max() <= 2.0 ** -16 * dense.abs().max() * 4  # weights of two bf16 terms against fp32's
    idx = torch.arange(room, device=device, dtype=torch.int32).expand(27, room).contiguous()
    count = (ln + 1).int().repeat_interleave(H)
    chosen = kernels.cache4_verify(q1, data, scales, idx, count, room, 0.125, None, first, ln + 1)
    assert (got - chosen).abs().max() <= 2.0 ** -16 * dense.abs().max() * 4
    plain = kernels.verify(q1, *rows, idx, count, 3 * room, 0.125, None, first, ln + 1)
    assert (chosen - plain).abs().max() <= 2.0 ** -16 * dense.abs().max()
    assert torch.isfinite(out).all()
