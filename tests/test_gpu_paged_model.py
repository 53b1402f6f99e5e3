"""A cache in pages in models, patched and not: prompts, cached decode, forks, beams, crops, compaction and sampled
generation, against the same model over its own cache.  A paged cache's attention is exact, so the logits may differ by
fp32 rounding alone (1e-4 of their largest, as for dense prompts)."""

from __future__ import annotations

import copy

import pytest
import torch
from transformers import DynamicCache

from sva import patch_llama_attention

from .test_gpu_prompt_and_cache4_model import near, setup, tokens

pytestmark = pytest.mark.gpu


@torch.no_grad()
def feed(model, cache, ids, a, b, mask=None):
    return model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True,
                 attention_mask=None if mask is None else mask[:, :b]).logits


CUTS = [0, 37, 38, 39, 44, 90, 91]  # a prompt, two tokens, a few, a chunk, a token


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("patched", ["all", "one", "none"])
def test_equals_the_model(device, batch, patched):
    from sva_amd import PagedCache

    model, bundle = setup(device)
    ids = tokens(device, batch, 91)
    dense = DynamicCache()
    want = [feed(model, dense, ids, a, b) for a, b in zip(CUTS, CUTS[1:])]
    cache = PagedCache(model.config)

    def run():
        for (a, b), w in zip(zip(CUTS, CUTS[1:]), want):
            near(feed(model, cache, ids, a, b), w)
        assert cache.get_seq_length() == 91 and cache.lens.tolist() == [91] * batch

    if patched == "none":
        run()
    else:
        with patch_llama_attention(model, bundle, layers=None if patched == "all" else [1]) as handle:
            run()
            assert handle.stats.summary()["queries"] == 0  # no lookup
    for layer, own in zip(cache.layers, dense.layers):  # the rows themselves
        keys, values = layer.read()
        near(keys, own.keys)
        near(values, own.values)


def test_a_padded_batch(device):
    from sva_amd import PagedCache

    model, bundle = setup(device)
    ids = tokens(device, 3, 40)
    mask = torch.ones(3, 40, dtype=torch.long, device=device)
    mask[1, :7] = 0
    mask[2, :25] = 0
    dense = DynamicCache()
    want = [feed(model, dense, ids, a, b, mask) for a, b in ((0, 38), (38, 39), (39, 40))]
    cache = PagedCache(model.config)
    with patch_llama_attention(model, bundle):
        got = [feed(model, cache, ids, a, b, mask) for a, b in ((0, 38), (38, 39), (39, 40))]
    for g, w in zip(got, want):
        for b, pad in enumerate((0, 7, 25)):
            near(g[b, pad if g.shape[1] > 1 else 0:], w[b, pad if g.shape[1] > 1 else 0:])


@pytest.mark.parametrize("page_rows", [16, 64])
def test_forks_share_pages_and_part(device, page_rows):
    """Forks of forks, more and fewer sequences, crops, a copy, a compaction: every sequence goes on as one that is run
    alone."""
    from sva_amd import PagedCache

    model, bundle = setup(device)
    prompts = tokens(device, 2, 70)
    more = tokens(device, 6, 60, seed=5)
    with patch_llama_attention(model, bundle), torch.no_grad():
        cache = PagedCache(model.config, page_rows=page_rows)
        feed(model, cache, prompts, 0, 70)
        used = lambda c: int((c.refs > 0).sum())  # noqa: E731
        before = used(cache)
        cache.fork([0, 0, 1, 0, 1])
        assert used(cache) == before and cache.tables.shape[0] == 5
        rows = [prompts[0], prompts[0], prompts[1], prompts[0], prompts[1]]

        def both(n, at):
            nonlocal rows
            new = more[:len(rows), at:at + n]
            got = model(input_ids=new, past_key_values=cache, use_cache=True).logits
            rows = [torch.cat([r, x]) for r, x in zip(rows, new)]
            fresh = PagedCache(model.config)
            near(got, feed(model, fresh, torch.stack(rows), 0, len(rows[0]))[:, -n:])

        both(1, 0)
        assert used(cache) > before
        both(3, 1)
        cache.reorder_cache(torch.tensor([4, 1, 1, 2, 0], device=device))
        rows = [rows[i] for i in (4, 1, 1, 2, 0)]
        both(1, 4)
        cache.batch_select_indices(torch.tensor([3, 0], device=device))
        rows = [rows[3], rows[0]]
        cache.compact()
        assert bool((cache.refs[:used(cache)] > 0).all())
        both(20, 5)
        kept = copy.deepcopy(cache)
        kept_rows = list(rows)
        cache.crop(-9)
        rows = [r[:-9] for r in rows]
        both(2, 30)
        cache.batch_repeat_interleave(3)
        rows = [r for r in rows for _ in range(3)]
        cache.compact(release=True)
        assert cache.pool.shape[1] == used(cache)
        both(17, 33)
        assert kept.get_seq_length() == len(kept_rows[0])
        near(model(input_ids=more[:2, :1], past_key_values=kept, use_cache=True).logits[:, -1],
             feed(model, PagedCache(model.config), torch.stack([torch.cat([r, x]) for r, x in zip(kept_rows, more[:2, :1])]), 0,
                  len(kept_rows[0]) + 1)[:, -1])
        cache.reset()
        assert cache.get_seq_length() == 0
        near(feed(model, cache, prompts, 0, 70), feed(model, PagedCache(model.config), prompts, 0, 70))


@pytest.mark.parametrize("patched", [True, False])
def test_beams(device, patched, monkeypatch):
    """Beam search chooses the same beams over a paged cache (fp32: scores of beams lie further apart than rounding)."""
    from sva_amd import PagedCache, kernels

    calls, attend = [], kernels.paged_attention
    monkeypatch.setattr(kernels, "paged_attention", lambda *a, **k: calls.append(1) or attend(*a, **k))

    model, bundle = setup(device)
    ids = tokens(device, 2, 30)
    # (without a mask given, tokens of the padding's number would be masked)
    ask = dict(max_new_tokens=25, num_beams=4, do_sample=False, pad_token_id=0, eos_token_id=None,
               attention_mask=torch.ones_like(ids))
    want = model.generate(ids, **ask)
    if patched:
        with patch_llama_attention(model, bundle):
            got = model.generate(ids, past_key_values=PagedCache(model.config), **ask)
    else:
        got = model.generate(ids, past_key_values=PagedCache(model.config), **ask)
    assert torch.equal(got, want) and len(calls) == (2 * 24 if patched else 0)


def test_generate_from_nothing(device):
    """Logits that are all NaN: -1, and what the model is given next is a token of it."""
    from sva_amd import generate

    model, _ = setup(device)
    ids = tokens(device, 2, 9)
    given = []
    inner = model.forward

    def forward(input_ids, **kw):
        given.append(input_ids.tolist())
        out = inner(input_ids=input_ids.clamp(0, 63), **kw)
        out.logits = torch.full_like(out.logits, float("nan"))
        return out

    model.forward = forward
    assert generate(model, ids, 3).tolist() == [row + [-1, -1, -1] for row in ids.tolist()]
    assert given == [ids.tolist(), [[0], [0]], [[0], [0]]]


def test_generate(device):
    """Samples of prompts drawn token by token as the definition draws them from the model's own logits."""
    from sva_amd import PagedCache, generate

    from .paged_reference import sample

    model, bundle = setup(device)
    ids = tokens(device, 2, 33)
    ask = dict(temperature=0.8, top_k=20, top_p=0.9, min_p=0.01)
    cache = PagedCache(model.config)
    with patch_llama_attention(model, bundle):
        out = generate(model, ids, 40, num_samples=5, generator=torch.Generator(device=device).manual_seed(3), cache=cache, **ask)
    assert out.shape == (10, 73) and cache.get_seq_length() == 72
    assert torch.equal(out[:, :33], ids.repeat_interleave(5, 0))
    assert len({tuple(r) for r in out.tolist()}) == 10
    gen = torch.Generator(device=device).manual_seed(3)
    uniforms = [torch.rand(10, device=device, generator=gen).tolist() for _ in range(40)]
    with torch.no_grad():
        logits = model(input_ids=out).logits[:, 32:72].double().cpu().numpy()
    known = 0
    for b in range(10):
        for t in range(40):
            # (logits within 1e-4 of their largest: weights, and borders, within 4e-4 / 0.8)
            want = sample(logits[b, t], uniforms[t][b], border=1e-3, **{k: v if k == "top_k" else float(torch.tensor(v))
                                                                        for k, v in ask.items()})
            known += want is not None
            assert want is None or want == int(out[b, 33 + t]), (b, t)
    assert known > 300
    greedy = generate(model, ids, 12, temperature=0.0)
    assert torch.equal(greedy, model.generate(ids, max_new_tokens=12, do_sample=False, pad_token_id=0, eos_token_id=None,
                                              attention_mask=torch.ones_like(ids)))
    stop = int(greedy[0, 35])
    ended = generate(model, ids[:1], 12, temperature=0.0, eos_token_id=stop)
    assert ended.shape[1] <= 36 and int(ended[0, -1]) == stop


def test_refusals(device):
    from sva_amd import PagedCache, generate

    model, bundle = setup(device)
    ids = tokens(device, 2, 20)
    with pytest.raises(RuntimeError, match="inference only"):
        model(input_ids=ids, past_key_values=PagedCache(model.config), use_cache=True)
    with patch_llama_attention(model, bundle), pytest.raises(RuntimeError, match="inference only"):
        model(input_ids=ids, past_key_values=PagedCache(model.config), use_cache=True)
    with pytest.raises(ValueError):
        PagedCache(model.config, page_rows=8)
    with pytest.raises(ValueError):
        generate(model, ids, 0)
    cache = PagedCache(model.config)
    feed(model, cache, ids, 0, 10)
    with pytest.raises(ValueError, match="sequences"):
        feed(model, cache, ids[:1], 0, 1)
    for bad in ([0, 2], [-1]):
        with pytest.raises(ValueError, match="forks"):
            cache.fork(bad)


def test_forks_of_no_sequence_are_refused(device):
    """Numbers on the device are looked at too, and nothing changes: the cache goes on, and a crop finds its pages."""
    from sva_amd import PagedCache

    model, bundle = setup(device)
    ids = tokens(device, 2, 60)
    cache = PagedCache(model.config)
    feed(model, cache, ids, 0, 40)
    held = cache.tables.clone(), cache.lens.clone(), cache.refs.clone()
    for bad in ([0, 2], [-1, 0], [0, 1, -1], [1, 0, 5], [2 ** 40, 0]):
        for call in (cache.fork, cache.reorder_cache):
            with pytest.raises(ValueError, match="forks"):
                call(torch.tensor(bad, device=device))
    for bad in ([0, 2], [-3]):
        with pytest.raises(IndexError):
            cache.batch_select_indices(torch.tensor(bad, device=device))
    assert all(torch.equal(a, b) for a, b in zip(held, (cache.tables, cache.lens, cache.refs)))
    cache.batch_select_indices(torch.tensor([False, True], device=device))
    cache.batch_repeat_interleave(2)
    cache.crop(-15)
    assert int(cache.refs.sum()) == 2 * 2 and cache.lens.tolist() == [25, 25]
    rows = torch.cat([ids[1:, :25], ids[1:, 40:]], 1).expand(2, -1)
    got = feed(model, cache, rows, 25, 45)
    near(got, feed(model, DynamicCache(), rows, 0, 45)[:, -20:])


@pytest.mark.parametrize("batch,samples", [(1, 1), (2, 3)])
def test_generate_takes_the_last_logits_alone(device, batch, samples):
    """Nothing but the last token of a prompt goes through the output layer; a model that takes no such wish gives all."""
    from sva_amd import generate

    model, bundle = setup(device)
    ids = tokens(device, batch, 50)
    seen = []
    hook = model.lm_head.register_forward_pre_hook(lambda m, args: seen.append(tuple(args[0].shape[:2])))
    with patch_llama_attention(model, bundle):
        got = generate(model, ids, 3, num_samples=samples, temperature=0.0)
        assert seen == [(batch, 1), (batch * samples, 1), (batch * samples, 1)]
        seen.clear()
        inner = model.forward
        model.forward = lambda input_ids, past_key_values, use_cache: inner(input_ids=input_ids, past_key_values=past_key_values,
                                                                            use_cache=use_cache)
        assert torch.equal(generate(model, ids, 3, num_samples=samples, temperature=0.0), got)
        assert seen == [(batch, 50), (batch * samples, 1), (batch * samples, 1)]
    hook.remove()
