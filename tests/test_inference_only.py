"""Dense prompts and the 4-bit cache have no backward pass: tensors that require a gradient are refused, from a patched
model and from an unpatched one on a 4-bit cache too, rather than answered without one."""

from __future__ import annotations

import pytest
import torch


def test_operators_refuse_before_any_device_work():
    from sva_amd import kernels
    from sva_amd.cache4 import FourBitLayer

    q, kv = torch.zeros(1, 4, 3, 64, requires_grad=True), torch.zeros(2, 8, 64)
    data, scales = kernels.cache4_alloc(2, 8, 64, "cpu")
    idx, count = torch.zeros(12, 5, dtype=torch.int32), torch.zeros(12, dtype=torch.int32)
    calls = [lambda q: kernels.prompt_attention(q, kv, kv, 8, 1.0),
             lambda q: kernels.cache4_attention(q, data, scales, 8, 1.0),
             lambda q: kernels.cache4_verify(q, data, scales, idx, count, 8, 1.0),
             lambda q: FourBitLayer().append(q, q)]
    for call in calls:
        with pytest.raises(RuntimeError, match="inference only"):
            call(q)
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm"):
            call(q)
        with pytest.raises(RuntimeError, match="ROCm"):
            call(q.detach())


@pytest.mark.gpu
def test_models_refuse(device):
    from transformers import DynamicCache

    from sva import patch_llama_attention
    from sva_amd import FourBitCache

    from .test_gpu_prompt_and_cache4_model import setup, tokens

    model, bundle = setup(device)
    ids = tokens(device, 1, 20)

    def refused(cache):
        with pytest.raises(RuntimeError, match="inference only"):
            model(input_ids=ids, past_key_values=cache, use_cache=True)
        assert cache.get_seq_length() == 0  # no layer has taken a row
        with torch.no_grad():
            out = model(input_ids=ids, past_key_values=cache, use_cache=True)
        assert torch.isfinite(out.logits).all() and out.past_key_values.get_seq_length() == 20
        for p in model.parameters():
            p.requires_grad_(False)
        model(input_ids=ids[:, :2], past_key_values=out.past_key_values, use_cache=True)  # nothing requires a gradient
        for p in model.parameters():
            p.requires_grad_(True)

    refused(FourBitCache())
    with patch_llama_attention(model, bundle, prompt_attention="dense"):
        refused(DynamicCache())
        refused(FourBitCache())
    with patch_llama_attention(model, bundle):
        refused(FourBitCache())


@pytest.mark.gpu
def test_a_query_alone_is_refused_before_the_cache_takes_a_row(device):
    from transformers import DynamicCache

    from sva import patch_llama_attention
    from sva_amd import FourBitCache

    from .test_gpu_prompt_and_cache4_model import setup, tokens

    model, bundle = setup(device)
    for name, p in model.named_parameters():
        p.requires_grad_("q_proj" in name)
    with patch_llama_attention(model, bundle, prompt_attention="dense"):
        for cache in (FourBitCache(), DynamicCache()):
            with pytest.raises(RuntimeError, match="inference only"):
                model(input_ids=tokens(device, 1, 20), past_key_values=cache, use_cache=True)
            assert cache.get_seq_length() == 0
