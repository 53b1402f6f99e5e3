"""A Hugging Face cache whose K and V are held in 4 bits (kernels.cache4_*):
about a quarter of a bf16 cache's memory.

``FourBitCache()`` goes where the model takes ``past_key_values``.  Layers
patched with scan-mode SVA attention read it in place: new rows are written
once, a decode token's lookup is verified on the 4-bit rows it chose
(``kernels.cache4_verify``), and the key catalog comes from the keys as the
model made them.  Other layers get the rows back in the model's type, so a
partly patched model runs too (the read costs what a 16-bit cache would).
One sequence per cache, head_dim a multiple of 32 up to 256.
"""

from __future__ import annotations

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import kernels


class FourBitLayer(CacheLayerMixin):
    """One layer's rows: data [G, capacity, 2, D / 2], scales [G, capacity, 2, D / 32], the first `length` in use."""

    is_sliding = False

    def __init__(self, **kwargs) -> None:
        super().__init__()
        self.data: torch.Tensor | None = None
        self.scales: torch.Tensor | None = None
        self.length = 0

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        self.dtype, self.device = key_states.dtype, key_states.device
        self.data, self.scales = kernels.cache4_alloc(key_states.shape[1], max(256, key_states.shape[2]),
                                                      key_states.shape[3], key_states.device)
        self.is_initialized = True

    def append(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Writes new rows [1, G, T, D] behind the ones in use."""

        if key_states.dim() != 4 or key_states.shape[0] != 1:
            raise ValueError(f"a 4-bit cache holds one sequence, got keys {tuple(key_states.shape)}")
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        end = self.length + key_states.shape[2]
        capacity = self.data.shape[1]
        if end > capacity:
            data, scales = kernels.cache4_alloc(self.data.shape[0], max(end, 2 * capacity), 2 * self.data.shape[3],
                                                self.device)
            data[:, :self.length].copy_(self.data[:, :self.length])
            scales[:, :self.length].copy_(self.scales[:, :self.length])
            self.data, self.scales = data, scales
        with torch.no_grad():
            kernels.cache4_write(key_states, value_states, self.data, self.scales, self.length)
        self.length = end

    def read(self, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [1, G, length, D] of the rows in use."""

        return kernels.cache4_read(self.data, self.scales, 0, self.length, dtype or self.dtype)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """For layers that attend by themselves: the rows so far, as they are held (a first prompt: as given)."""

        first = self.length == 0
        self.append(key_states, value_states)
        return (key_states, value_states) if first else self.read()

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.length + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_length(self) -> int:
        return -1

    def reset(self) -> None:
        self.length = 0

    def crop(self, tokens_to_remove: int) -> None:
        """Drops the last -tokens_to_remove rows (a positive number: rows behind it)."""

        keep = tokens_to_remove if tokens_to_remove > 0 else self.length + tokens_to_remove
        self.length = max(0, min(self.length, keep))

    def offload(self) -> None:
        raise NotImplementedError("a 4-bit cache stays on the GPU")

    prefetch = offload

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        raise NotImplementedError("a 4-bit cache holds one sequence")

    def batch_repeat_interleave(self, repeats: int) -> None:
        if repeats != 1:
            raise NotImplementedError("a 4-bit cache holds one sequence")

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        raise NotImplementedError("a 4-bit cache holds one sequence")


class FourBitCache(Cache):
    """past_key_values with every layer a FourBitLayer."""

    def __init__(self) -> None:
        super().__init__(layer_class_to_replicate=FourBitLayer)


def layer_of(past_key_values, layer_idx: int) -> FourBitLayer | None:
    """The 4-bit layer of a cache, or None where it holds another kind."""

    if not isinstance(past_key_values, FourBitCache):
        return None
    while len(past_key_values.layers) <= layer_idx:
        past_key_values.layers.append(FourBitLayer())
    return past_key_values.layers[layer_idx]
