"""A Hugging Face cache whose K and V are held in 4 bits (kernels.cache4_*):
about a quarter of a bf16 cache's memory.

``FourBitCache()`` goes where the model takes ``past_key_values``.  Layers
patched with scan-mode SVA attention read it in place: new rows are written
once, a decode token's lookup is verified on the 4-bit rows it chose
(``kernels.cache4_verify``), and the key catalog comes from the keys as the
model made them.  The catalog is kept with the cache, so caches may be decoded
in turn, cut and copied.  Other layers get the rows back in the model's type, so a
partly patched model runs too (the read costs what a 16-bit cache would).
One sequence per cache, head_dim a multiple of 32 up to 256.  Inference only:
rows that require a gradient are refused (run the model under
``torch.no_grad()``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import kernels


@dataclass
class Catalog:
    """The key catalog of one patched layer over a FourBitLayer: k_low [H, capacity, R] and codes [H, capacity, S], of
    which the first `rows` rows are those of the cache."""

    owner: str
    k_low: torch.Tensor
    codes: torch.Tensor
    rows: int = 0


class FourBitLayer(CacheLayerMixin):
    """One layer's rows: data [G, capacity, 2, D / 2], scales [G, capacity, 2, D / 32], the first `length` in use."""

    is_sliding = False

    def __init__(self, **kwargs) -> None:
        super().__init__()
        self.data: torch.Tensor | None = None
        self.scales: torch.Tensor | None = None
        self.length = 0
        self.catalog: Catalog | None = None

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
        kernels.cache4_write(key_states, value_states, self.data, self.scales, self.length)
        self.length = end

    def read(self, dtype: torch.dtype | None = None, begin: int = 0,
             end: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [1, G, rows, D] of the rows in use, or of [begin, end) of them."""

        end = self.length if end is None else end
        return kernels.cache4_read(self.data, self.scales, begin, end - begin, dtype or self.dtype)

    def catalog_of(self, owner: str, heads: int, rank: int, subspaces: int, code_dtype: torch.dtype) -> Catalog:
        """The catalog of the patched layer `owner`, with room for every row of the cache: the one kept here, or an
        empty one in its place where that is another layer's."""

        kept, capacity = self.catalog, self.data.shape[1]
        if kept is not None and kept.owner == owner and kept.k_low.shape[1] >= capacity:
            return kept
        self.catalog = Catalog(owner, torch.empty(heads, capacity, rank, device=self.device),
                               torch.empty(heads, capacity, subspaces, device=self.device, dtype=code_dtype))
        if kept is not None and kept.owner == owner:
            self.catalog.rows = n = kept.rows
            self.catalog.k_low[:, :n].copy_(kept.k_low[:, :n])
            self.catalog.codes[:, :n].copy_(kept.codes[:, :n])
        return self.catalog

    def _cut(self, length: int) -> None:
        self.length = length
        if self.catalog is not None:
            self.catalog.rows = min(self.catalog.rows, length)

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
        self._cut(0)

    def crop(self, tokens_to_remove: int) -> None:
        """Drops the last -tokens_to_remove rows (a positive number: rows behind it)."""

        keep = tokens_to_remove if tokens_to_remove > 0 else self.length + tokens_to_remove
        self._cut(max(0, min(self.length, keep)))

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
