"""A Hugging Face cache whose K and V are held in pages (kernels.paged_*,
kernels.pages_*), and sampled generation over it.

``PagedCache(model.config)`` goes where the model takes ``past_key_values``.
Every layer's rows lie in one pool of pages that the sequences name in a table:
a fork of a sequence (``fork``, beam search, several samples of one prompt)
shares its pages, and only the last one is copied, where the two part.  Layers
patched with SVA attention read the pages in place, by attention over every row:
no lookup, no key catalog and no statistics.  Other layers get the rows back as
the model's own cache would hold them.

The sequences of a batch have one length.  Inference only: rows that require a
gradient are refused (run the model under ``torch.no_grad()``).
"""

from __future__ import annotations

import inspect

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import kernels


class PagedLayer(CacheLayerMixin):
    """One layer's view of a PagedCache: `pool` [pages, 2, G, P, D], the first `length` rows of every sequence in use."""

    is_sliding = False

    def __init__(self, cache: "PagedCache", index: int) -> None:
        super().__init__()
        self.cache, self.index, self.length = cache, index, 0

    @property
    def pool(self) -> torch.Tensor:
        return self.cache.pool[self.index]

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def append(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Writes new rows [B, G, T, D] behind the ones in use."""

        kernels._inference_only("a paged cache", key_states, value_states)
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        first = self.cache.rows_for(self.length, key_states)
        kernels.paged_write(key_states, value_states, self.pool, self.cache.tables, first)
        self.length += key_states.shape[2]

    def read(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [B, G, length, D]."""

        return kernels.paged_read(self.pool, self.cache.tables, self.cache.zeros, self.length)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """For layers that attend by themselves: the rows so far (a first prompt: as given)."""

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

    def offload(self) -> None:
        raise NotImplementedError("a paged cache stays on the GPU")

    prefetch = offload

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        raise NotImplementedError("the layers of a paged cache are reordered together")


class PagedCache(Cache):
    """past_key_values in pages: pool [layers, pages, 2, G, P, D], tables [B, entries], lens [B] and refs [pages]
    (kernels.pages_*).  page_rows: a power of two from 16 to 1024."""

    def __init__(self, config, page_rows: int = 16) -> None:
        config = config.get_text_config(decoder=True) if hasattr(config, "get_text_config") else config
        heads = config.num_attention_heads
        self.kv_heads = getattr(config, "num_key_value_heads", None) or heads
        self.head_dim = getattr(config, "head_dim", None) or config.hidden_size // heads
        self.page_rows, self.n_layers = page_rows, config.num_hidden_layers
        kernels._check_page_shape(page_rows, self.head_dim)
        super().__init__(layers=[PagedLayer(self, i) for i in range(self.n_layers)])
        self.pool: torch.Tensor | None = None
        self.tables = self.lens = self.refs = self.zeros = None
        self.length = 0                               # rows that every sequence has room for
        self.first_rows: torch.Tensor | None = None   # of the newest ones
        self._used_most = 0                           # pages in use: at most this many

    # ------------------------------------------------------------------ rows
    def rows_for(self, length: int, key_states: torch.Tensor) -> torch.Tensor:
        """First rows [B] on the device for key_states [B, G, T, D] behind `length` rows: the first layer that asks has
        pages handed out, the others get the same."""

        batch, kv_heads, n_rows, dim = key_states.shape
        if (kv_heads, dim) != (self.kv_heads, self.head_dim):
            raise ValueError(f"a paged cache of {self.kv_heads} KV heads of {self.head_dim}, got keys "
                             f"{tuple(key_states.shape)}")
        if self.pool is None:
            self._begin(batch, key_states)
        if batch != self.tables.shape[0]:
            raise ValueError(f"{batch} sequences of a paged cache of {self.tables.shape[0]}")
        if length + n_rows > self.length:
            if length != self.length:
                raise ValueError(f"rows {length} to {length + n_rows} of a paged cache of {self.length}: its layers are "
                                 f"not at one length")
            self._reserve(n_rows)
        elif length + n_rows != self.length:
            raise ValueError("the layers of a paged cache take the same rows")
        return self.first_rows

    def _begin(self, batch: int, like: torch.Tensor) -> None:
        self.tables = torch.full((batch, 0), -1, device=like.device, dtype=torch.int32)
        self.lens = torch.zeros(batch, device=like.device, dtype=torch.int64)
        self.zeros = torch.zeros_like(self.lens)
        self.refs = torch.zeros(0, device=like.device, dtype=torch.int32)
        self.pool = torch.empty((self.n_layers, 0, 2, self.kv_heads, self.page_rows, self.head_dim), device=like.device,
                                dtype=like.dtype)

    def _pages(self, rows: int) -> int:
        return -(-rows // self.page_rows)

    def _reserve(self, n_rows: int) -> None:
        batch, entries = self.tables.shape
        old, new = self._pages(self.length), self._pages(self.length + n_rows)
        if new > entries:
            wide = torch.full((batch, max(new, 2 * entries)), -1, device=self.tables.device, dtype=torch.int32)
            wide[:, :entries] = self.tables
            self.tables = wide
        # a page more for each sequence that may share its last one
        need = batch * (new - old + (1 if self.length % self.page_rows else 0))
        if self._used_most + need > self.refs.shape[0]:
            self._used_most = int((self.refs > 0).sum())
            if self._used_most + need > self.refs.shape[0]:
                self._grow(max(self._used_most + need, 2 * self.refs.shape[0]))
        self._used_most += need
        self.first_rows, src, dst = kernels.pages_reserve(self.tables, self.lens, self.refs, n_rows, self.page_rows)
        if self.length % self.page_rows:
            kernels.pages_copy(self.pool, src, dst)
        self.length += n_rows

    def _grow(self, pages: int) -> None:
        held = self.refs.shape[0]
        pool = kernels.pages_alloc(pages, self.kv_heads, self.page_rows, self.head_dim, self.pool.device, self.pool.dtype,
                                   layers=self.n_layers)
        pool[:, :held].copy_(self.pool)
        refs = torch.zeros(pages, device=self.refs.device, dtype=torch.int32)
        refs[:held].copy_(self.refs)
        self.pool, self.refs = pool, refs

    # ------------------------------------------------------------------ sequences
    def fork(self, sources) -> None:
        """The batch becomes forks of its sequences: new sequence i of `sources` (int64 tensor, or ints; any number of
        them, each a sequence's) shares the pages of sequence sources[i].  Those that are not named are freed.  The
        numbers are looked at by the host, which waits for those that are on the device."""

        if self.pool is None:
            return
        sources = torch.as_tensor(sources, dtype=torch.int64).flatten()
        host, old = sources.cpu(), self.tables.shape[0]
        if not bool(((host >= 0) & (host < old)).all()):
            raise ValueError(f"forks of {host.tolist()} from a paged cache of {old} sequences")
        self._fork(sources.to(self.tables.device))

    def _fork(self, sources: torch.Tensor) -> None:
        """The same for int64 numbers on the device that are known to be sequences'."""

        old, new = self.tables.shape[0], sources.shape[0]
        if new > old:
            self.tables = torch.cat([self.tables, self.tables.new_full((new - old, self.tables.shape[1]), -1)])
            self.lens = torch.cat([self.lens, self.lens.new_zeros(new - old)])
        elif new < old:
            sources = torch.cat([sources, sources.new_full((old - new,), -1)])
        kernels.pages_fork(self.tables, self.lens, self.refs, sources, self.page_rows)
        if new < old:
            self.tables, self.lens = self.tables[:new].contiguous(), self.lens[:new].contiguous()
        self.zeros = torch.zeros_like(self.lens)
        self.first_rows = None

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        self.fork(beam_idx)

    def batch_repeat_interleave(self, repeats: int) -> None:
        if self.pool is not None:
            self._fork(torch.arange(self.tables.shape[0], device=self.tables.device).repeat_interleave(repeats))

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        if self.pool is not None:
            self.fork(torch.arange(self.tables.shape[0])[torch.as_tensor(indices).cpu()])

    def crop(self, tokens_to_remove: int) -> None:
        """Drops the last -tokens_to_remove rows (a positive number: rows behind it)."""

        keep = tokens_to_remove if tokens_to_remove > 0 else self.length + tokens_to_remove
        keep = max(0, min(self.length, keep))
        for layer in self.layers:
            layer.length = min(layer.length, keep)
        if self.pool is None or keep == self.length:
            return
        gone = self.tables[:, self._pages(keep):self._pages(self.length)]
        pages = gone.flatten().long()
        there = (pages >= 0) & (pages < self.refs.shape[0])  # (a sequence that kernels.pages_fork freed has none)
        if self.refs.shape[0] > 0:
            self.refs.index_add_(0, torch.where(there, pages, 0), -there.int())
        gone.fill_(-1)
        self.lens.clamp_(max=keep)
        self.length, self.first_rows = keep, None

    def compact(self, release: bool = False) -> None:
        """Moves the pages in use together; `release` gives the others' memory back."""

        if self.pool is None or self.refs.shape[0] == 0:
            return
        src, dst, used = kernels.pages_compact(self.tables, self.refs)
        kernels.pages_copy(self.pool, src, dst)
        self._used_most = int(used)
        if release:
            self.pool, self.refs = self.pool[:, :self._used_most].clone(), self.refs[:self._used_most].clone()

    def reset(self) -> None:
        for layer in self.layers:
            layer.reset()
        self.pool = self.tables = self.lens = self.refs = self.zeros = self.first_rows = None
        self.length = self._used_most = 0


def layer_of(past_key_values, layer_idx: int) -> PagedLayer | None:
    """The paged layer of a cache, or None where it holds another kind."""

    return past_key_values.layers[layer_idx] if isinstance(past_key_values, PagedCache) else None


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int, num_samples: int = 1, temperature: float = 1.0,
             top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, generator: torch.Generator | None = None,
             eos_token_id: int | None = None, cache: PagedCache | None = None) -> torch.Tensor:
    """`num_samples` continuations of each prompt of input_ids [B, T], drawn by kernels.sample_tokens over a paged cache:
    tokens [B * num_samples, T + new], the samples of a prompt one after another.  The prompts are run once, their pages
    shared by the samples.  Sequences that have ended go on as eos_token_id; all having ended, the rest is left out.
    cache: rows before input_ids (of B sequences), extended in place.  A token -1 says that its logits were all NaN or
    -inf; the sequence goes on from token 0."""

    if max_new_tokens < 1 or num_samples < 1:
        raise ValueError(f"{num_samples} samples of {max_new_tokens} tokens")
    cache = PagedCache(model.config) if cache is None else cache
    # (a prompt's other logits, 2 T V bytes of them in bf16, are not asked for where the model can leave them out)
    last = {"logits_to_keep": 1} if "logits_to_keep" in inspect.signature(model.forward).parameters else {}
    logits = model(input_ids=input_ids, past_key_values=cache, use_cache=True, **last).logits[:, -1]
    if num_samples > 1:
        cache.batch_repeat_interleave(num_samples)
        logits = logits.repeat_interleave(num_samples, 0)
    out = [input_ids.repeat_interleave(num_samples, 0)]
    ended = torch.zeros(logits.shape[0], device=logits.device, dtype=torch.bool)
    for step in range(max_new_tokens):
        uniforms = torch.rand(logits.shape[0], device=logits.device, generator=generator)
        token = kernels.sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p)
        if eos_token_id is not None:
            token = torch.where(ended, eos_token_id, token)
            ended |= token == eos_token_id
        out.append(token[:, None])
        if step + 1 == max_new_tokens or (eos_token_id is not None and bool(ended.all())):
            break
        logits = model(input_ids=token[:, None].clamp_min(0), past_key_values=cache, use_cache=True).logits[:, -1]
    return torch.cat(out, 1)
