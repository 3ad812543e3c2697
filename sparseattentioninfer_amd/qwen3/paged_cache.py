"""Hugging Face ``Cache`` over paged K/V: the bridge between HF generation and the paged decode kernel.

``PagedKVCache`` is a ``transformers.cache_utils.Cache`` whose layers keep
their K/V in a :class:`~sparseattentioninfer_amd.models.kv_cache.PagedKVStore`
(page pool + block table).  HF code that calls ``update()`` gets contiguous
``[B, H_kv, T, D]`` copies gathered from the pages (correct, but a copy per
call); :class:`~sparseattentioninfer_amd.qwen3.modeling_sparse_qwen3.Qwen3SparseKernelAttention`
instead writes the new tokens with :meth:`PagedKVLayer.write` and decodes straight
from the pages, with no ``repeat_kv`` and no ``torch.cat`` growth of the cache.
"""
from __future__ import annotations

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from ..models.kv_cache import PagedChunk, PagedKVStore


class PagedKVLayer(CacheLayerMixin):
    """One decoder layer's paged K/V, allocated on the first write."""

    is_sliding = False
    is_compileable = False

    def __init__(self, max_len: int, *, page: int = 64, shuffle_seed: int | None = None, bounds: bool = False, bits: int = 16):
        super().__init__()
        self.max_len, self.page, self.shuffle_seed, self.bounds, self.bits = max_len, page, shuffle_seed, bounds, bits
        self.store: PagedKVStore | None = None

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        B, H, _, D = key_states.shape
        self._make_store(B, H, D, key_states)

    def _make_store(self, B: int, H: int, D: int, like: torch.Tensor) -> None:
        self.dtype, self.device = like.dtype, like.device
        self.store = PagedKVStore(B, H, D, self.max_len, page=self.page, dtype=like.dtype, device=like.device,
                                  shuffle_seed=self.shuffle_seed, bounds=self.bounds, bits=self.bits)
        self.is_initialized = True

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, counts, **rope) -> PagedChunk:
        """:meth:`PagedKVStore.append` of packed ``[N, H, D]`` projections (queries too), allocating on first use."""
        if self.is_initialized:
            return self.store.append(k, v, counts, q=q, **rope)
        self._make_store(len(counts), k.size(1), k.size(2), k)
        try:
            return self.store.append(k, v, counts, q=q, **rope)
        except BaseException:      # a store of the refused tensors' type and device would refuse the right ones
            self.store, self.is_initialized = None, False
            raise

    def write(self, key_states: torch.Tensor, value_states: torch.Tensor) -> PagedKVStore:
        """Appends ``[B, H_kv, t, D]`` K/V to the pages; returns the store."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        self.store.write(key_states, value_states)
        return self.store

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """HF interface: appends, then returns contiguous copies of the whole cache."""
        self.write(key_states, value_states)
        return self.store.gather()

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.get_seq_length() + query_length, 0

    def get_seq_length(self) -> int:
        return self.store.seq_len() if self.store is not None else 0

    def get_max_length(self) -> int:
        return self.max_len

    def reset(self) -> None:
        if self.store is not None:
            self.store.reset()

    def offload(self):
        raise NotImplementedError("PagedKVCache does not offload to the host")

    def prefetch(self):
        raise NotImplementedError("PagedKVCache does not offload to the host")

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        raise NotImplementedError("PagedKVCache does not reorder sequences (no beam search)")

    def crop(self, tokens_to_remove: int) -> None:
        raise NotImplementedError("PagedKVCache does not crop")


class PagedKVCache(Cache):
    """``num_layers`` paged layers of up to ``max_len`` tokens per sequence; with ``bounds`` their pages keep the
    key bounds that the ``"block_topk"`` pattern selects by, with ``bits=4`` they hold 4-bit codes.  A prompt into an empty
    cache attends its own keys and values (``block_topk``: the pages), everything after it what the pages hold."""

    def __init__(self, num_layers: int, max_len: int, *, page: int = 64, shuffle_seed: int | None = None,
                 bounds: bool = False, bits: int = 16):
        if bits not in (4, 16):
            raise ValueError(f"a PagedKVCache holds 16 or 4 bits, not {bits}")
        super().__init__(layers=[PagedKVLayer(max_len, page=page, shuffle_seed=shuffle_seed, bounds=bounds, bits=bits)
                                 for _ in range(num_layers)])
        self.page, self.bits = page, bits

    @property
    def max_cache_len(self) -> int:
        return self.layers[0].max_len
