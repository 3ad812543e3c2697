"""``BlockTopKPattern``: blocks of a paged cache chosen for each query by the bounds of their keys.

The reference's patterns fix their blocks in advance, and its data-dependent top-k keeps single keys, which no
block kernel runs.  Here the choice is made per block on the device, when the queries are known: the pattern
only carries the numbers, and the backend's ``forward_packed`` ranks the pages
(:func:`~sparseattentioninfer_amd.ops.paged_block_select`) and attends the chosen ones.
"""
from __future__ import annotations

import torch

from .base import PatternMetadata, SparsePattern


class BlockTopKPattern(SparsePattern):
    """The first ``sink`` blocks, the last ``recent`` and the ``top_k`` best of those between."""

    def __init__(self, top_k: int, *, block_size: int = 64, sink: int = 1, recent: int = 2):
        if top_k < 0 or sink < 0 or recent < 1:
            raise ValueError(f"top_k={top_k} and sink={sink} must not be negative, recent={recent} at least 1")
        self.top_k, self.block_size, self.sink, self.recent = top_k, block_size, sink, recent

    def build(self, q: torch.Tensor, k: torch.Tensor, causal: bool = True) -> PatternMetadata:
        blocks = max(1, -(-k.size(2) // self.block_size))
        kept = min(blocks, self.sink + self.top_k + self.recent)
        return PatternMetadata(kind="block_topk", topk=self.top_k, block_size=self.block_size, sink=self.sink,
                               recent=self.recent, keep_ratio=kept / blocks)
