"""KV caches for decoding: the reference's per-layer ``KVCache`` API over preallocated storage, and
a paged cache (page pool + block table) that the paged decode kernel reads directly.

``KVCache`` keeps the method names and meaning of
``sparse_attentions/models/kv_cache.py:7-59`` (``init``, ``clone``, ``append``,
``seq_len``, ``clear``) but stores each layer in a ``[B, H, capacity, D]`` buffer:
``append`` writes the new tokens in place and returns ``[B, H, T, D]`` views
(head dim contiguous, token stride D), where the reference concatenates and
copies the whole cache on every step.  The capacity grows by doubling (one
copy) only when exceeded.

``PagedKVStore`` holds one layer's pages ``[P, H, page, D]``, a block table
``[B, max_blocks]`` (logical block -> page) and the sequence lengths; pages
are taken from a free list as sequences grow.  It is the layout
``sa_decode`` reads in paged mode.  ``append`` takes a chunk of new tokens whose
number differs from sequence to sequence.  With ``bits=4`` the pages hold 4-bit
codes with a scale and a minimum for each 32 dims (``ops.paged_append_q4``),
3.2 times fewer bytes.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from itertools import accumulate

import torch

from .. import ops


def _round_up(x: int, m: int) -> int:
    return -(-x // m) * m


class KVCache:
    """Per-layer KV cache for autoregressive decoding (reference API, in-place storage).

    ``max_len`` (optional) sizes every layer's buffer up front; otherwise the
    first ``init``/``append`` sizes it and later appends double it as needed.
    """

    GRANULE = 64   # capacity rounding, one KV block

    def __init__(self, num_layers: int, max_len: int | None = None):
        self.num_layers = num_layers
        self.max_len = max_len
        self._kbuf: list[torch.Tensor | None] = [None] * num_layers
        self._vbuf: list[torch.Tensor | None] = [None] * num_layers
        self._len = [0] * num_layers

    # -- storage -------------------------------------------------------------------------
    def _reserve(self, layer_idx: int, like: torch.Tensor, need: int) -> None:
        kb = self._kbuf[layer_idx]
        if kb is not None and kb.size(2) >= need and kb.shape[:2] == like.shape[:2] and kb.size(3) == like.size(3):
            return
        cap = max(need, self.max_len or 0, 2 * kb.size(2) if kb is not None else 0)
        cap = _round_up(cap, self.GRANULE)
        B, H, _, D = like.shape
        nk = torch.empty(B, H, cap, D, dtype=like.dtype, device=like.device)
        nv = torch.empty_like(nk)
        n = self._len[layer_idx]
        if kb is not None and n:
            nk[:, :, :n].copy_(kb[:, :, :n])
            nv[:, :, :n].copy_(self._vbuf[layer_idx][:, :, :n])
        self._kbuf[layer_idx], self._vbuf[layer_idx] = nk, nv

    def _view(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        n = self._len[layer_idx]
        return self._kbuf[layer_idx][:, :, :n], self._vbuf[layer_idx][:, :, :n]

    # -- reference API -------------------------------------------------------------------
    def init(self, k_list: list[torch.Tensor], v_list: list[torch.Tensor]) -> None:
        """Fills every layer from a prefill's K/V (``[B, H, T, D]`` each)."""
        assert len(k_list) == self.num_layers
        assert len(v_list) == self.num_layers
        self.clear()
        for i, (k, v) in enumerate(zip(k_list, v_list)):
            self.append(i, k, v)

    def clone(self) -> "KVCache":
        """Deep copy, so decode benchmarks can reuse a fixed prefix."""
        out = KVCache(self.num_layers, self.max_len)
        for i in range(self.num_layers):
            if self._kbuf[i] is not None:
                out._kbuf[i] = self._kbuf[i].clone()
                out._vbuf[i] = self._vbuf[i].clone()
            out._len[i] = self._len[i]
        return out

    def append(self, layer_idx: int, k_new: torch.Tensor, v_new: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Appends ``[B, H, t, D]`` new K/V and returns the full ``[B, H, T + t, D]`` views."""
        if k_new.shape != v_new.shape:
            raise ValueError(f"k_new {tuple(k_new.shape)} and v_new {tuple(v_new.shape)} differ")
        n, t = self._len[layer_idx], k_new.size(2)
        self._reserve(layer_idx, k_new, n + t)
        self._kbuf[layer_idx][:, :, n:n + t].copy_(k_new)
        self._vbuf[layer_idx][:, :, n:n + t].copy_(v_new)
        self._len[layer_idx] = n + t
        return self._view(layer_idx)

    def seq_len(self, layer_idx: int = 0) -> int:
        return self._len[layer_idx]

    def clear(self) -> None:
        """Forgets the cached tokens; the buffers are kept for reuse."""
        self._len = [0] * self.num_layers

    def truncate(self, length: int) -> None:
        """Drops every layer's tokens past ``length`` (no copy): a benchmark's decode step can
        restart from the same prefix."""
        self._len = [min(n, length) for n in self._len]

    def get(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The cached ``[B, H, T, D]`` views of one layer."""
        if self._kbuf[layer_idx] is None:
            raise KeyError(f"layer {layer_idx} holds no tokens")
        return self._view(layer_idx)


@dataclass
class PagedChunk:
    """New tokens that :meth:`PagedKVStore.append` has written: those of sequence b are rows
    ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` of the packed tensors."""
    cu_seqlens: torch.Tensor            # [B + 1] int32, on the store's device
    counts: tuple[int, ...]             # new tokens of each sequence
    q: torch.Tensor | None              # the normed and rotated queries, if any were given

    @property
    def single_tokens(self) -> bool:
        """Whether every sequence has exactly one."""
        return all(n == 1 for n in self.counts)


class PagedKVStore:
    """One layer's paged K/V: ``k_pages, v_pages [P, H, page, D]``, ``block_table [B, max_blocks]``.

    Pages are handed out from a free list (in a seeded shuffled order when
    ``shuffle_seed`` is given, to exercise non-contiguous tables) as
    sequences grow; ``lens`` counts the valid tokens per sequence on the host
    and ``kv_lens`` mirrors it on the device.  With ``bounds`` (on the GPU) ``k_bounds [P, H, 2, D]`` keeps
    the smallest and largest key of each page in each dim, which ``ops.paged_block_select`` ranks pages by.
    With ``bits=4`` (on the GPU) the pools are uint8 ``[P, H, ops.q4_block_bytes(page, D)]``, for tensors of ``dtype``; what
    is read or attended from the pages is what the codes stand for, not the tensors that were written.
    """

    def __init__(self, batch: int, heads: int, head_dim: int, max_len: int, *, page: int = 64,
                 dtype=torch.bfloat16, device="cuda", num_pages: int | None = None,
                 shuffle_seed: int | None = None, bounds: bool = False, bits: int = 16):
        if bits not in (4, 16):
            raise ValueError(f"a PagedKVStore holds 16 or 4 bits, not {bits}")
        if bits == 4 and torch.device(device).type != "cuda":
            raise ValueError("a PagedKVStore of 4 bits lives on the GPU (its append kernel quantises)")
        if bits == 4 and (dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128)):
            raise ValueError(f"a PagedKVStore of 4 bits holds fp16 or bf16 heads of 64 or 128 dims, not {dtype} of {head_dim}")
        if bounds and torch.device(device).type != "cuda":
            raise ValueError("a PagedKVStore with key bounds lives on the GPU (its append kernel keeps them)")
        if page % 16 or not 16 <= page <= 128:
            raise ValueError(f"page {page} must be a multiple of 16 in [16, 128]")
        self.batch, self.heads, self.head_dim, self.page = batch, heads, head_dim, page
        self.max_blocks = -(-max_len // page)
        self.num_pages = num_pages if num_pages is not None else batch * self.max_blocks
        self.bits, self.dtype = bits, dtype
        if bits == 4:
            self.k_pages = torch.empty(self.num_pages, heads, ops.q4_block_bytes(page, head_dim), dtype=torch.uint8, device=device)
        else:
            self.k_pages = torch.empty(self.num_pages, heads, page, head_dim, dtype=dtype, device=device)
        self.v_pages = torch.empty_like(self.k_pages)
        self.k_bounds = torch.zeros(self.num_pages, heads, 2, head_dim, dtype=dtype, device=device) if bounds else None
        self.block_table = torch.zeros(batch, self.max_blocks, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.lens = [0] * batch
        self._table_host = [[] for _ in range(batch)]
        self._page_cols: dict = {}
        order = torch.arange(self.num_pages)
        if shuffle_seed is not None:
            order = order[torch.randperm(self.num_pages, generator=torch.Generator().manual_seed(shuffle_seed))]
        self._free = order.tolist()[::-1]   # pop() hands out order[0] first

    def _grow_all(self, new_len: int) -> None:
        """Gives every sequence the pages that ``new_len`` tokens need (one table update)."""
        self._grow_each([new_len] * self.batch)

    def _grow_each(self, new_lens: list[int]) -> None:
        """Gives each sequence the pages that its ``new_lens`` tokens need (one table update), or none of them."""
        need = [-(-n // self.page) for n in new_lens]
        if max(need) > self.max_blocks:
            raise ValueError(f"sequences need {max(need)} blocks > max_blocks {self.max_blocks}")
        more = [max(0, n - len(row)) for n, row in zip(need, self._table_host)]
        if not any(more):
            return
        if len(self._free) < sum(more):
            raise RuntimeError("paged KV cache: out of pages")
        first = min(len(row) for row, n in zip(self._table_host, more) if n)
        for row, n in zip(self._table_host, more):
            row.extend(self._free.pop() for _ in range(n))
        self._upload_table(first, max(need))

    def _shrink_each(self, blocks: list[int]) -> None:
        """Takes each sequence's pages past its first ``blocks[b]`` back, in the order that undoes :meth:`_grow_each`."""
        last = max(len(row) for row in self._table_host)
        if all(len(row) == n for row, n in zip(self._table_host, blocks)):
            return
        for row, n in zip(reversed(self._table_host), reversed(blocks)):
            while len(row) > n:
                self._free.append(row.pop())
        self._upload_table(min(blocks), last)

    def _upload_table(self, first: int, last: int) -> None:
        """Brings columns ``first .. last - 1`` of the device's table up to date; 0 where a sequence has no page."""
        cols = [row[first:last] + [0] * (last - max(first, len(row))) for row in self._table_host]
        self.block_table[:, first:last] = self._upload(cols)
        self._page_cols.clear()

    def _upload(self, values) -> torch.Tensor:
        """int32 values on the store's device; from pinned memory, as a copy from other memory waits for the stream."""
        dev = self.kv_lens.device
        return torch.tensor(values, dtype=torch.int32, pin_memory=dev.type == "cuda").to(dev, non_blocking=True)

    def _uniform_len(self, what: str) -> int:
        if any(n != self.lens[0] for n in self.lens):
            raise ValueError(f"{what} needs sequences of one length, got {self.lens}")
        return self.lens[0]

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, counts, *, inv_freq: torch.Tensor | None = None,
               positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
               q: torch.Tensor | None = None, q_weight: torch.Tensor | None = None) -> PagedChunk:
        """Appends ``counts[b]`` new tokens to each sequence b, packed in ``k_new, v_new [N, H, D]`` (on the GPU).

        Keys are normed (``k_weight``) and rotated (``inv_freq``, by their places in the cache or by ``positions``
        int64 ``[N]``) on the way where those are given, and queries ``q [N, Hq, D]`` with them
        (:func:`~sparseattentioninfer_amd.ops.paged_append` or, in 4 bits, ``paged_append_q4``; one launch).  A call that is refused leaves the store as it was.
        Nothing here waits for the GPU.  The lengths are kept on the host, so the call cannot be captured into a graph.
        """
        if self.kv_lens.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKVStore.append advances lengths on the host; a captured graph would not")
        counts = tuple(int(n) for n in counts)
        if len(counts) != self.batch or min(counts) < 0 or sum(counts) != k_new.size(0):
            raise ValueError(f"counts {counts} do not split {k_new.size(0)} tokens over {self.batch} sequences")
        new_lens = [n + t for n, t in zip(self.lens, counts)]
        blocks = [len(row) for row in self._table_host]
        self._grow_each(new_lens)
        try:
            if min(counts) == max(counts) > 0:
                cu = torch.arange(0, k_new.size(0) + 1, counts[0], dtype=torch.int32, device=self.kv_lens.device)
            else:
                cu = self._upload([0, *accumulate(counts)])
            if min(new_lens) == max(new_lens):
                self.kv_lens.fill_(new_lens[0])
            else:
                self.kv_lens.copy_(self._upload(new_lens))
            if self.bits == 4 and k_new.dtype != self.dtype:
                raise ValueError(f"tensors of {k_new.dtype} for a store of {self.dtype}")
            write = ops.paged_append_q4 if self.bits == 4 else ops.paged_append
            q_out = write(k_new, v_new, self.k_pages, self.v_pages, self.block_table, cu, self.kv_lens,
                          inv_freq=inv_freq, positions=positions, k_weight=k_weight, eps=eps, k_bounds=self.k_bounds,
                          q=q, q_weight=q_weight)
        except BaseException:
            self._shrink_each(blocks)
            self.kv_lens.copy_(torch.tensor(self.lens, dtype=torch.int32))
            raise
        self.lens = new_lens
        return PagedChunk(cu, counts, q_out)

    def refresh_bounds(self, start: int) -> None:
        """Key bounds of the pages that hold the tokens from position ``start`` on, from their keys: for those who write
        pages themselves, as a captured decode does (``append`` and ``write`` keep the bounds)."""
        n = self._uniform_len("refresh_bounds")
        first, last = start // self.page, -(-n // self.page)
        if self.k_bounds is None or first >= last:
            return
        pages = self.block_table[:, first:last].long()                         # [B, nb]
        if self.bits == 4:                                                      # what the keys are read back as
            t = n - first * self.page
            k = torch.zeros(self.batch, (last - first) * self.page, self.heads, self.head_dim, dtype=self.dtype,
                            device=self.kv_lens.device)
            k[:, :t] = self._read(t)[0].unflatten(0, (self.batch, t))
            k = k.unflatten(1, (last - first, self.page)).transpose(2, 3)
        else:
            k = self.k_pages[pages]                                             # [B, nb, H, page, D]
        pos = torch.arange(first * self.page, last * self.page, device=k.device).view(-1, 1, self.page, 1)
        held = (pos < n) & ~k.isnan()
        lo, hi = torch.where(held, k, math.inf).amin(3), torch.where(held, k, -math.inf).amax(3)
        self.k_bounds[pages] = torch.stack([lo, hi], dim=3)

    def _read(self, t: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The last ``t`` tokens of each sequence of a 4-bit store, ``[B * t, H, D]`` keys and values."""
        cu = torch.arange(self.batch + 1, dtype=torch.int32, device=self.kv_lens.device) * t
        return ops.paged_read_q4(self.k_pages, self.v_pages, self.block_table, cu, self.kv_lens, rows=self.batch * t,
                                 head_dim=self.head_dim, dtype=self.dtype)

    def _page_col(self, lb: int) -> torch.Tensor:
        """Pages of logical block ``lb`` for every sequence, as a device index tensor (cached)."""
        col = self._page_cols.get(lb)
        if col is None:
            col = self.block_table[:, lb].long()
            self._page_cols[lb] = col
        return col

    def write(self, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Appends ``[B, H, t, D]`` K/V at every sequence's end (all sequences advance by t)."""
        B, H, t, D = k_new.shape
        if (B, H, D) != (self.batch, self.heads, self.head_dim) or v_new.shape != k_new.shape:
            raise ValueError(f"write of {tuple(k_new.shape)} into a [{self.batch}, {self.heads}, *, "
                             f"{self.head_dim}] store")
        start = self._uniform_len("write")
        if self.k_bounds is not None or self.bits == 4:      # the append kernel keeps the bounds, and quantises
            k, v = (x.to(self.dtype).transpose(1, 2).reshape(B * t, H, D) for x in (k_new, v_new))
            self.append(k, v, [t] * B)
            return
        self._grow_all(start + t)
        if t == 1:   # decode: one slot of one page per sequence
            idx = self._page_col(start // self.page)
            slot = start % self.page
            self.k_pages[idx, :, slot] = k_new[:, :, 0].to(self.k_pages.dtype)
            self.v_pages[idx, :, slot] = v_new[:, :, 0].to(self.v_pages.dtype)
        else:
            pos = torch.arange(start, start + t, device=k_new.device)
            pages = self.block_table[:, pos // self.page].long()          # [B, t]
            slots = (pos % self.page).expand(B, t)                         # [B, t]
            # advanced indices on dims 0 and 2 put [B, t] first: [B, t, H, D]
            self.k_pages[pages, :, slots] = k_new.transpose(1, 2).to(self.k_pages.dtype)
            self.v_pages[pages, :, slots] = v_new.transpose(1, 2).to(self.v_pages.dtype)
        self.lens = [start + t] * B
        self.kv_lens.fill_(start + t)

    def gather(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Contiguous ``[B, H, T, D]`` copies of the cached K/V (slow path for generic callers)."""
        T = self._uniform_len("gather")
        if self.bits == 4:
            k, v = (x.view(self.batch, T, self.heads, self.head_dim).transpose(1, 2).contiguous() for x in self._read(T))
            return k, v
        nb = -(-T // self.page)
        pages = self.block_table[:, :nb].long()                         # [B, nb]
        k = self.k_pages[pages].permute(0, 2, 1, 3, 4).reshape(self.batch, self.heads, nb * self.page, -1)
        v = self.v_pages[pages].permute(0, 2, 1, 3, 4).reshape(self.batch, self.heads, nb * self.page, -1)
        return k[:, :, :T].contiguous(), v[:, :, :T].contiguous()

    def seq_len(self) -> int:
        return self._uniform_len("seq_len")

    def reset(self) -> None:
        """Returns every page to the free list (contents are left as they are)."""
        for row in self._table_host:
            self._free.extend(reversed(row))
            row.clear()
        self._page_cols.clear()
        self.lens = [0] * self.batch
        self.kv_lens.zero_()
