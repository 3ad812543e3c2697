"""The paged store's bookkeeping on the CPU: a refused append changes nothing, sequences of unequal page counts grow
into pages of their own, and what the block_topk pattern's refusals say."""
from types import SimpleNamespace

import pytest
import torch

from sparseattentioninfer_amd import _lib
from sparseattentioninfer_amd.attention import get_backend
from sparseattentioninfer_amd.models import PagedKVStore
from sparseattentioninfer_amd.patterns import BlockTopKPattern
from sparseattentioninfer_amd.qwen3.paged_cache import PagedKVLayer

BF = torch.bfloat16


def _state(st):
    return (list(st.lens), st.kv_lens.tolist(), [list(r) for r in st._table_host], list(st._free), st.block_table.tolist())


def test_a_refused_append_leaves_the_store_as_it_was():
    """The operator runs on the GPU only, so here it refuses each call, with pages to hand out and without."""
    st = PagedKVStore(2, 1, 64, 100, page=16, device="cpu", shuffle_seed=3)
    before = _state(st)
    k = torch.zeros(5, 1, 64, dtype=BF)
    for counts in ([3, 2], [5, 0], [0, 5]):
        with pytest.raises(AssertionError, match="GPU"):
            st.append(k, k, counts)
        assert _state(st) == before
    st.write(torch.ones(2, 1, 20, 64, dtype=BF), torch.ones(2, 1, 20, 64, dtype=BF))
    before = _state(st)
    with pytest.raises(AssertionError, match="GPU"):
        st.append(torch.zeros(40, 1, 64, dtype=BF), torch.zeros(40, 1, 64, dtype=BF), [1, 39])
    assert _state(st) == before and st.seq_len() == 20


def test_a_layer_whose_first_append_is_refused_has_no_store():
    """It would keep the refused tensors' type and device."""
    layer = PagedKVLayer(64, page=16)
    x = torch.zeros(4, 1, 64)
    with pytest.raises(AssertionError):
        layer.append(x, x, x, [4])
    assert layer.store is None and not layer.is_initialized and layer.get_seq_length() == 0


def test_sequences_with_unequal_page_counts_grow_into_their_own_pages():
    st = PagedKVStore(2, 1, 64, 200, page=16, device="cpu", dtype=torch.float32)
    st._grow_each([70, 3])
    k = torch.arange(2 * 60, dtype=torch.float32).view(2, 1, 60, 1).expand(2, 1, 60, 64) + 1
    st.write(k, -k)
    assert [len(r) for r in st._table_host] == [5, 4] and len(set(sum(st._table_host, []))) == 9
    got_k, got_v = st.gather()
    assert torch.equal(got_k, k) and torch.equal(got_v, -k)
    st._grow_all(100)
    assert [len(r) for r in st._table_host] == [7, 7] and len(set(sum(st._table_host, []))) == 14
    for b in range(2):
        assert st.block_table[b, :7].tolist() == st._table_host[b]


def test_a_block_topk_caller_is_told_where_it_runs():
    be = get_backend("hip_block_sparse")
    pattern = BlockTopKPattern(4).build(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))
    q = SimpleNamespace(is_cuda=True, dtype=BF, size=lambda d: 64)
    assert "forward_packed" in be.unsupported_reason(q, pattern)
    with pytest.raises(NotImplementedError, match="forward_packed"):
        be._schedule(1, 64, 1, "cpu", pattern)
