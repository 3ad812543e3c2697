"""Callers of the chunk operators: the ragged paged store, the backend over packed chunks, and Qwen3 with the
block_topk pattern, prompt, chunk and single tokens, against float64 on the pages that they leave."""
import pytest
import torch

from sparseattentioninfer_amd import ops
from sparseattentioninfer_amd.attention import HipBlockSparseBackend
from sparseattentioninfer_amd.models import PagedKVStore
from sparseattentioninfer_amd.patterns import BlockTopKPattern, DenseCausalPattern
from sparseattentioninfer_amd.qwen3 import PagedKVCache
from sparseattentioninfer_amd.qwen3.graph_decode import GraphDecoder
from sparseattentioninfer_amd.qwen3.runtime import build_model, greedy_generate, qwen3_config
from tests.chunk_reference import Ragged, assert_rotated, attention, bounds_of, randn, rotate, select

pytestmark = pytest.mark.gpu


def _view(store, counts):
    """The store's cache as the float64 forms read it."""
    r = Ragged.__new__(Ragged)
    r.q_lens, r.lens, r.page, r.Hkv, r.D, r.dtype = list(counts), list(store.lens), store.page, store.heads, store.head_dim, \
        store.k_pages.dtype
    r.table, r.k_pages, r.v_pages = store.block_table.cpu(), store.k_pages.cpu(), store.v_pages.cpu()
    r.N = sum(counts)
    return r


def _check(got, want, tol, live, what):
    err = (got.cpu().double() - want).abs()
    bad = ~(err <= tol) & live[:, None, None]
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {(err / tol)[live].max():.2f} of it"


def test_store_append_and_backend_in_steps():
    """Three sequences that grow unevenly; every step attends densely and over selected pages."""
    store = PagedKVStore(3, 2, 64, 900, page=32, num_pages=70, shuffle_seed=1, bounds=True)
    be = HipBlockSparseBackend()
    total = [0, 0, 0]
    for step, counts in enumerate([(300, 0, 65), (1, 1, 1), (0, 200, 1), (1, 1, 1), (130, 2, 0)]):
        print("[chunk-callers] store step", step, counts, flush=True)
        n = sum(counts)
        q, k, v = (randn(n, h, 64, seed=10 * step + i) for i, h in enumerate((4, 2, 2)))
        chunk = store.append(k.cuda(), v.cuda(), counts, q=q.cuda())
        total = [a + b for a, b in zip(total, counts)]
        assert store.lens == total == store.kv_lens.tolist() and chunk.single_tokens == (counts == (1, 1, 1))
        r = _view(store, counts)
        assert torch.equal(chunk.q.cpu(), q)      # no norm, no rotation
        at = 0
        for b, t in enumerate(counts):
            assert torch.equal(r.cached(r.k_pages, b, total[b])[:, total[b] - t:], k[at:at + t].double().transpose(0, 1))
            at += t
        used = torch.cat([r.table[b, :-(-total[b] // 32)] for b in range(3)]).long()
        assert torch.equal(store.k_bounds.cpu()[used], bounds_of(r)[used])
        _check(be.forward_packed(chunk.q, store, chunk, DenseCausalPattern().build(q, q)), *attention(r, q), "dense")
        pat = BlockTopKPattern(2, block_size=32, sink=1, recent=1)
        out = be.forward_packed(chunk.q, store, chunk, pat.build(q, q[None].transpose(1, 2)))
        assert be.last_kernel == ("decode" if chunk.single_tokens else "chunk") and be.actual_backend == "hip_block_sparse"
        sel, off = select(r, q, store.k_bounds.cpu(), top_k=2, sink=1, recent=1, tokens=chunk.single_tokens)
        _check(out, *attention(r, q, sel, off), "block_topk")


def test_store_write_keeps_bounds_and_backend_refuses_what_it_cannot_run():
    store = PagedKVStore(2, 2, 64, 200, page=64, bounds=True)
    for t in (70, 1, 5):
        k, v = randn(2, 2, t, 64, seed=t).cuda(), randn(2, 2, t, 64, seed=t + 1).cuda()
        store.write(k, v)
    r = _view(store, (0, 0))
    pages = r.table[:, :2].flatten().long()
    assert store.seq_len() == 76 and torch.equal(store.k_bounds.cpu()[pages], bounds_of(r)[pages])
    assert torch.equal(store.gather()[0][:, :, 71:], k)
    be = HipBlockSparseBackend()
    chunk = store.append(randn(2, 2, 64, seed=9).cuda(), randn(2, 2, 64, seed=8).cuda(), (1, 1))
    q = randn(2, 4, 64, seed=7).cuda()
    with pytest.raises(ValueError, match="page"):
        be.forward_packed(q, store, chunk, BlockTopKPattern(2, block_size=32).build(q[None], q[None]))
    plain = PagedKVStore(2, 2, 64, 200, page=64)
    with pytest.raises(ValueError, match="bounds"):
        be.forward_packed(q, plain, chunk, BlockTopKPattern(2).build(q[None], q[None]))


class _Recorder(HipBlockSparseBackend):
    def __init__(self):
        super().__init__()
        self.calls = []

    def forward_packed(self, q, store, chunk, pattern):
        out = super().forward_packed(q, store, chunk, pattern)
        r = _view(store, chunk.counts)
        self.calls.append((q.cpu(), r, store.k_bounds.cpu(), chunk.single_tokens, out.cpu()))
        return out


@torch.no_grad()
@pytest.mark.parametrize("head_dim", [128, 64])
def test_qwen3_block_topk(head_dim):
    """A prompt, a chunk after it and two single tokens: projections through the norm, rotation and append into the
    pages, and every layer's attention over the selected pages."""
    print("[chunk-callers] qwen3 block_topk", head_dim, flush=True)
    cfg = qwen3_config(pattern="block_topk", block_size=32, vocab_size=512, hidden_size=256, intermediate_size=256,
                       num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=head_dim)
    cfg.sparse_attention_topk_pages, cfg.sparse_attention_recent_pages = 3, 1
    model = build_model(cfg, seed=3)
    recs = [_Recorder() for _ in model.model.layers]
    seen = []
    for layer, rec in zip(model.model.layers, recs):
        a = layer.self_attn
        a.sparse_backends = {a.backend_name: rec}
        a.register_forward_pre_hook(lambda m, args, kw: seen.append((m, kw["hidden_states"])), with_kwargs=True)
    cache = PagedKVCache(2, 400, page=32, shuffle_seed=4, bounds=True)
    g = torch.Generator().manual_seed(5)
    at = 0
    for t in (200, 70, 1, 1):
        ids = torch.randint(0, 512, (2, t), generator=g).cuda()
        out = model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1)
        assert torch.isfinite(out.logits).all()
        pos = torch.arange(at, at + t).repeat(2)
        at += t
        for (attn, x), rec in zip(seen, recs):
            q, r, bounds, tokens, got = rec.calls[-1]
            inv = attn._inv_freq.cpu()
            eps = cfg.rms_norm_eps
            proj = lambda m: m(x).view(2 * t, -1, head_dim).cpu()
            assert_rotated(q, *rotate(proj(attn.q_proj), attn.q_norm.weight.cpu(), pos, inv, eps), "q")
            keys = torch.cat([r.cached(r.k_pages, b, at)[:, at - t:].transpose(0, 1) for b in range(2)]).to(torch.bfloat16)
            assert_rotated(keys, *rotate(proj(attn.k_proj), attn.k_norm.weight.cpu(), pos, inv, eps), "k")
            sel, off = select(r, q, bounds, top_k=3, sink=1, recent=1, tokens=tokens)
            _check(got, *attention(r, q, sel, off), f"layer attention, {t} new tokens")
        seen.clear()
    assert cache.get_seq_length() == at


@torch.no_grad()
def test_generate_with_block_topk_and_the_graph_decoders_refusal():
    cfg = qwen3_config(pattern="block_topk", vocab_size=512, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=128, sparse_layers=[1])
    model = build_model(cfg, seed=6)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(7)).cuda()
    res = greedy_generate(model, ids, 3)
    assert res["tokens"].shape == (2, 4) and res["cache"].get_seq_length() == 153
    with pytest.raises(ValueError, match="block_topk"):
        GraphDecoder(model, res["cache"], res["tokens"][:, -1], 153)


def test_other_gpu_streams_are_the_current_streams_of_the_tensors():
    """Work goes to the stream that is current where the call is made."""
    store = PagedKVStore(1, 1, 64, 64, page=16)
    side = torch.cuda.Stream()
    k = randn(40, 1, 64, seed=11).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        chunk = store.append(k, k, (40,))
        out = ops.paged_chunk_attn(k.expand(40, 2, 64).contiguous(), store.k_pages, store.v_pages, store.block_table,
                                   chunk.cu_seqlens, store.kv_lens)
    side.synchronize()
    r = _view(store, (40,))
    q = k.cpu().expand(40, 2, 64)
    _check(out, *attention(r, q), "side stream")
