"""Callers of the 4-bit cache: the paged store, the backend over it, the Hugging Face cache and Qwen3's generation, eager and by
graph, against float64 over what their pages hold."""
import pytest
import torch

from sparseattentioninfer_amd.attention import HipBlockSparseBackend
from sparseattentioninfer_amd.models import PagedKVStore
from sparseattentioninfer_amd.patterns import BlockTopKPattern, DenseCausalPattern, SeededBigBirdPattern
from sparseattentioninfer_amd.qwen3 import PagedKVCache
from sparseattentioninfer_amd.qwen3.graph_decode import GraphDecoder
from sparseattentioninfer_amd.qwen3.runtime import build_model, greedy_generate, qwen3_config
from tests.chunk_reference import randn, select
from tests.q4_reference import Q4Ragged, assert_attention, quantise, unpack, value_of

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[q4-callers]", *msg, flush=True)


def _view(store, counts):
    """The store's cache as the float64 forms read it."""
    r = Q4Ragged.__new__(Q4Ragged)
    r.q_lens, r.lens, r.page, r.Hkv, r.D, r.dtype = list(counts), list(store.lens), store.page, store.heads, store.head_dim, store.dtype
    r.table, r.k4, r.v4 = store.block_table.cpu(), store.k_pages.cpu(), store.v_pages.cpu()
    r.k_pages, r.v_pages = (unpack(p, r.page, r.D, r.dtype, v) for p, v in ((r.k4, False), (r.v4, True)))
    r.held = torch.zeros(r.k4.size(0), r.page, dtype=torch.bool)
    for b, n in enumerate(r.lens):
        for lb in range(-(-n // r.page)):
            r.held[r.table[b, lb].item(), :min(r.page, n - lb * r.page)] = True
    r.N = sum(counts)
    return r


def _bounds_of(r):
    """[P, Hkv, 2, D] of the keys as they are read back."""
    keep = r.held[:, None, :, None]
    k = r.k_pages.float().to(r.dtype)
    inf = torch.finfo(r.dtype).max
    return torch.stack([torch.where(keep, k, inf).amin(2), torch.where(keep, k, -inf).amax(2)], dim=2)


def test_store_append_and_backend_in_steps():
    """Three sequences that grow unevenly; every step attends densely and over selected pages."""
    for dtype, D in ((BF, 64), (HF, 128)):
        store = PagedKVStore(3, 2, D, 900, page=32, num_pages=70, shuffle_seed=1, bounds=True, bits=4, dtype=dtype)
        assert store.k_pages.numel() * 16 == 70 * 2 * 32 * D * 10
        be = HipBlockSparseBackend()
        total = [0, 0, 0]
        for step, counts in enumerate([(300, 0, 65), (1, 1, 1), (0, 200, 1), (1, 1, 1), (130, 2, 0)]):
            _say("store step", step, counts)
            n = sum(counts)
            q, k, v = (randn(n, h, D, seed=10 * step + i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
            chunk = store.append(k.cuda(), v.cuda(), counts, q=q.cuda())
            total = [a + b for a, b in zip(total, counts)]
            assert store.lens == total == store.kv_lens.tolist() and chunk.single_tokens == (counts == (1, 1, 1))
            r = _view(store, counts)
            at = 0
            for b, t in enumerate(counts):
                for pool, new in ((r.k_pages, k), (r.v_pages, v)):
                    assert torch.equal(r.cached(pool, b, total[b])[:, total[b] - t:], value_of(*quantise(new[at:at + t])).transpose(0, 1))
                at += t
            used = torch.cat([r.table[b, :-(-total[b] // 32)] for b in range(3)]).long()
            assert torch.equal(store.k_bounds.cpu()[used], _bounds_of(r)[used])
            assert_attention(be.forward_packed(chunk.q, store, chunk, DenseCausalPattern().build(q, q)), r, q, what="dense")
            pat = BlockTopKPattern(2, block_size=32, sink=1, recent=1)
            out = be.forward_packed(chunk.q, store, chunk, pat.build(q, q[None].transpose(1, 2)))
            assert be.last_kernel == ("decode" if chunk.single_tokens else "chunk") and be.actual_backend == "hip_block_sparse"
            sel, off = select(r, q, store.k_bounds.cpu(), top_k=2, sink=1, recent=1, tokens=chunk.single_tokens)
            assert_attention(out, r, q, sel, off, "block_topk")


def test_store_write_gather_and_bounds():
    _say("store write, gather")
    store = PagedKVStore(2, 2, 128, 200, page=64, bounds=True, bits=4)
    parts = []
    for t in (70, 1, 5):
        k, v = randn(2, 2, t, 128, seed=t), randn(2, 2, t, 128, seed=t + 1)
        store.write(k.cuda(), v.cuda())
        parts.append((k, v))
    assert store.seq_len() == 76
    for got, x in zip(store.gather(), zip(*parts)):
        assert torch.equal(got.cpu(), value_of(*quantise(torch.cat(x, dim=2))).float().to(BF))
    r = _view(store, (0, 0))
    pages = r.table[:, :2].flatten().long()
    want = _bounds_of(r)[pages]
    assert torch.equal(store.k_bounds.cpu()[pages], want)
    store.k_bounds.fill_(7.0)
    store.refresh_bounds(0)
    assert torch.equal(store.k_bounds.cpu()[pages], want)
    store.reset()
    assert store.gather()[0].shape == (2, 2, 0, 128)


def test_backend_decodes_a_pattern_over_4_bits():
    """forward_paged: a schedule of one CSR row per KV group, and per query head."""
    _say("forward_paged")
    for rows in (2, 8):
        store = PagedKVStore(2, 2, 128, 600, page=64, bits=4, shuffle_seed=2)
        store.write(randn(2, 2, 500, 128, seed=1).cuda(), randn(2, 2, 500, 128, seed=2).cuda())
        q = randn(2, 8, 1, 128, seed=3)
        be = HipBlockSparseBackend()
        pattern = SeededBigBirdPattern(rows=rows, block_size=64, window=2, global_blocks=1, random_blocks=2, seed=4)
        meta = pattern.build(q.cuda(), torch.empty(2, 2, 500, 0, device="cuda"), causal=True)
        out = be.forward_paged(q.cuda(), store, meta)
        pairs, offsets, _ = be._schedule(1, 500, 2, q.device, meta)
        sel = pairs.cpu()[None].expand(2, -1, -1)
        off = offsets.cpu()[None].expand(2, -1, -1)
        r = _view(store, (1, 1))
        for h in range(0, 8, 8 // rows):
            heads = slice(h, h + 8 // rows)
            one = Q4Ragged.__new__(Q4Ragged)
            one.__dict__ = dict(r.__dict__, Hkv=1)
            for x in ("k_pages", "v_pages", "k4", "v4"):
                setattr(one, x, getattr(r, x)[:, h // 4:h // 4 + 1])
            row = h * rows // 8
            assert_attention(out[:, heads, 0], one, q[:, heads, 0], sel[:, row:row + 1], off[:, row:row + 1], f"heads {heads}")
        with pytest.raises(ValueError, match="float16"):
            be.forward_paged(q.half().cuda(), store, meta)


def test_store_refuses_other_types():
    _say("store refusals")
    store = PagedKVStore(1, 1, 64, 64, page=16, bits=4, dtype=HF)
    x = randn(3, 1, 64, seed=1).cuda()
    with pytest.raises(ValueError, match="bfloat16"):
        store.append(x, x, [3])
    assert store.lens == [0]
    store.append(x.half(), x.half(), [3])
    with pytest.raises(ValueError, match="bfloat16"):
        HipBlockSparseBackend().forward_packed(x, store, store.append(x.half(), x.half(), [3]), DenseCausalPattern().build(x, x))


def _config(pattern, **more):
    return qwen3_config(pattern=pattern, vocab_size=512, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                        num_attention_heads=8, num_key_value_heads=2, head_dim=128, **more)


@torch.no_grad()
@pytest.mark.parametrize("pattern", ["dense", "seeded_bigbird", "block_topk"])
def test_qwen3_generates_over_4_bits(pattern):
    _say("qwen3", pattern)
    model = build_model(_config(pattern), seed=6)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(7)).cuda()
    res = greedy_generate(model, ids, 3, cache_bits=4)
    assert res["tokens"].shape == (2, 4) and res["cache"].get_seq_length() == 153 and res["cache"].bits == 4
    assert all(l.store.k_pages.dtype == torch.uint8 for l in res["cache"].layers)
    with pytest.raises(ValueError, match="4 bits"):
        greedy_generate(model, ids, 1, cache="dynamic", cache_bits=4)


@torch.no_grad()
def test_a_chunk_after_a_prompt_attends_what_the_pages_hold():
    """Hugging Face's update() and the chunked prefill gather the read-back values."""
    _say("chunked prefill")
    model = build_model(_config("dense"), seed=8)
    cache = PagedKVCache(2, 300, bits=4)
    g = torch.Generator().manual_seed(9)
    for t in (100, 40, 1):
        out = model(input_ids=torch.randint(0, 512, (2, t), generator=g).cuda(), past_key_values=cache, use_cache=True, logits_to_keep=1)
        assert torch.isfinite(out.logits).all()
    assert cache.get_seq_length() == 141
    k, v = randn(2, 2, 3, 128, seed=1).cuda(), randn(2, 2, 3, 128, seed=2).cuda()
    kk, vv = cache.layers[0].update(k, v)
    assert kk.shape == (2, 2, 144, 128)
    assert torch.equal(kk[:, :, 141:].cpu(), value_of(*quantise(k.cpu())).float().to(BF))


@torch.inference_mode()
def test_graph_decode_modules_equal_the_eager_decode():
    """Positions 150..157 lie in one page, so selections and splits are the eager ones and the logits agree bit for bit."""
    _say("graph, modules")
    cfg = _config("seeded_bigbird")
    model = build_model(cfg, seed=1)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(8)).cuda()
    ce, cg = (PagedKVCache(2, 160, page=64, shuffle_seed=4, bits=4) for _ in "ab")
    first = [model(input_ids=ids, past_key_values=c, use_cache=True, logits_to_keep=1).logits[:, -1].argmax(-1) for c in (ce, cg)]
    dec = GraphDecoder(model, cg, first[1], 158, keep_logits=True, fused=False)
    nxt = first[0]
    for s in range(8):
        want = model(input_ids=nxt[:, None], past_key_values=ce, use_cache=True, logits_to_keep=1).logits[:, -1]
        got = dec.step().clone()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, want), s
        nxt = want.argmax(-1)
        assert torch.equal(got, nxt), s
    assert dec.graph is not None
    dec.finish()
    for a, b in zip(ce.layers, cg.layers):
        for x, y in zip(a.store.gather(), b.store.gather()):
            assert torch.equal(x, y)


@torch.inference_mode()
def test_graph_decode_fused_writes_the_eager_cache():
    """The first layer's cache of a fused run against the eager one, tokens given.  Projections by other products differ by a
    step of theirs; keys that Hugging Face then rounds five times and the append kernel once differ by at most 8 half steps
    of their terms in all (the sum of two magnitudes of 128-dim normed heads, below 2 * 128 ** 0.5), and so by that and half
    a step of each scale when held in 4 bits."""
    _say("graph, fused")
    cfg = _config("dense")
    model = build_model(cfg, seed=2)
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(8)).cuda()
    ce, cg = (PagedKVCache(2, 170, page=64, shuffle_seed=4, bits=4) for _ in "ab")
    nxt = [model(input_ids=ids, past_key_values=c, use_cache=True, logits_to_keep=1).logits[:, -1].argmax(-1) for c in (ce, cg)][0]
    dec = GraphDecoder(model, cg, nxt, 165, keep_logits=True)
    for s in range(15):
        dec.ids.copy_(nxt)
        logits = model(input_ids=nxt[:, None], past_key_values=ce, use_cache=True, logits_to_keep=1).logits[:, -1]
        dec.step()
        torch.cuda.synchronize()
        assert torch.isfinite(dec.logits).all()
        nxt = logits.argmax(-1)
    dec.finish()
    (ke, ve), (kg, vg) = ce.layers[0].store.gather(), cg.layers[0].store.gather()
    assert ke.shape == kg.shape == (2, 2, 165, 128)
    assert torch.equal(ke[:, :, :150], kg[:, :, :150])
    tol = 8 * 2.0 ** -9 * 2 * 128 ** 0.5
    x = ke[:, :, 150:].float().unflatten(-1, (4, 32))
    step = (x.amax(-1) - x.amin(-1) + 2 * tol) / 15
    err = (ke - kg)[:, :, 150:].float().abs().unflatten(-1, (4, 32)).amax(-1)
    assert (err <= step + tol).all()
    v_step = (ve.float().unflatten(-1, (4, 32)).amax(-1) - ve.float().unflatten(-1, (4, 32)).amin(-1)) / 15
    assert ((ve - vg).float().abs().unflatten(-1, (4, 32)).amax(-1) <= 1.1 * v_step + 2.0 ** -8 * ve.float().abs().max()).all()
