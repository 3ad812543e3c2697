"""What Qwen3 attends over a 4-bit cache, eager and by graph: each layer's attention against float64 over what its pages hold."""
import pytest
import torch

from sparseattentioninfer_amd.attention import HipBlockSparseBackend
from sparseattentioninfer_amd.qwen3 import PagedKVCache
from sparseattentioninfer_amd.qwen3.graph_decode import GraphDecoder
from sparseattentioninfer_amd.qwen3.runtime import build_model, greedy_generate, qwen3_config
from tests.q4_bounds import forms, good_rows
from tests.q4_reference import Q4Ragged, unpack

pytestmark = pytest.mark.gpu
H, HKV, D = 8, 2, 128


def _say(*msg):
    print("[q4-model]", *msg, flush=True)


def _config(pattern, **more):
    return qwen3_config(pattern=pattern, vocab_size=512, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                        num_attention_heads=H, num_key_value_heads=HKV, head_dim=D, **more)


def _ids(B, T, seed=7):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def _view(store, lens, new):
    """The store's pages as the float64 forms read them, with `lens` tokens of which the last `new` are queries."""
    r = Q4Ragged.__new__(Q4Ragged)
    r.q_lens, r.lens, r.page, r.Hkv, r.D, r.dtype = [new] * len(lens), list(lens), store.page, store.heads, store.head_dim, store.dtype
    r.table, r.k4, r.v4, r.N = store.block_table.cpu(), store.k_pages.cpu(), store.v_pages.cpu(), new * len(lens)
    r.k_pages, r.v_pages = (unpack(p, r.page, r.D, r.dtype, v) for p, v in ((r.k4, False), (r.v4, True)))
    return r


def _lists(sel, off, B):
    return (x.cpu().expand(B, *x.shape[1:]) for x in (sel, off))


def _assert(out, store, lens, new, q, sel, off, what, codes=(True,)):
    """out, q [B * new, H, D]."""
    r = _view(store, lens, new)
    bounds = [forms(r, q.cpu(), sel, off, codes=c) for c in codes]
    good = good_rows(out, bounds)
    assert good.all(), f"{what}: {int((~good).sum())} of {good.numel()} rows"


@torch.inference_mode()
@pytest.mark.parametrize("pattern", ["dense", "seeded_bigbird"])
@pytest.mark.parametrize("fused", [True, False])
def test_graph_decode_attends_its_pages(pattern, fused):
    """Every step of a run, eager and replayed: what the last layer attends, and that its queries are the step's own."""
    model = build_model(_config(pattern, window=1, global_blocks=1, random_blocks=1), seed=2)
    cache = PagedKVCache(2, 420, page=64, shuffle_seed=4, bits=4)
    nxt = model(input_ids=_ids(2, 380), past_key_values=cache, use_cache=True, logits_to_keep=1).logits[:, -1].argmax(-1)
    calls = []
    attend = GraphDecoder._attend

    class Recorded(GraphDecoder):
        def _attend(self, q, store, sched, kv_lens, out=None):
            got = attend(self, q, store, sched, kv_lens, out)
            calls.append((q, store, sched, kv_lens, got))
            return got

    dec = Recorded(model, cache, nxt, 392, fused=fused)
    last_q = None
    for s in range(10):
        _say("graph", pattern, fused, s)
        calls.clear() if dec.graph is None else None
        dec.step()
        torch.cuda.synchronize()
        q, store, sched, kv_lens, got = calls[-1]
        assert store is dec.stores[1] and kv_lens.tolist() == [381 + s] * 2
        sel, off = _lists(sched.sel, sched.sel_off, 2)
        listed = (off[..., 1] - off[..., 0]).unique().tolist()
        assert listed == [6 if 381 + s <= 384 else 7] if pattern == "dense" else max(listed) < 6
        _assert(got, store, kv_lens.tolist(), 1, q, sel, off, f"{pattern} step {s}")
        assert last_q is None or not torch.equal(last_q, q)
        last_q = q.clone()
    assert dec.graph is not None


@torch.inference_mode()
@pytest.mark.parametrize("pattern", ["dense", "seeded_bigbird", "block_topk"])
def test_generated_tokens_attend_their_pages(pattern, monkeypatch):
    """Every layer's attention of every generated token; 230 tokens are four pages, all of which block_topk keeps."""
    _say("generate", pattern)
    calls = []
    for name in ("forward_paged", "forward_packed"):
        run = getattr(HipBlockSparseBackend, name)

        def record(self, q, store, *args, run=run):
            out = run(self, q, store, *args)
            calls.append((self, q, store, args, store.kv_lens.tolist(), out))
            return out

        monkeypatch.setattr(HipBlockSparseBackend, name, record)
    model = build_model(_config(pattern), seed=6)
    res = greedy_generate(model, _ids(2, 227), 3, cache_bits=4)
    if pattern == "block_topk":              # the prompt is attended from its pages too
        for be, q, store, args, lens, out in calls[:2]:
            assert lens == [227, 227]
            _assert(out, store, lens, 227, q, None, None, "prompt", codes=(True, False))
        calls = calls[2:]
    assert len(calls) == 3 * 2
    for i, (be, q, store, args, lens, out) in enumerate(calls):
        assert lens == [228 + i // 2] * 2 and store is res["cache"].layers[i % 2].store
        sel = off = None
        if pattern == "seeded_bigbird":
            pairs, offsets, _ = be._schedule(1, lens[0], HKV, q.device, args[0])
            sel, off = _lists(pairs[None], offsets[None], 2)
        q, out = (x.reshape(2, H, D) for x in (q, out))
        _assert(out, store, lens, 1, q, sel, off, f"{pattern} call {i}")


@torch.inference_mode()
def test_a_chunk_after_a_prompt_attends_what_was_read_back(monkeypatch):
    """A prompt by itself attends its own keys and values; the chunk after it those of the whole cache, its own among them, as
    they are read back; a single token the pages."""
    _say("chunk after a prompt")
    seen, paged = [], []
    forward, forward_paged = HipBlockSparseBackend.forward, HipBlockSparseBackend.forward_paged

    def record(self, q, k, v, pattern):
        seen.append((k, v))
        return forward(self, q, k, v, pattern)

    def record_paged(self, q, store, pattern):
        out = forward_paged(self, q, store, pattern)
        paged.append((q, store, store.kv_lens.tolist(), out))
        return out

    monkeypatch.setattr(HipBlockSparseBackend, "forward", record)
    monkeypatch.setattr(HipBlockSparseBackend, "forward_paged", record_paged)
    model = build_model(_config("dense"), seed=8)
    cache = PagedKVCache(2, 300, bits=4)
    for t in (100, 40, 1):
        model(input_ids=_ids(2, t, seed=t), past_key_values=cache, use_cache=True, logits_to_keep=1)
    assert len(seen) == 4 and len(paged) == 2
    for i, layer in enumerate(cache.layers):
        r = _view(layer.store, [141] * 2, 1)
        for j, pages in enumerate((r.k_pages, r.v_pages)):
            held = torch.stack([r.cached(pages, b, 140) for b in range(2)]).float().to(r.dtype)
            prompt, chunk = seen[i][j].cpu(), seen[2 + i][j].cpu()
            assert torch.equal(chunk, held)
            assert prompt.shape[2] == 100 and not torch.equal(prompt, held[:, :, :100])      # not quantised
            span = prompt.float().unflatten(-1, (4, 32))
            step = (span.amax(-1) - span.amin(-1)) / 15
            err = (prompt.double() - torch.stack([r.cached(pages, b, 100) for b in range(2)])).abs().unflatten(-1, (4, 32)).amax(-1)
            assert (err <= step.double() / 2 * (1 + 2.0 ** -7)).all()
        q, store, lens, out = paged[i]
        assert store is layer.store and lens == [141, 141]
        _assert(out[:, :, 0], store, lens, 1, q[:, :, 0], None, None, f"layer {i}")
