"""Callers of the paged append on the GPU: positions that are given, refusals that leave the cache as it was, no upload
that waits for the stream, key bounds after a captured decode."""
import pytest
import torch
from transformers.models.qwen3.modeling_qwen3 import apply_rotary_pos_emb

from sparseattentioninfer_amd import ops
from sparseattentioninfer_amd.attention import HipBlockSparseBackend
from sparseattentioninfer_amd.models import PagedChunk, PagedKVStore
from sparseattentioninfer_amd.qwen3 import PagedKVCache
from sparseattentioninfer_amd.qwen3.graph_decode import GraphDecoder
from sparseattentioninfer_amd.qwen3.runtime import build_model, qwen3_config
from tests.chunk_reference import Ragged, assert_rotated, bounds_of, randn, rotate

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
EPS = 1e-6


def _say(*msg):
    print("[paged-store]", *msg, flush=True)


def _view(store):
    r = Ragged.__new__(Ragged)
    r.lens, r.page, r.Hkv, r.D, r.dtype = list(store.lens), store.page, store.heads, store.head_dim, store.k_pages.dtype
    r.table, r.k_pages, r.v_pages = store.block_table.cpu(), store.k_pages.cpu(), store.v_pages.cpu()
    return r


def _state(st):
    return (list(st.lens), st.kv_lens.tolist(), [list(r) for r in st._table_host], list(st._free), st.block_table.tolist())


def _inv(D):
    return (1.0 / 1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()


@pytest.mark.parametrize("stride", [1, 0, 3])
@pytest.mark.parametrize("D,dtype,norm,bounds", [(128, BF, True, True), (64, HF, False, False)])
def test_append_at_given_positions(D, dtype, norm, bounds, stride):
    """Angles follow ``positions``; places in the cache, and so what attention sees, follow the lengths."""
    _say("positions", D, dtype, norm, bounds, stride)
    q_lens, kv_lens = [40, 0, 1, 100], [40, 5, 300, 131]
    r = Ragged(q_lens, kv_lens, page=32, Hkv=2, D=D, dtype=dtype, seed=600, pad_rows=2, poison=False)
    q, k, v = (randn(r.N, h, D, seed=601 + h, dtype=dtype) for h in (6, 2, 2))
    w = randn(D, seed=610, dtype=dtype, scale=0.3) + 1 if norm else None
    wide = torch.randint(0, 131072, (r.N, max(stride, 1)), generator=torch.Generator().manual_seed(611))
    positions = wide[:1, 0].expand(r.N) if stride == 0 else wide[:, 0]
    dev = wide.cuda()
    dev_positions = dev[:1, 0].expand(r.N) if stride == 0 else dev[:, 0]
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    bd = torch.zeros(kp.size(0), 2, 2, D, dtype=dtype, device="cuda") if bounds else None
    q_out = torch.full((r.N, 6, D), 7.0, dtype=dtype, device="cuda")
    gw = None if w is None else w.cuda()
    ops.paged_append(k.cuda(), v.cuda(), kp, vp, table, cu, lens, inv_freq=_inv(D).cuda(), positions=dev_positions,
                     k_weight=gw, q=q.cuda(), q_weight=gw, q_out=q_out, eps=EPS, k_bounds=bd)
    kp, vp = kp.cpu(), vp.cpu()
    for b, at, t, n in r.rows():
        rows, p = slice(at, at + t), torch.arange(n - t, n)
        phys, slot = r.table[b, p // 32].long(), p % 32
        assert_rotated(q_out[rows], *rotate(q[rows], w, positions[rows], _inv(D), EPS), f"q of {b}")
        assert_rotated(kp[phys, :, slot], *rotate(k[rows], w, positions[rows], _inv(D), EPS), f"k of {b}")
        assert torch.equal(vp[phys, :, slot], v[rows])
    assert (q_out[r.N - 2:] == 7.0).all()


def test_append_refuses_positions_that_do_not_fit():
    r = Ragged([4], [70], page=64, Hkv=2, D=64, seed=615)
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    k, inv = randn(4, 2, 64, seed=616).cuda(), _inv(64).cuda()
    pos = torch.arange(4, device="cuda")
    for bad in (dict(positions=pos, inv_freq=None), dict(positions=pos[:3]), dict(positions=pos.int()),
                dict(positions=pos.cpu()), dict(positions=pos[None])):
        with pytest.raises(AssertionError, match="positions"):
            ops.paged_append(k, k, kp, vp, table, cu, lens, **{"inv_freq": inv, **bad})


def test_appends_from_many_refusals_go_on_where_they_were():
    _say("refused appends")
    st = PagedKVStore(2, 2, 64, 400, page=16, shuffle_seed=2, bounds=True)
    k = randn(60, 2, 64, seed=620).cuda()
    st.append(k[:21], k[:21], [20, 1])
    before = _state(st)
    for bad in (dict(k_new=k.float(), v_new=k), dict(k_new=k[:, :1], v_new=k), dict(k_new=k, v_new=k[:50]),
                dict(k_new=k, v_new=k, k_weight=torch.ones(32, dtype=BF, device="cuda")),
                dict(k_new=k, v_new=k, q_weight=torch.ones(64, dtype=BF, device="cuda"))):
        with pytest.raises(AssertionError):
            st.append(counts=[59, 1], **bad)
        assert _state(st) == before
    st.append(k[21:], k[21:], [9, 30])
    r = _view(st)
    assert torch.equal(r.cached(r.k_pages, 0, 29), torch.cat([k[:20], k[21:30]]).cpu().double().transpose(0, 1))
    assert torch.equal(r.cached(r.k_pages, 1, 31), torch.cat([k[20:21], k[30:]]).cpu().double().transpose(0, 1))


def test_appends_do_not_wait_for_the_stream():
    """Uniform and ragged counts, with new pages and without, and a write that keeps bounds."""
    _say("no waits")
    st = PagedKVStore(2, 2, 64, 900, page=16, bounds=True)
    k = randn(80, 2, 64, seed=630).cuda()
    w = randn(2, 2, 3, 64, seed=631).cuda()
    want, steps = [0, 0], ([40, 40], [1, 1], [0, 33], [5, 0], [1, 1], [0, 0])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        chunks = [st.append(k[:sum(c)], k[:sum(c)], c) for c in steps]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    for c, chunk in zip(steps, chunks):
        want = [a + b for a, b in zip(want, c)]
        assert chunk.cu_seqlens.tolist() == [0, c[0], sum(c)] and chunk.cu_seqlens.dtype == torch.int32
    assert st.lens == want == st.kv_lens.tolist()
    st.reset()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(7):
            st.write(w, w)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert st.lens == [21, 21] == st.kv_lens.tolist()
    r = _view(st)
    pages = r.table[:, :2].flatten().long()
    assert torch.equal(st.k_bounds.cpu()[pages], bounds_of(r)[pages])
    assert torch.equal(st.gather()[0], w.repeat(1, 1, 7, 1))


def test_an_append_under_capture_is_refused(monkeypatch):
    """Host lengths would not advance on a replay."""
    st = PagedKVStore(1, 1, 64, 64, page=16)
    k = randn(3, 1, 64, seed=635).cuda()
    before = _state(st)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        st.append(k, k, [3])
    assert _state(st) == before


def _model(pattern="block_topk", block_size=32):
    cfg = qwen3_config(pattern=pattern, block_size=block_size, vocab_size=512, hidden_size=256, intermediate_size=256,
                       num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    return build_model(cfg, seed=8)


@torch.no_grad()
@pytest.mark.parametrize("per_row", [False, True])
def test_qwen3_block_topk_rotates_at_the_positions_it_is_given(per_row):
    """A prompt, a chunk and a token whose position_ids are not the cache's own: one row for the batch, or a row each."""
    _say("qwen3 positions", per_row)
    model = _model()
    cache = PagedKVCache(2, 400, page=32, shuffle_seed=4, bounds=True)
    seen = []
    for layer in model.model.layers:
        layer.self_attn.register_forward_pre_hook(lambda m, a, kw: seen.append((m, kw["hidden_states"])), with_kwargs=True)
    at = 0
    for t in (150, 40, 1):
        ids = torch.randint(0, 512, (2, t), generator=torch.Generator().manual_seed(t)).cuda()
        pos = (torch.arange(at, at + t) + 1000)[None]
        if per_row:
            pos = torch.cat([pos, pos + 777])
        model(input_ids=ids, position_ids=pos.cuda(), past_key_values=cache, use_cache=True, logits_to_keep=1)
        at += t
        for attn, x in seen:
            r = _view(cache.layers[attn.layer_idx].store)
            keys = torch.cat([r.cached(r.k_pages, b, at)[:, at - t:].transpose(0, 1) for b in range(2)]).to(BF)
            proj = attn.k_proj(x).view(2 * t, -1, 128).cpu()
            assert_rotated(keys, *rotate(proj, attn.k_norm.weight.cpu(), pos.expand(2, t).reshape(-1), attn._inv_freq.cpu(),
                                         model.config.rms_norm_eps), "k")
        seen.clear()


@torch.no_grad()
def test_qwen3_block_topk_called_with_cos_and_sin_alone():
    """The attention module called by itself, without position_ids: it rotates with the cos and sin it is given."""
    _say("qwen3 cos sin")
    model = _model()
    attn = model.model.layers[1].self_attn
    cache = PagedKVCache(2, 200, page=32, bounds=True)
    x = randn(2, 70, 256, seed=640).cuda()
    cos, sin = model.model.rotary_emb(x, (torch.arange(70, device="cuda") * 3 + 11)[None])
    out, _ = attn(x, (cos, sin), None, past_key_values=cache)
    q = attn.q_norm(attn.q_proj(x).view(2, 70, -1, 128)).transpose(1, 2)
    k = attn.k_norm(attn.k_proj(x).view(2, 70, -1, 128)).transpose(1, 2)
    q, k = apply_rotary_pos_emb(q, k, cos, sin)
    store = cache.layers[1].store
    assert torch.equal(store.gather()[0], k)
    assert torch.equal(store.gather()[1], attn.v_proj(x).view(2, 70, -1, 128).transpose(1, 2))
    chunk = PagedChunk(torch.tensor([0, 70, 140], dtype=torch.int32, device="cuda"), (70, 70), None)
    want = HipBlockSparseBackend().forward_packed(q.transpose(1, 2).reshape(140, 4, 128), store, chunk,
                                                  attn.sparse_pattern.build(q, k))
    assert torch.equal(out, attn.o_proj(want.reshape(2, 70, -1)))


@torch.no_grad()
def test_qwen3_block_topk_refuses_a_page_that_is_not_its_block_before_it_appends():
    _say("qwen3 page")
    model = _model()
    cache = PagedKVCache(2, 400, page=64, bounds=True)
    with pytest.raises(ValueError, match="page"):
        model(input_ids=torch.zeros(1, 40, dtype=torch.long, device="cuda"), past_key_values=cache, use_cache=True)
    assert cache.get_seq_length() == 0


@torch.no_grad()
@pytest.mark.parametrize("fused", [True, False])
def test_a_captured_decode_leaves_key_bounds_of_what_it_wrote(fused):
    """Its steps write keys without the append kernel; ``finish`` brings the pages' bounds up to date."""
    _say("bounds after GraphDecoder", fused)
    model = _model("dense", 64)
    cache = PagedKVCache(2, 200, page=64, shuffle_seed=5, bounds=True)
    ids = torch.randint(0, 512, (2, 90), generator=torch.Generator().manual_seed(9)).cuda()
    out = model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1)
    dec = GraphDecoder(model, cache, out.logits[:, -1].argmax(-1), 140, fused=fused)
    for _ in range(12):
        dec.step()
    dec.finish()
    for layer in cache.layers:
        r = _view(layer.store)
        assert r.lens == [102, 102]
        pages = r.table[:, :2].flatten().long()
        assert torch.equal(layer.store.k_bounds.cpu()[pages], bounds_of(r)[pages])


@torch.no_grad()
@pytest.mark.parametrize("pattern,page,text", [("block_topk", 32, "block_topk"), ("dense", 32, "page 32")])
def test_a_refused_graph_decoder_takes_no_pages(pattern, page, text):
    _say("refused GraphDecoder", pattern)
    model = _model(pattern)
    cache = PagedKVCache(2, 200, page=page, bounds=True)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(10)).cuda()
    model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1)
    before = [_state(layer.store) for layer in cache.layers]
    with pytest.raises(ValueError, match=text):
        GraphDecoder(model, cache, ids[:, -1], 180)
    assert [_state(layer.store) for layer in cache.layers] == before
