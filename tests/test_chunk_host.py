"""Refusals and bookkeeping of the chunk operators that need no GPU: the C entry points' argument checks (every call
returns before any device access), the ragged paged store, the block_topk pattern and its caller."""
import pytest
import torch

from sparseattentioninfer_amd import _lib
from sparseattentioninfer_amd.attention import get_backend
from sparseattentioninfer_amd.models import PagedKVStore
from sparseattentioninfer_amd.patterns import BlockTopKPattern
from sparseattentioninfer_amd.qwen3 import PagedKVCache
from sparseattentioninfer_amd.qwen3.runtime import build_model, qwen3_config

FAKE = 1 << 12      # a 16-byte aligned stand-in address
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        from sparseattentioninfer_amd import _build
        _build.build(verbose=False)
    return _lib.load()


def _norm_rope(lib, **o):
    a = dict(dtype=0, q=FAKE, sb=0, st=1024, sh=128, k=FAKE, qo=FAKE, ko=FAKE, qw=None, kw=None, inv=FAKE, pos=FAKE,
             B=1, T=4, Hq=8, Hkv=2, D=128)
    a.update(o)
    s = (a["sb"], a["st"], a["sh"])
    return lib.sa_qk_norm_rope(a["dtype"], a["q"], *s, a["k"], *s, a["qo"], *s, a["ko"], *s, a["qw"], a["kw"], a["inv"],
                               a["pos"], 0, a["B"], a["T"], a["Hq"], a["Hkv"], a["D"], 1e-6, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), -1, b"dtype 7"), (dict(D=96), -3, b"head dim 96"), (dict(B=-1), -2, b"B=-1"),
    (dict(T=1 << 30, B=2), -2, b"too many"), (dict(q=None), -6, b"NULL"), (dict(inv=None), -6, b"NULL"),
    (dict(pos=None), -6, b"NULL"), (dict(q=FAKE + 2), -8, b"aligned"), (dict(st=1020), -8, b"aligned"),
    (dict(kw=FAKE + 8), -8, b"aligned")])
def test_norm_rope_refusals(lib, change, code, text):
    assert _norm_rope(lib, **change) == code and text in lib.sa_last_error()


def test_norm_rope_nothing_to_do(lib):
    assert _norm_rope(lib, T=0, q=None) == 0 and _norm_rope(lib, B=0) == 0
    assert _norm_rope(lib, Hq=0, Hkv=0, q=None, k=None) == 0


def _append(lib, **o):
    a = dict(dtype=0, q=None, k=FAKE, v=FAKE, qo=None, st=1024, sh=128, inv=None, kp=FAKE, vp=FAKE, pst=128, pages=8,
             bd=None, table=FAKE, ts=4, mb=4, cu=FAKE, lens=FAKE, N=4, B=2, Hq=0, Hkv=2, D=128, page=64)
    a.update(o)
    s = (a["st"], a["sh"])
    return lib.sa_paged_append(a["dtype"], a["q"], *s, a["k"], *s, a["v"], *s, a["qo"], *s, None, None, a["inv"], a["kp"],
                               a["vp"], 16384, 8192, a["pst"], a["pages"], a["bd"], 512, 256, a["table"], a["ts"], a["mb"],
                               a["cu"], a["lens"], a["N"], a["B"], a["Hq"], a["Hkv"], a["D"], a["page"], 1e-6, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), -1, b"dtype"), (dict(D=80), -3, b"head dim 80"), (dict(page=24), -4, b"page 24"),
    (dict(page=144), -4, b"page 144"), (dict(page=0), -4, b"page 0"), (dict(ts=3), -2, b"4 columns"),
    (dict(N=-1), -2, b"N=-1"), (dict(Hkv=0), -2, b"Hkv=0"), (dict(N=(1 << 31) - 1, B=1 << 30), -2, b"too many"),
    (dict(k=None), -6, b"NULL"), (dict(cu=None), -6, b"NULL"), (dict(table=None), -6, b"NULL"),
    (dict(Hq=4), -6, b"NULL"), (dict(vp=FAKE + 4), -8, b"aligned"), (dict(bd=FAKE + 1), -8, b"aligned"),
    (dict(pst=100), -8, b"aligned")])
def test_append_refusals(lib, change, code, text):
    assert _append(lib, **change) == code and text in lib.sa_last_error()


def test_append_nothing_to_do(lib):
    assert _append(lib, N=0, k=None) == 0 and _append(lib, B=0) == 0


def _chunk(lib, **o):
    a = dict(dtype=0, q=FAKE, o=FAKE, st=1024, sh=128, kp=FAKE, pst=128, pages=8, table=FAKE, ts=4, mb=4, cu=FAKE, lens=FAKE,
             sel=None, rows=0, width=0, off=None, N=4, B=2, Hq=8, Hkv=2, D=128, page=64, scale=0.1, splits=1, ws=None, wsb=0)
    a.update(o)
    return lib.sa_paged_chunk_attn(a["dtype"], a["q"], a["st"], a["sh"], a["kp"], FAKE, 16384, 8192, a["pst"], a["pages"],
                                   a["table"], a["ts"], a["mb"], a["cu"], a["lens"], a["sel"], 8, 4, a["rows"], a["width"],
                                   a["off"], 8, 4, a["o"], a["st"], a["sh"], a["N"], a["B"], a["Hq"], a["Hkv"], a["D"],
                                   a["page"], a["scale"], a["splits"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), -1, b"dtype"), (dict(D=256), -3, b"head dim 256"), (dict(page=40), -4, b"page 40"),
    (dict(Hq=7), -2, b"Hq=7"), (dict(splits=65), -2, b"65 splits"), (dict(splits=-1), -2, b"-1 splits"),
    (dict(scale=0.0), -2, b"scale"), (dict(scale=1e-40), -2, b"scale"), (dict(scale=-1.0), -2, b"scale"), (dict(scale=float("nan")), -2, b"scale"), (dict(N=1 << 30), -2, b"too many"),
    (dict(sel=FAKE), -2, b"selection"), (dict(sel=FAKE, off=FAKE, rows=1, width=4), -2, b"selection"),
    (dict(q=None), -6, b"NULL"), (dict(lens=None), -6, b"NULL"), (dict(o=FAKE + 2), -8, b"aligned"),
    (dict(st=1026), -8, b"aligned"), (dict(pst=1 << 25), -2, b"token stride"), (dict(pst=-128), -2, b"token stride"),
    (dict(splits=4), -7, b"workspace"), (dict(splits=4, ws=FAKE, wsb=64), -7, b"workspace"),
    (dict(N=1 << 25, splits=16, ws=FAKE, wsb=BIG), -2, b"partial rows")])
def test_chunk_refusals(lib, change, code, text):
    assert _chunk(lib, **change) == code and text in lib.sa_last_error()


def test_chunk_workspace_sizes(lib):
    size = lib.sa_paged_chunk_workspace_bytes
    assert size(4, 2, 8, 2, 128, 256, 1) == 0                    # one workgroup leaves no partials
    assert size(4, 2, 8, 2, 128, 256, 3) == 256 + 3 * 4 * 8 * 130 * 4
    assert size(4, 2, 8, 2, 128, 100, 3) == 256 + 2 * 4 * 8 * 130 * 4    # at most one for 64 keys
    assert size(4, 2, 8, 2, 128, 1 << 16, 0) > 0
    assert size(4, 2, 8, 2, 128, 256, 0) == 0                    # too few keys to divide
    assert size(4, 2, 8, 2, 128, 1024, 0) == 0 and size(40, 2, 8, 2, 128, 512, 0) == 0
    assert size(0, 2, 8, 2, 128, 1 << 16, 0) == 0 and size(4, 2, 8, 2, 128, 0, 4) == 0


def test_select_workspace_sizes(lib):
    size = lib.sa_paged_block_select_workspace_bytes
    assert size(8, 8, 257) == 64 * 257 * 8 and size(1, 1, 4096) == 4096 * 8     # few lists of many pages
    assert size(8, 8, 256) == 0 and size(9, 8, 257) == 0 and size(9, 8, 4096) == 0
    assert size(9, 8, 4097) == 72 * 4097 * 8
    assert size(0, 8, 5000) == 0 and size(8, 8, 0) == 0


def _select(lib, **o):
    a = dict(dtype=0, q=FAKE, st=1024, sh=128, bd=FAKE, pages=8, table=FAKE, ts=4, mb=4, cu=None, lens=FAKE, N=2, B=2, Hq=8,
             Hkv=2, D=128, page=64, topk=2, sink=1, recent=1, sel=FAKE, rows=2, width=4, off=FAKE, ws=None, wsb=0)
    a.update(o)
    return lib.sa_paged_block_select(a["dtype"], a["q"], a["st"], a["sh"], a["bd"], 512, 256, a["pages"], a["table"], a["ts"],
                                     a["mb"], a["cu"], a["lens"], a["N"], a["B"], a["Hq"], a["Hkv"], a["D"], a["page"],
                                     a["topk"], a["sink"], a["recent"], a["sel"], 8, 4, a["rows"], a["width"], a["off"],
                                     a["ws"], a["wsb"], None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=5), -1, b"dtype"), (dict(D=32), -3, b"head dim 32"), (dict(page=20), -4, b"page 20"),
    (dict(topk=-1), -2, b"top_k=-1"), (dict(recent=0), -2, b"recent=0"), (dict(sink=-2), -2, b"sink=-2"),
    (dict(N=3), -2, b"one token per sequence"), (dict(rows=3), -2, b"lists [3"), (dict(width=3), -2, b"needed [2"),
    (dict(cu=FAKE, N=70, rows=2, width=9), -2, b"needed [3"), (dict(ts=2), -2, b"columns"),
    (dict(mb=(1 << 21) + 1, ts=1 << 22), -2, b"columns"), (dict(N=1 << 22, B=1 << 22, rows=1 << 22), -2, b"too many"), (dict(bd=None), -6, b"NULL"), (dict(off=None), -6, b"NULL"),
    (dict(q=FAKE + 4), -8, b"aligned"), (dict(mb=5000, ts=5000), -7, b"workspace")])
def test_select_refusals(lib, change, code, text):
    assert _select(lib, **change) == code and text in lib.sa_last_error()


def test_store_appends_need_counts_that_fit_and_a_gpu_for_bounds():
    with pytest.raises(ValueError, match="GPU"):
        PagedKVStore(2, 1, 64, 100, page=16, device="cpu", bounds=True)
    st = PagedKVStore(2, 1, 64, 100, page=16, device="cpu", num_pages=6)
    k = torch.zeros(5, 1, 64, dtype=torch.bfloat16)
    for counts in ([5], [2, 2], [6, -1], [1, 1, 3]):
        with pytest.raises(ValueError, match="counts"):
            st.append(k, k, counts)
    st._grow_each([40, 3])
    assert [len(r) for r in st._table_host] == [3, 1]
    assert st.block_table[0, :3].tolist() == st._table_host[0] and st.block_table[1, 0].item() == st._table_host[1][0]
    st._grow_each([40, 20])
    assert [len(r) for r in st._table_host] == [3, 2] and len(set(sum(st._table_host, []))) == 5
    with pytest.raises(RuntimeError, match="out of pages"):
        st._grow_each([40, 60])
    with pytest.raises(ValueError, match="max_blocks"):
        st._grow_each([200, 1])
    assert [len(r) for r in st._table_host] == [3, 2]
    st.lens = [40, 20]
    for f in (st.seq_len, st.gather, lambda: st.write(torch.zeros(2, 1, 1, 64), torch.zeros(2, 1, 1, 64))):
        with pytest.raises(ValueError, match="one length"):
            f()


def test_block_topk_pattern_and_its_refusals():
    with pytest.raises(ValueError):
        BlockTopKPattern(-1)
    with pytest.raises(ValueError):
        BlockTopKPattern(4, recent=0)
    q, k = torch.zeros(1, 4, 3, 64), torch.zeros(1, 2, 6400, 64)
    p = BlockTopKPattern(16, sink=1, recent=3).build(q, k)
    assert p.kind == "block_topk" and p.topk == 16 and p.keep_ratio == 0.2 and (p.sink, p.recent) == (1, 3)
    be = get_backend("hip_block_sparse")
    with pytest.raises(RuntimeError, match="CPU"):
        be.forward(q, k, k, p)
    with pytest.raises(RuntimeError, match="GPU"):
        be.forward_packed(q[0], None, None, p)


def test_qwen3_block_topk_needs_a_cache_with_bounds():
    small = dict(vocab_size=128, hidden_size=128, intermediate_size=128, num_hidden_layers=1, num_attention_heads=2,
                 num_key_value_heads=1, head_dim=64)
    model = build_model(qwen3_config(pattern="block_topk", **small), device="cpu", dtype=torch.float32)
    ids = torch.zeros(1, 4, dtype=torch.long)
    for cache in (None, PagedKVCache(1, 64)):
        with pytest.raises(ValueError, match="bounds=True"):
            model(input_ids=ids, past_key_values=cache, use_cache=cache is not None)
    scaled = qwen3_config(pattern="block_topk", **small)
    scaled.rope_parameters = {"rope_type": "linear", "rope_theta": 1e6, "factor": 2.0}
    with pytest.raises(NotImplementedError, match="linear"):
        build_model(scaled, device="cpu", dtype=torch.float32)
