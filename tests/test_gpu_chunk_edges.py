"""The chunk operators at the edges of their definitions: selections without entries, tables and pools without any,
values that are not finite."""
import math

import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import Ragged, attention, bounds_of, randn, select

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[chunk-edges]", *msg, flush=True)


def _attend(r, q, **kw):
    out = torch.full_like(q, 9.0).cuda()
    ops.paged_chunk_attn(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens"), out=out, **kw)
    return out.cpu()


@pytest.mark.parametrize("splits", [1, 0, 3])
def test_a_selection_of_width_zero_selects_nothing(splits):
    """Narrow and wide sequences: their rows are 0, rows of no sequence stay."""
    _say("width 0", splits)
    r = Ragged([2, 100, 0], [300, 2000, 70], page=64, Hkv=2, D=128, seed=400, pad_rows=3)
    q = randn(r.N, 8, 128, seed=401)
    rows = r.N // 64 + 3
    sel = torch.zeros(rows, 2, 0, dtype=torch.int32, device="cuda")
    got = _attend(r, q, sel=sel, sel_off=torch.zeros(rows, 2, 2, dtype=torch.int32, device="cuda"), num_splits=splits)
    assert not got[:102].any() and (got[102:] == 9.0).all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("q_lens,kv_lens,D,dtype", [([3], [900], 128, BF), ([90], [900], 128, BF), ([3], [500], 64, HF),
                                                    ([70, 2], [400, 700], 64, BF)])
def test_nan_rows_stay_nan_however_the_keys_are_divided(q_lens, kv_lens, D, dtype, splits):
    """A query of NaN, and one key of NaN: the rows that see them are NaN, the others as without them."""
    _say("nan rows", q_lens, kv_lens, D, dtype, splits)
    r = Ragged(q_lens, kv_lens, page=64, Hkv=2, D=D, dtype=dtype, seed=410)
    q = randn(r.N, 8, D, seed=411, dtype=dtype)
    want, tol, _ = attention(r, q)
    q[1, 2] = math.nan
    got = _attend(r, q, num_splits=splits)
    assert got[1, 2].isnan().all()
    bad = ~((got.double() - want).abs() <= tol)
    bad[1, 2] = False
    assert not bad.any()
    # key of the first sequence's second new token (position n - t + 1) in KV head 1: rows from that token on see it
    q = randn(r.N, 8, D, seed=411, dtype=dtype)
    t, n = q_lens[0], kv_lens[0]
    p = n - t + 1
    r.k_pages[r.table[0, p // 64].long(), 1, p % 64] = math.nan
    got = _attend(r, q, num_splits=splits)
    assert got[1:t, 4:].isnan().all()
    bad = ~((got.double() - want).abs() <= tol)
    bad[1:t, 4:] = False
    assert not bad.any()
    # a whole share of the keys
    r.k_pages[r.table[0, 0].long(), 0] = math.nan
    assert _attend(r, q, num_splits=splits)[:t, :4].isnan().all()


@pytest.mark.parametrize("tokens", [True, False])
def test_select_ranks_infinite_bounds_by_the_definition(tokens):
    """Largest products of +inf rank first (ties to the lower page); an infinite bound on the side that a query's sign
    does not take changes nothing."""
    _say("infinite bounds", tokens)
    r = Ragged([1, 1], [64 * 20, 64 * 14 + 3], page=64, Hkv=2, D=64, seed=420, poison=False)
    bounds = bounds_of(r)
    q = randn(2, 2, 64, seed=421)           # one head a group: one sign for each dim
    for b in range(2):
        for g in range(2):
            up, down = (q[b, g] > 0).nonzero().flatten(), (q[b, g] < 0).nonzero().flatten()
            pg = r.table[b].long()
            bounds[pg[9], g, 1, up[3]] = math.inf
            bounds[pg[5], g, 0, down[2]] = -math.inf
            bounds[pg[7], g, 1, down[1]] = math.inf         # not the side that counts
            bounds[pg[8], g, 0, up[1]] = -math.inf
    for top_k in (1, 2, 4):
        args = dict(top_k=top_k, sink=1, recent=1)
        want = select(r, q, bounds, tokens=tokens, **args)
        got = ops.paged_block_select(q.cuda(), bounds.cuda(), *r.gpu("table", "kv_lens"), page=64,
                                     cu_seqlens=None if tokens else r.cu.cuda(), **args)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
        kept = got[0][..., :top_k + 2].cpu()
        assert (kept == 5).any(-1).all() and (top_k == 1 or (kept == 9).any(-1).all())


def test_select_infinite_bounds_and_a_zero_query():
    """0 times an infinite bound counts as 0: the page is ranked by its other dims."""
    _say("infinite bounds, zero query")
    r = Ragged([1], [64 * 10], page=64, Hkv=1, D=64, seed=425, poison=False)
    q = randn(1, 2, 64, seed=426)
    q[:, :, 7] = 0
    bounds = bounds_of(r)
    bounds[..., 7] = 0
    args = dict(top_k=4, sink=0, recent=1)
    want = select(r, q, bounds, tokens=True, **args)
    bounds[r.table[0, 2].long(), 0, 1, 7] = math.inf
    bounds[r.table[0, 4].long(), 0, 0, 7] = -math.inf
    got = ops.paged_block_select(q.cuda(), bounds.cuda(), *r.gpu("table", "kv_lens"), page=64, **args)
    assert torch.equal(got[0].cpu(), want[0])


def test_select_nan_queries_leave_the_lowest_pages():
    """Every score of a list with a NaN query is NaN: all rank last, so the lowest pages are kept.  Other lists, the same
    block's of another KV head among them, are as without it."""
    _say("nan queries")
    r = Ragged([1, 130], [64 * 20, 64 * 12], page=64, Hkv=2, D=128, seed=430, poison=False)
    bounds = bounds_of(r)
    args = dict(top_k=3, sink=1, recent=1)
    q = randn(131, 4, 128, seed=431)
    clean = select(r, q, bounds, tokens=False, **args)[0]
    q[0, 3, 5] = math.nan           # list 0, KV head 1
    q[1 + 64 + 9, 0, 77] = math.nan     # second block of the second sequence, KV head 0
    got = ops.paged_block_select(q.cuda(), bounds.cuda(), *r.gpu("table", "kv_lens"), page=64, cu_seqlens=r.cu.cuda(),
                                 **args)[0].cpu()
    assert got[0, 1].tolist()[:5] == [0, 1, 2, 3, 19]
    assert got[2, 0].tolist()[:4] == [0, 1, 2, 3]
    same = torch.ones(got.shape[:2], dtype=torch.bool)
    same[0, 1] = same[2, 0] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("what", ["table", "pool"])
def test_tables_without_columns_and_pools_without_pages(what):
    """Nothing can be read or written: outputs are 0, lists hold no page that is not there, the pools stay."""
    _say("empty", what)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cols, pages = (0, 3) if what == "table" else (2, 0)
    table = torch.zeros(2, cols, dtype=torch.int32, device="cuda")
    kp, vp = (torch.full((pages, 2, 64, 64), 5.0, dtype=BF, device="cuda") for _ in range(2))
    bd = torch.full((pages, 2, 2, 64), 5.0, dtype=BF, device="cuda")
    cu, lens = i32(0, 70, 71), i32(100, 30)
    q, k = randn(71, 4, 64, seed=440).cuda(), randn(71, 2, 64, seed=441).cuda()
    qo = ops.paged_append(k, k, kp, vp, table, cu, lens, q=q, k_bounds=bd)
    assert torch.equal(qo, q) and (kp == 5.0).all() and (vp == 5.0).all() and (bd == 5.0).all()
    assert not ops.paged_chunk_attn(q, kp, vp, table, cu, lens).any()
    sel, off = ops.paged_block_select(q, bd, table, lens, page=64, top_k=1, cu_seqlens=cu)
    assert sel.max() < max(cols, 1) and off.max() <= cols
    assert not ops.paged_chunk_attn(q, kp, vp, table, cu, lens, sel=sel, sel_off=off).any()
    sel, off = ops.paged_block_select(q[:2], bd, table, lens, page=64, top_k=1)
    assert sel.max() < max(cols, 1) and off.max() <= cols
