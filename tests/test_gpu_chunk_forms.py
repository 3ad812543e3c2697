"""Forms of the chunk operators' calls that their documentation allows beside the usual ones: groups larger than a narrow
item, a scale that is given, lengths past the table, rows before the first sequence, more new tokens than tokens, tensors
written over themselves, pools whose offsets pass 32 bits, positions of stride 0, no query or no key heads."""
import math

import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import Ragged, assert_rotated, attention, bounds_of, half_step, randn, rotate, select

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[chunk-forms]", *msg, flush=True)


def _inv(D):
    return (1.0 / 1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()


def _check(got, want, tol, live, what):
    err = (got.cpu().double() - want).abs()
    bad = ~(err <= tol) & live[:, None, None]
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {(err / tol)[live].max():.2f} of it"


@pytest.mark.parametrize("splits", [1, 0, 3])
@pytest.mark.parametrize("Hq,Hkv,D", [(71, 1, 64), (128, 1, 128), (96, 1, 64), (260, 2, 64)])
def test_groups_larger_than_a_narrow_item(Hq, Hkv, D, splits):
    """One token of more than 64 heads a group is a wide item; dense and over lists."""
    _say("groups", Hq, Hkv, D, splits)
    r = Ragged([1, 3, 0, 1], [1500, 200, 9, 64], page=64, Hkv=Hkv, D=D, seed=700, pad_rows=1)
    q = randn(r.N, Hq, D, seed=701)
    args = (q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens"))
    _check(ops.paged_chunk_attn(*args, num_splits=splits), *attention(r, q), "dense")
    sel, off = select(r, q, bounds_of(r), top_k=3, sink=1, recent=1, tokens=False)
    got = ops.paged_block_select(args[0], bounds_of(r).cuda(), args[3], args[5], page=64, top_k=3, cu_seqlens=args[4])
    assert torch.equal(got[0].cpu(), sel) and torch.equal(got[1].cpu(), off)
    _check(ops.paged_chunk_attn(*args, sel=got[0], sel_off=got[1], num_splits=splits), *attention(r, q, sel, off), "lists")


@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("q_lens,kv_lens", [([2], [700]), ([40], [700])])
def test_a_scale_that_is_given(q_lens, kv_lens, scale):
    """The default scale of queries that carry the rest of it; 2^k factors, so that the queries stay exact."""
    _say("scale", q_lens, scale)
    r = Ragged(q_lens, kv_lens, page=64, Hkv=2, D=64, seed=710)
    q = randn(r.N, 8, 64, seed=711)
    want, tol, live = attention(r, q)
    args = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    for k in (-2, 3):
        _check(ops.paged_chunk_attn((q * 2.0 ** -k).cuda(), *args, sm_scale=2.0 ** k / 8), want, tol, live, f"2^{k}")
    # another scale is the default one of queries in float64
    x = q.double() * scale * 8
    r2 = attention(r, x.to(torch.float64))[0]
    mag = torch.zeros_like(r2) + r.v_pages.nan_to_num().abs().max()
    h = half_step(BF)
    tol = 2 * h * mag + (64 * 64 * 2.0 ** -24 * max(1.0, scale * 8)) * mag
    _check(ops.paged_chunk_attn(q.cuda(), *args, sm_scale=scale), r2, tol, live, f"scale {scale}")


@pytest.mark.parametrize("t", [3, 40])
def test_lengths_past_the_table_end_with_it(t):
    """Rows whose positions lie past the last column see the keys of the columns that are there."""
    _say("past the table", t)
    r = Ragged([t, 1], [700, 30], page=64, Hkv=2, D=64, seed=720)
    q = randn(r.N, 8, 64, seed=721)
    all_pages = torch.arange(4, dtype=torch.int32).expand(r.N // 64 + 2, 2, 4).clone()
    off = torch.tensor([0, 4], dtype=torch.int32).expand(r.N // 64 + 2, 2, 2).clone()
    off[-1] = 0
    off[1, :, 1] = 1                # the second sequence has one page
    want, tol, live = attention(r, q, all_pages, off)
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    short = table[:, :4]            # the rows keep the stride of the whole table
    for splits in (1, 0, 3):
        _check(ops.paged_chunk_attn(q.cuda(), kp, vp, short, cu, lens, num_splits=splits), want, tol, live, f"{splits}")
    # single tokens: all four columns are ranked, the page of the token itself is not there
    bounds = bounds_of(r)
    x = randn(2, 8, 64, seed=722)
    got = ops.paged_block_select(x.cuda(), bounds.cuda(), short, lens, page=64, top_k=4, sink=1, recent=1)
    assert got[0][0, 0].tolist()[:4] == [0, 1, 2, 3] and got[1][0, 0].tolist() == [0, 4]


def test_rows_before_the_first_sequence_are_left():
    _say("rows before")
    r = Ragged([0, 70, 2], [40, 300, 9], page=32, Hkv=2, D=64, seed=730, pad_rows=4, poison=False)
    first = 5
    q, k, v = (randn(first + r.N, h, 64, seed=731 + h) for h in (4, 2, 2))
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    cu = cu + first
    q_out = torch.full_like(q, 7.0).cuda()
    ops.paged_append(k.cuda(), v.cuda(), kp, vp, table, cu, lens, q=q.cuda(), q_out=q_out)
    live = torch.zeros(q.size(0), dtype=torch.bool)
    live[first:first + 72] = True
    assert torch.equal(q_out.cpu()[live], q[live]) and (q_out.cpu()[~live] == 7.0).all()
    r.k_pages, r.v_pages = kp.cpu(), vp.cpu()
    assert torch.equal(r.cached(r.k_pages, 1, 300)[:, 230:], k[first:first + 70].double().transpose(0, 1))
    out = torch.full_like(q, 9.0).cuda()
    ops.paged_chunk_attn(q.cuda(), kp, vp, table, cu, lens, out=out)
    want, tol, _ = attention(r, q[first:])
    _check(out[first:], want, tol, live[first:], "rows before")
    assert (out.cpu()[~live] == 9.0).all()
    sel, off = ops.paged_block_select(q.cuda(), bounds_of(r).cuda(), table, lens, page=32, top_k=2, cu_seqlens=cu)
    want = select(r, q[first:], bounds_of(r), top_k=2, sink=1, recent=1, tokens=False)
    n = want[0].size(0)
    assert torch.equal(sel.cpu()[:n], want[0]) and torch.equal(off.cpu()[:n], want[1]) and not off[n:].any()


def test_selection_with_more_new_tokens_than_tokens():
    """Blocks whose queries all lie before position 0 have empty lists; one that reaches 0 counts from there."""
    _say("more new tokens than tokens")
    r = Ragged([150, 70], [40, 64], page=16, Hkv=2, D=64, seed=740, poison=False)
    q = randn(r.N, 4, 64, seed=741)
    bounds = bounds_of(r)
    args = dict(top_k=1, sink=0, recent=1)
    want = select(r, q, bounds, tokens=False, **args)
    got = ops.paged_block_select(q.cuda(), bounds.cuda(), *r.gpu("table", "kv_lens"), page=16, cu_seqlens=r.cu.cuda(), **args)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]) and not got[1][0].any()
    out = ops.paged_chunk_attn(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens"), sel=got[0], sel_off=got[1])
    _check(out, *attention(r, q, *want), "attention")


def test_append_writes_queries_over_themselves():
    _say("in place")
    r = Ragged([100, 1, 33], [130, 64, 33], page=64, Hkv=2, D=128, seed=750, poison=False)
    row = randn(r.N, (8 + 2 + 2) * 128, seed=751)
    q, k, v = (x.unflatten(1, (-1, 128)) for x in row.cuda().split([8 * 128, 256, 256], dim=1))
    want = q.cpu().clone()
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    out = ops.paged_append(k, v, kp, vp, table, cu, lens, inv_freq=_inv(128).cuda(), q=q, q_out=q)
    assert out is q
    for b, at, t, n in r.rows():
        assert_rotated(q[at:at + t], *rotate(want[at:at + t], None, torch.arange(n - t, n), _inv(128), 1e-6), f"q of {b}")


def test_pools_whose_offsets_pass_32_bits():
    """Pages 2^30 elements apart (and their bounds), in pools of more than 2^32 elements: append, attend, select."""
    _say("far pages")
    r = Ragged([3, 20], [200, 20], page=64, Hkv=2, D=64, seed=760, poison=False)
    P, step = r.k_pages.size(0), 1 << 30
    far = []
    for pool in (r.k_pages, r.v_pages):
        size = (P - 1) * step + pool[0].numel()
        big = torch.empty(size, dtype=BF, device="cuda")
        view = big.as_strided(pool.shape, (step, *pool.stride()[1:]))
        view.copy_(pool.cuda())
        far.append(view)
    assert (P - 1) * step > 1 << 32
    bounds = bounds_of(r)
    fb = torch.empty((P - 1) * step + bounds[0].numel(), dtype=BF, device="cuda").as_strided(bounds.shape,
                                                                                           (step, *bounds.stride()[1:]))
    fb.copy_(bounds.cuda())
    q, k, v = (randn(r.N, h, 64, seed=761 + h) for h in (8, 2, 2))
    table, cu, lens = r.gpu("table", "cu", "kv_lens")
    ops.paged_append(k.cuda(), v.cuda(), *far, table, cu, lens, k_bounds=fb)
    r.k_pages, r.v_pages = (x.cpu() for x in far)
    at = 0
    for b, t, n in ((0, 3, 200), (1, 20, 20)):
        assert torch.equal(r.cached(r.k_pages, b, n)[:, n - t:], k[at:at + t].double().transpose(0, 1))
        assert torch.equal(r.cached(r.v_pages, b, n)[:, n - t:], v[at:at + t].double().transpose(0, 1))
        at += t
    for splits in (1, 3):
        _check(ops.paged_chunk_attn(q.cuda(), *far, table, cu, lens, num_splits=splits), *attention(r, q), "dense")
    pick = dict(top_k=1, sink=0, recent=1)
    sel, off = ops.paged_block_select(q.cuda(), fb, table, lens, page=64, cu_seqlens=cu, **pick)
    want = select(r, q, fb.cpu(), tokens=False, **pick)
    assert torch.equal(sel.cpu(), want[0])
    _check(ops.paged_chunk_attn(q.cuda(), *far, table, cu, lens, sel=sel, sel_off=off), *attention(r, q, *want), "lists")


def test_norm_rope_positions_shared_by_the_batch_and_missing_heads():
    _say("norm_rope forms")
    q, k = randn(3, 9, 4, 64, seed=770), randn(3, 9, 2, 64, seed=771)
    pos = torch.arange(9) * 11 + 4
    inv = _inv(64)
    dev_pos = pos.cuda().expand(3, 9)
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), dev_pos, inv.cuda())
    for x, y in ((q, got[0]), (k, got[1])):
        want, terms = rotate(x.flatten(0, 1), None, pos.repeat(3), inv, 1e-6)
        assert_rotated(y.flatten(0, 1), want, terms, "shared positions")
    none = torch.zeros(3, 9, 0, 64, dtype=BF, device="cuda")
    assert torch.equal(ops.qk_norm_rope(q.cuda(), none, dev_pos, inv.cuda())[0], got[0])
    assert torch.equal(ops.qk_norm_rope(none, k.cuda(), dev_pos, inv.cuda())[1], got[1])
