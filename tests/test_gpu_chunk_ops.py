"""Operators of a chunk of new tokens over a paged cache against their float64 definitions: head norms with
rotation, the paged append with key bounds, chunk attention over whole caches and over selected pages, and the
selection itself, at the lengths, pages, groups and strides where they can go wrong."""
import math

import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import Ragged, assert_rotated, attention, bounds_of, randn, rotate, select

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[chunk-ops]", *msg, flush=True)


def _inv(D, theta=1e6):
    return (1.0 / theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()


# ---- qk_norm_rope ------------------------------------------------------------------------------

@pytest.mark.parametrize("N,Hq,Hkv,D,dtype,norm", [
    (1, 32, 8, 128, BF, True), (7, 5, 5, 64, HF, False), (33, 14, 2, 64, BF, True), (100, 3, 1, 128, HF, True),
    (129, 8, 8, 128, BF, False), (1000, 40, 8, 128, BF, True)])
def test_qk_norm_rope(N, Hq, Hkv, D, dtype, norm):
    _say("qk_norm_rope", N, Hq, Hkv, D, dtype, norm)
    q, k = randn(N, Hq, D, seed=1, dtype=dtype, scale=3.0), randn(N, Hkv, D, seed=2, dtype=dtype, scale=0.2)
    qw, kw = (randn(D, seed=s, dtype=dtype, scale=0.3) + 1 if norm else None for s in (3, 4))
    pos = torch.randint(0, 131072, (N,), generator=torch.Generator().manual_seed(5))
    pos[0] = 131071
    inv = _inv(D)
    dev = lambda t: None if t is None else t.cuda()
    got = ops.qk_norm_rope(dev(q), dev(k), dev(pos), dev(inv), q_weight=dev(qw), k_weight=dev(kw), eps=EPS)
    for x, w, y, what in ((q, qw, got[0], "q"), (k, kw, got[1], "k")):
        assert_rotated(y, *rotate(x, w, pos, inv, EPS), what)


def test_qk_norm_rope_batched_strided_in_place():
    """[B, T, H, D] views of one projection row, written over themselves; then into [B, H, T, D] buffers."""
    _say("qk_norm_rope strided")
    B, T, Hq, Hkv, D = 3, 19, 6, 2, 128
    row = randn(B, T, (Hq + 2 * Hkv) * D, seed=6)
    pos = torch.arange(B * T).view(B, T) * 7
    inv = _inv(D)
    qw, kw = randn(D, seed=7) + 1, randn(D, seed=8) + 1
    split = lambda t: [x.unflatten(-1, (-1, D)) for x in t.split([Hq * D, Hkv * D, Hkv * D], dim=-1)]
    q, k, v = split(row)
    dev = row.cuda()
    dq, dk, dv = split(dev)
    qo, ko = (torch.full((B, h, T, D), math.nan, dtype=BF, device="cuda") for h in (Hq, Hkv))
    args = dict(q_weight=qw.cuda(), k_weight=kw.cuda(), eps=EPS)
    ops.qk_norm_rope(dq, dk, pos.cuda(), inv.cuda(), q_out=qo.transpose(1, 2), k_out=ko.transpose(1, 2), **args)
    ops.qk_norm_rope(dq, dk, pos.cuda(), inv.cuda(), q_out=dq, k_out=dk, **args)
    for x, w, over, out, what in ((q, qw, dq, qo, "q"), (k, kw, dk, ko, "k")):
        want, terms = rotate(x.reshape(B * T, -1, D), w, pos.view(-1), inv, EPS)
        assert_rotated(out.transpose(1, 2).reshape(B * T, -1, D), want, terms, what)
        assert torch.equal(over, out.transpose(1, 2))
    assert torch.equal(dv.cpu(), v)     # the values beside them are untouched


def test_qk_norm_rope_zero_rows_and_values():
    inv = _inv(128).cuda()
    q, k = torch.zeros(0, 4, 128, dtype=BF, device="cuda"), torch.zeros(0, 2, 128, dtype=BF, device="cuda")
    got = ops.qk_norm_rope(q, k, torch.zeros(0, dtype=torch.int64, device="cuda"), inv)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    z = torch.zeros(3, 4, 128, dtype=BF, device="cuda")
    w = torch.ones(128, dtype=BF, device="cuda")
    got = ops.qk_norm_rope(z, z, torch.arange(3, device="cuda"), inv, q_weight=w, k_weight=w)
    assert not got[0].any() and not got[1].any()


# ---- paged_append ------------------------------------------------------------------------------

def _append_case(q_lens, kv_lens, page, Hq, Hkv, D, dtype, norm, rope, bounds, pad=0, seed=10):
    r = Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=seed, pad_rows=pad, poison=False)
    row = randn(r.N, (Hq + 2 * Hkv) * D, seed=seed + 3, dtype=dtype, scale=2.0)
    q, k, v = (x.unflatten(1, (-1, D)) for x in row.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    qw, kw = (randn(D, seed=seed + s, dtype=dtype, scale=0.3) + 1 if norm else None for s in (4, 5))
    inv = _inv(D) if rope else None
    old = Ragged([0] * len(q_lens), [max(0, n - t) for t, n in zip(q_lens, kv_lens)], page=page, Hkv=Hkv, D=D,
                 dtype=dtype, seed=seed, poison=False)
    old.table, old.k_pages = r.table, r.k_pages
    bd = bounds_of(old) if bounds else None
    g = lambda t: None if t is None else t.cuda()
    kp, vp, gb, grow = g(r.k_pages), g(r.v_pages), g(bd), g(row)
    gq, gk, gv = (x.unflatten(1, (-1, D)) for x in grow.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    q_out = torch.full((r.N, Hq, D), 7.0, dtype=dtype, device="cuda")
    ops.paged_append(gk, gv, kp, vp, g(r.table), g(r.cu), g(r.kv_lens), inv_freq=g(inv), k_weight=g(kw), eps=EPS,
                     k_bounds=gb, q=gq, q_weight=g(qw), q_out=q_out)
    kp, vp, q_out = kp.cpu(), vp.cpu(), q_out.cpu()
    written = torch.zeros(kp.size(0), page, dtype=torch.bool)
    for b, at, t, n in r.rows():
        p = torch.arange(n - t, n)
        want, terms = rotate(q[at:at + t], qw, p, inv, EPS)
        assert_rotated(q_out[at:at + t], want, terms, f"q of sequence {b}")
        want, terms = rotate(k[at:at + t], kw, p, inv, EPS)
        ok = p >= 0
        phys, slot = r.table[b, p[ok] // page].long(), p[ok] % page
        assert_rotated(kp[phys, :, slot], want[ok], terms[ok], f"k of sequence {b}")
        assert torch.equal(vp[phys, :, slot], v[at:at + t][ok])
        written[phys, slot] = True
    used = sum(q_lens)
    assert (q_out[used:] == 7.0).all()          # rows of no sequence
    keep = ~written[:, None, :, None].expand_as(kp)
    assert torch.equal(kp[keep], r.k_pages[keep]) and torch.equal(vp[keep], r.v_pages[keep])
    if bounds:
        r.k_pages = kp
        want = bounds_of(r)
        touched = written.any(1)
        assert torch.equal(gb.cpu()[touched], want[touched])
        assert torch.equal(gb.cpu()[~touched], bd[~touched])


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_paged_append_ragged(page, D, dtype):
    _say("append", page, D, dtype)
    _append_case([130, 0, 1, 77, 16, 300], [130, 40, 90, 200, 16, 431], page, 6, 2, D, dtype, True, True, True, pad=5)


@pytest.mark.parametrize("B", [1, 64, 65, 130])
def test_paged_append_single_tokens(B):
    """One token each: fresh pages, filled ones, the last slot; more sequences than lanes of a wave."""
    _say("append tokens", B)
    lens = [(1, 64, 65, 1000, 128, 7)[b % 6] for b in range(B)]
    _append_case([1] * B, lens, 64, 4, 2, 128, BF, True, True, True)


@pytest.mark.parametrize("norm,rope,bounds", [(False, False, False), (False, True, True), (True, False, True)])
def test_paged_append_without_parts(norm, rope, bounds):
    _say("append parts", norm, rope, bounds)
    _append_case([65, 3], [65, 100], 64, 3, 3, 64, BF, norm, rope, bounds)


def test_paged_append_in_steps_keeps_bounds():
    """A page filled by several calls ends with the bounds of all its keys; without queries."""
    r = Ragged([0], [200], page=64, Hkv=2, D=128, seed=20, poison=False)
    k, v = randn(200, 2, 128, seed=21), randn(200, 2, 128, seed=22)
    kp, vp, table = r.gpu("k_pages", "v_pages", "table")
    bd = torch.full((kp.size(0), 2, 2, 128), math.nan, dtype=BF, device="cuda")
    at = 0
    for t in (3, 60, 1, 1, 100, 35):
        cu = torch.tensor([0, t], dtype=torch.int32, device="cuda")
        n = torch.tensor([at + t], dtype=torch.int32, device="cuda")
        assert ops.paged_append(k[at:at + t].cuda(), v[at:at + t].cuda(), kp, vp, table, cu, n, k_bounds=bd) is None
        at += t
    r.k_pages = kp.cpu()
    pages = r.table[0, :4].long()
    assert torch.equal(bd.cpu()[pages], bounds_of(r)[pages])
    assert torch.equal(r.cached(r.k_pages, 0, 200), k.double().transpose(0, 1))


def test_paged_append_bad_pages_and_positions_are_not_written():
    """Page ids outside the pool, positions past the table, more new tokens than tokens."""
    r = Ragged([40, 40, 10], [40, 40, 4], page=16, Hkv=2, D=64, seed=23, extra_cols=0, poison=False)
    table = r.table.clone()
    table[0, 1] = 10 ** 6
    table[1, 0] = -3
    k, v = randn(90, 2, 64, seed=24), randn(90, 2, 64, seed=25)
    kp, vp = r.gpu("k_pages", "v_pages")
    bd = torch.zeros(kp.size(0), 2, 2, 64, dtype=BF, device="cuda")
    lens = torch.tensor([40, 300, 4], dtype=torch.int32, device="cuda")     # positions 260.. lie past the table
    ops.paged_append(k.cuda(), v.cuda(), kp, vp, table.cuda(), r.cu.cuda(), lens, k_bounds=bd)
    want = r.k_pages.clone()
    for i in [x for x in range(40) if x // 16 != 1]:
        want[table[0, i // 16].long(), :, i % 16] = k[i]
    for i in range(4):                                                      # the last four of ten tokens
        want[table[2, 0].long(), :, i] = k[80 + 6 + i]
    assert torch.equal(kp.cpu(), want)


# ---- paged_chunk_attn --------------------------------------------------------------------------

def _attend(r, q, **kw):
    out = torch.full_like(q, 9.0).cuda()
    ops.paged_chunk_attn(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens"), out=out, **kw)
    return out.cpu()


def _check(got, want, tol, live, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & live[:, None, None]
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {(err / tol)[live].max():.2f} of it"
    assert (got[~live] == 9.0).all(), f"{what}: rows of no sequence were written"


SHAPES = [  # q_lens, kv_lens, page, Hq, Hkv, D, dtype
    ([1], [1], 64, 4, 1, 128, BF),
    ([1, 1, 1], [1, 64, 129], 64, 8, 2, 128, BF),
    ([5, 0, 33, 64], [5, 30, 33, 200], 16, 4, 4, 64, HF),
    ([17, 130], [300, 131], 32, 14, 2, 64, BF),
    ([3, 2], [1000, 65], 128, 6, 2, 128, HF),
    ([70, 1], [71, 500], 48, 3, 1, 128, BF),
    ([129, 4], [129, 260], 80, 8, 1, 128, BF),
    ([200], [520], 64, 32, 8, 128, BF),
    ([300, 150], [700, 150], 64, 4, 1, 64, BF),
    ([10, 6], [4, 6], 16, 4, 2, 128, BF),          # more new tokens than tokens: the first six see nothing
]


@pytest.mark.parametrize("splits", [1, 0, 3])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_chunk_attention(case, splits):
    q_lens, kv_lens, page, Hq, Hkv, D, dtype = SHAPES[case]
    _say("chunk", *SHAPES[case], "splits", splits)
    r = Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=30 + case, pad_rows=3)
    q = randn(r.N, Hq, D, seed=60 + case, dtype=dtype)
    want, tol, live = attention(r, q)
    _check(_attend(r, q, num_splits=splits), want, tol, live, f"case {case}")


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("case", range(1, len(SHAPES) - 1))
def test_chunk_attention_over_a_selection(case, splits):
    q_lens, kv_lens, page, Hq, Hkv, D, dtype = SHAPES[case]
    _say("chunk sel", *SHAPES[case], "splits", splits)
    r = Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=90 + case, pad_rows=70)
    q = randn(r.N, Hq, D, seed=120 + case, dtype=dtype)
    rows = r.N // 64 + len(q_lens)
    g = torch.Generator().manual_seed(case)
    cols = r.table.size(1)
    sel = torch.stack([torch.stack([torch.randperm(cols, generator=g) for _ in range(Hkv)]) for _ in range(rows)]).to(torch.int32)
    n = torch.randint(0, cols + 1, (rows, Hkv), generator=g)
    for i in range(rows):
        for h in range(Hkv):
            sel[i, h, :n[i, h]] = sel[i, h, :n[i, h]].sort().values
    off = torch.stack([torch.zeros_like(n), n], dim=2).to(torch.int32)
    off[0, 0, 0] = min(1, int(off[0, 0, 1]))       # a list that starts inside its row
    want, tol, live = attention(r, q, _clip(sel, off, r), off)
    _check(_attend(r, q, sel=sel.cuda(), sel_off=off.cuda(), num_splits=splits), want, tol, live, f"case {case}")


def _clip(sel, off, r):
    """For the plain form: entries past a sequence's pages select nothing; they are replaced by the list's first
    entry where that is a page, which is in the list anyway."""
    out = sel.clone()
    blk = 0
    for b, at, t, n in r.rows():
        pages = -(-n // r.page)
        for i in range(blk, blk + -(-t // 64)):
            for h in range(r.Hkv):
                lo, hi = off[i, h].tolist()
                ids = [x for x in sel[i, h, lo:hi].tolist() if x < pages]
                if ids:
                    out[i, h, lo:hi] = torch.tensor(ids + [ids[0]] * (hi - lo - len(ids)), dtype=torch.int32)
                else:
                    off[i, h] = torch.tensor([lo, lo], dtype=torch.int32)
        blk += -(-t // 64)
    return out


def test_chunk_attention_scores_that_grow():
    """Scores that rise by hundreds along the keys: the row reference must follow; and very negative ones."""
    for sign in (1.0, -1.0):
        r = Ragged([40], [900], page=64, Hkv=1, D=128, seed=150)
        ramp = torch.linspace(0, 40, 15 * 64).view(15, 64)
        for lb in range(15):
            r.k_pages[r.table[0, lb].long(), 0] += (sign * ramp[lb])[:, None].to(BF)
        q = randn(40, 4, 128, seed=151) * 0.1 + 1.0
        q = q.to(BF)
        x = q.double().abs().amax().item() * 128 * 45 / math.sqrt(128)     # |score| bound: its fp32 error
        want, tol, live = attention(r, q)
        tol = tol + 2 * x * 128 * 2.0 ** -24 * r.v_pages.nan_to_num().abs().max().item()
        for splits in (1, 4):
            _check(_attend(r, q, num_splits=splits), want, tol, live, f"sign {sign} splits {splits}")


def test_chunk_attention_bad_pages_are_skipped():
    r = Ragged([64], [400], page=32, Hkv=2, D=64, seed=152)
    q = randn(64, 4, 64, seed=153)
    table = r.table.clone()
    table[0, 2], table[0, 5] = 10 ** 6, -1
    sel = torch.tensor([[x for x in range(13) if x not in (2, 5)] + [0, 0]] * 2, dtype=torch.int32).expand(2, 2, 13)
    off = torch.tensor([[0, 11]] * 2, dtype=torch.int32).expand(2, 2, 2)
    want, tol, live = attention(r, q, sel, off)
    r.table = table
    _check(_attend(r, q), want, tol, live, "bad pages")


def test_chunk_attention_strided_and_out_of_pool_rows():
    """Queries and outputs as views of wider rows, pools as views of [P, page, Hkv, D] storage."""
    r = Ragged([40, 9], [100, 9], page=16, Hkv=2, D=64, seed=154)
    wide = randn(49, 3 * 6 * 64, seed=155)
    q = wide.view(49, 18, 64)[:, 6:12]
    pools = [p.transpose(1, 2).contiguous().cuda().transpose(1, 2) for p in (r.k_pages, r.v_pages)]
    out = torch.zeros(49, 8, 64, dtype=BF, device="cuda")
    ops.paged_chunk_attn(wide.cuda().view(49, 18, 64)[:, 6:12], *pools, *r.gpu("table", "cu", "kv_lens"), out=out[:, 1:7])
    want, tol, live = attention(r, q)
    _check(out[:, 1:7].cpu(), want, tol, live, "strided")
    assert not out[:, 0].any() and not out[:, 7].any()


# ---- paged_block_select ------------------------------------------------------------------------

def _select_case(q_lens, kv_lens, page, Hq, Hkv, D, dtype, top_k, sink, recent, tokens, ties=False, seed=200):
    r = Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=seed, poison=False)
    r.k_pages += randn(r.k_pages.size(0), Hkv, 1, D, seed=seed + 5, dtype=dtype)
    bounds = bounds_of(r)
    if ties:
        bounds[:] = bounds[:1]
    q = randn(r.N, Hq, D, seed=seed + 6, dtype=dtype)
    want = select(r, q, bounds, top_k=top_k, sink=sink, recent=recent, tokens=tokens)
    table, cu, lens = r.gpu("table", "cu", "kv_lens")
    got = ops.paged_block_select(q.cuda(), bounds.cuda(), table, lens, page=page, top_k=top_k, sink=sink, recent=recent,
                                 cu_seqlens=None if tokens else cu)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    return r, q, got


@pytest.mark.parametrize("page,D,dtype,top_k,sink,recent", [
    (64, 128, BF, 4, 1, 2), (16, 64, HF, 20, 2, 1), (32, 128, BF, 0, 1, 1), (128, 128, BF, 3, 0, 3), (48, 64, BF, 7, 0, 1)])
def test_select_single_tokens(page, D, dtype, top_k, sink, recent):
    _say("select tokens", page, D, dtype, top_k, sink, recent)
    lens = [1, page, page + 1, 0, 10 * page, 37 * page + 5, 300, 5]
    r, q, (sel, off) = _select_case([1] * 8, lens, page, 6, 2, D, dtype, top_k, sink, recent, True)
    out = ops.paged_sparse_decode(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "kv_lens"), sel, off, num_splits=0)
    want, tol, live = attention(r, q, sel.cpu(), off.cpu())
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.2f} of the bound"


@pytest.mark.parametrize("lists", [1, 200])
def test_select_many_pages(lists):
    """300 pages and more, few lists (scores by workgroups of their own) and many (by the list's own)."""
    _say("select many", lists)
    _select_case([1] * lists, [16 * 300 + 3 + 16 * (b % 40) for b in range(lists)], 16, 2, 1, 64, BF, 33, 1, 2, True)


@pytest.mark.parametrize("lists,pages", [(1, 257), (64, 257), (65, 257), (3, 600), (65, 513), (1, 4096)])
@pytest.mark.parametrize("ties", [False, True])
def test_select_borders_of_the_forms(lists, pages, ties):
    """On both sides of where pages are scored apart, and of where a list takes a larger workgroup; short lists among them."""
    _say("select borders", lists, pages, ties)
    _select_case([1] * lists, [16 * pages - 7 * b for b in range(lists - 1)] + [16 * pages if lists == 1 else 20], 16, 2, 1,
                 64, BF, 33, 1, 2, True, ties=ties, seed=230)


def test_select_chunks_scored_apart():
    _say("select chunks apart")
    _select_case([130, 0, 1, 64, 65], [16 * 300, 50, 16 * 280 + 3, 64, 16 * 520], 16, 4, 2, 128, HF, 20, 1, 1, False, seed=240)


def test_select_apart_on_a_replayed_graph():
    """Each replay scores the queries of that moment, in the same workspace."""
    _say("select graph")
    r, q, (sel, off) = _select_case([1] * 2, [16 * 400, 16 * 300 + 3], 16, 4, 2, 64, BF, 9, 1, 1, True, seed=250)
    bounds, (table, lens) = bounds_of(r).cuda(), r.gpu("table", "kv_lens")
    x = q.cuda()
    pick = dict(page=16, top_k=9, sink=1, recent=1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.paged_block_select(x, bounds, table, lens, **pick)
    for i in range(4):
        x.copy_(randn(*q.shape, seed=260 + i))
        g.replay()
        want = ops.paged_block_select(x, bounds, table, lens, **pick)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert torch.equal(got[0].cpu(), select(r, x.cpu(), bounds.cpu(), tokens=True, top_k=9, sink=1, recent=1)[0]), i


def test_select_in_a_given_workspace():
    """What the workspace holds does not matter, and what is behind the bytes needed stays; one too small is refused."""
    _say("select workspace")
    r, q, (sel, off) = _select_case([1] * 2, [16 * 400, 16 * 300 + 3], 16, 4, 2, 64, BF, 9, 1, 1, True, seed=270)
    bounds, (table, lens) = bounds_of(r).cuda(), r.gpu("table", "kv_lens")
    need = 2 * 2 * table.size(1) * 8
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    pick = dict(page=16, top_k=9, sink=1, recent=1)
    got = ops.paged_block_select(q.cuda(), bounds, table, lens, workspace=ws, **pick)
    assert torch.equal(got[0], sel) and torch.equal(got[1], off)
    assert (ws[need:] == 255).all()
    with pytest.raises(AssertionError, match="workspace"):
        ops.paged_block_select(q.cuda(), bounds, table, lens, workspace=ws[:need - 16], **pick)


@pytest.mark.parametrize("ties", [False, True])
def test_select_more_pages_than_lds_holds(ties):
    _say("select 5000 pages")
    _select_case([1] * 2, [16 * 5000, 16 * 4999 + 1], 16, 2, 1, 64, BF, 100, 1, 1, True, ties=ties)


@pytest.mark.parametrize("page,D,dtype,top_k,sink,recent", [
    (64, 128, BF, 3, 1, 2), (16, 64, HF, 9, 2, 1), (32, 64, BF, 0, 0, 1), (128, 128, BF, 2, 0, 1)])
def test_select_chunks_and_attend(page, D, dtype, top_k, sink, recent):
    _say("select chunk", page, D, dtype, top_k, sink, recent)
    r, q, (sel, off) = _select_case([130, 0, 1, 64, 65], [1000, 50, 700, 64, 1500], page, 4, 2, D, dtype, top_k, sink,
                                    recent, False)
    got = _attend(r, q, sel=sel, sel_off=off)
    want, tol, live = attention(r, q, sel.cpu(), off.cpu())
    _check(got, want, tol, live, "selected chunk")


def test_more_sequences_than_new_tokens():
    """Two new tokens among nine sequences, and none at all: rows of lists past the last block are empty."""
    r, q, (sel, off) = _select_case([0, 0, 1, 0, 0, 0, 1, 0, 0], [70, 0, 900, 1, 5, 64, 333, 8, 2], 64, 4, 2, 128, BF, 2, 1, 1,
                                    False)
    assert sel.size(0) == 9 and not off[2:].any()
    want, tol, live = attention(r, q, sel.cpu(), off.cpu())
    _check(_attend(r, q, sel=sel, sel_off=off), want, tol, live, "two of nine")
    for n in (0, 3):
        q = torch.zeros(0, 4, 64, dtype=BF, device="cuda")
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
        bd, table = torch.zeros(2, 2, 2, 64, dtype=BF, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda")
        cu, lens = i32(*[0] * (n + 1)), i32(*[9] * n)
        sel, off = ops.paged_block_select(q, bd, table, lens, page=64, top_k=1, cu_seqlens=cu)
        assert sel.shape[:2] == (n, 2) and not sel.any() and not off.any()
        pool = torch.zeros(2, 2, 64, 64, dtype=BF, device="cuda")
        assert ops.paged_chunk_attn(q, pool, pool, table, cu, lens, sel=sel, sel_off=off).shape == q.shape
        ops.paged_append(q[:, :2], q[:, :2], pool, pool.clone(), table, cu, lens, k_bounds=bd)


@pytest.mark.parametrize("tokens", [True, False])
def test_select_ties_go_to_the_lowest_page(tokens):
    _select_case([1, 1], [64 * 30, 64 * 9], 64, 4, 2, 128, BF, 5, 1, 1, tokens, ties=True)


def test_select_nan_bounds_and_bad_pages_rank_last():
    r = Ragged([1], [64 * 12], page=64, Hkv=1, D=64, seed=230, poison=False)
    bounds = bounds_of(r)
    q = randn(1, 2, 64, seed=231)
    plain = select(r, q, bounds, top_k=11, sink=0, recent=1, tokens=True)[0]
    assert plain[0, 0].tolist() == list(range(12))
    bounds[r.table[0, 3].long()] = math.nan
    table = r.table.clone()
    table[0, 7] = 10 ** 6
    got = ops.paged_block_select(q.cuda(), bounds.cuda(), table.cuda(), r.kv_lens.cuda(), page=64, top_k=9, sink=0, recent=1)
    assert got[0][0, 0].tolist() == [0, 1, 2, 4, 5, 6, 8, 9, 10, 11]


# ---- together, streams, graphs -------------------------------------------------------------------

def _step(st, r, x, sel_args):
    q, k, v = x
    qo = ops.paged_append(k, v, st["kp"], st["vp"], st["table"], st["cu"], st["lens"], inv_freq=st["inv"], k_weight=st["w"],
                          eps=EPS, k_bounds=st["bd"], q=q, q_weight=st["w"])
    dense = ops.paged_chunk_attn(qo, st["kp"], st["vp"], st["table"], st["cu"], st["lens"])
    sel, off = ops.paged_block_select(qo, st["bd"], st["table"], st["lens"], page=r.page, cu_seqlens=st["cu"], **sel_args)
    sparse = ops.paged_chunk_attn(qo, st["kp"], st["vp"], st["table"], st["cu"], st["lens"], sel=sel, sel_off=off)
    return qo, dense, sel, off, sparse


def _state(r, D):
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    return dict(kp=kp, vp=vp, table=table, cu=cu, lens=lens, inv=_inv(D).cuda(), w=(randn(D, seed=9) * 0.1 + 1).cuda(),
                bd=bounds_of(r).cuda())


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [700, 65, 2000]), ([100, 3, 0, 250], [400, 900, 77, 250])])
def test_a_step_of_all_four(q_lens, kv_lens):
    """Append, attend, select, attend, each on what the one before left: against float64 on the same pages."""
    r = Ragged(q_lens, kv_lens, page=64, Hkv=2, D=128, seed=240, poison=False)
    st = _state(r, 128)
    x = [randn(r.N, h, 128, seed=241 + i).cuda() for i, h in enumerate((8, 2, 2))]
    pick = dict(top_k=2, sink=1, recent=1)
    qo, dense, sel, off, sparse = _step(st, r, x, pick)
    r.k_pages, r.v_pages = st["kp"].cpu(), st["vp"].cpu()
    q = qo.cpu()
    want, tol, live = attention(r, q)
    _check(dense.cpu(), want, tol, live, "dense")
    ws, wo = select(r, q, st["bd"].cpu(), top_k=2, sink=1, recent=1, tokens=False)
    assert torch.equal(sel.cpu(), ws) and torch.equal(off.cpu(), wo)
    want, tol, live = attention(r, q, ws, wo)
    _check(sparse.cpu(), want, tol, live, "sparse")


def test_graph_replays_give_the_eager_bits():
    """The four in one captured graph; inputs, lengths and table entries change between the replays."""
    r = Ragged([1] * 6, [700, 65, 2000, 64, 1, 900], page=64, Hkv=2, D=128, seed=250, poison=False)
    pick = dict(top_k=3, sink=1, recent=2)
    st, ref = _state(r, 128), _state(r, 128)
    x = [randn(6, h, 128, seed=251 + i).cuda() for i, h in enumerate((8, 2, 2))]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(st, r, x, pick)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(st, r, x, pick)
    for i in range(4):
        for t, h in zip(x, (8, 2, 2)):
            t.copy_(randn(6, h, 128, seed=260 + 10 * i + h))
        if i % 2:
            for s in (st, ref):
                s["lens"].sub_(1).clamp_(min=1)
        want = _step(ref, r, x, pick)
        torch.cuda.synchronize()
        st["kp"].copy_(ref["kp"])
        st["vp"].copy_(ref["vp"])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), f"replay {i}"
        st["bd"].copy_(ref["bd"])


def test_two_streams_at_once():
    """Calls on two streams, each with tensors and workspaces of its own, give their single-stream bits."""
    cases = []
    for s in range(2):
        r = Ragged([64, 3], [640 + 64 * s, 300], page=32, Hkv=2, D=128, seed=270 + s)
        cases.append((r, randn(r.N, 8, 128, seed=280 + s)))
    alone = [_attend(r, q, num_splits=4) for r, q in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    args = [(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")) for r, q in cases]
    torch.cuda.synchronize()
    outs = [[] for _ in cases]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.paged_chunk_attn(*args[i], num_splits=4))
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        for o in got:
            assert torch.equal(o.cpu(), want)


# ---- refusals ----------------------------------------------------------------------------------

def test_refusals():
    r = Ragged([4], [70], page=64, Hkv=2, D=64, seed=290)
    kp, vp, table, cu, lens = r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens")
    q, k = randn(4, 4, 64, seed=291).cuda(), randn(4, 2, 64, seed=292).cuda()
    inv = _inv(64).cuda()
    pos = torch.arange(4, device="cuda")
    bad = [
        lambda: ops.qk_norm_rope(q.float(), k.float(), pos, inv),
        lambda: ops.qk_norm_rope(q, k, pos.int(), inv),
        lambda: ops.qk_norm_rope(q, k[:3], pos, inv),
        lambda: ops.qk_norm_rope(q, k, pos, inv.double()),
        lambda: ops.qk_norm_rope(q, k, pos, inv, q_weight=torch.ones(32, dtype=BF, device="cuda")),
        lambda: ops.qk_norm_rope(q.transpose(1, 2).contiguous().transpose(1, 2), k, pos, inv),
        lambda: ops.paged_append(k, k.half(), kp, vp, table, cu, lens),
        lambda: ops.paged_append(k, k, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), table, cu, lens),
        lambda: ops.paged_append(k, k, kp, vp, table, cu[:1], lens),
        lambda: ops.paged_append(k, k, kp, vp, table.long(), cu, lens),
        lambda: ops.paged_append(k, k, kp, vp, table, cu, lens, k_bounds=torch.zeros(2, 2, 2, 64, dtype=BF, device="cuda")),
        lambda: ops.paged_append(k, k, kp, vp, table, cu, lens, q_weight=torch.ones(64, dtype=BF, device="cuda")),
        lambda: ops.paged_append(k, k, kp, vp, table, cu, lens.cpu()),
        lambda: ops.paged_chunk_attn(q[:, :3], kp, vp, table, cu, lens),
        lambda: ops.paged_chunk_attn(q, kp, vp, table, cu, lens, sel=torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")),
        lambda: ops.paged_chunk_attn(q, kp, vp, table, cu, lens, num_splits=2,
                                     workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")),
        lambda: ops.paged_chunk_attn(q, kp, vp, table, cu, lens, out=torch.zeros_like(q, dtype=HF)),
        lambda: ops.paged_block_select(q, torch.zeros(4, 2, 2, 64, dtype=BF, device="cuda"), table, lens, page=64, top_k=1),
        lambda: ops.paged_block_select(q[:1], torch.zeros(4, 2, 2, 64, dtype=BF, device="cuda"), table, lens, page=64,
                                       top_k=-1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            pytest.fail(f"call {i} was let through")
    from sparseattentioninfer_amd._lib import HipCallError
    for f in (lambda: ops.paged_chunk_attn(q, kp, vp, table, cu, lens, num_splits=65),
              lambda: ops.paged_chunk_attn(q, kp, vp, table, cu, lens, sm_scale=0.0),
              lambda: ops.paged_block_select(q[:1], torch.zeros(4, 2, 2, 64, dtype=BF, device="cuda"), table, lens,
                                             page=24, top_k=1)):
        with pytest.raises(HipCallError):
            f()
