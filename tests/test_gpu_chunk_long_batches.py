"""Chunk attention and page selection where the work of one item or one batch passes what its first look-up holds:
more key tiles than a window of 64, more sequences than the 64 lanes of a wave, planned divisions over whole caches
and over lists.

The values are sparse: token j holds 1 + (sequence % 7) in dim (j // 16) % D and 0 elsewhere, so every output is a sum of
few probabilities and its bound, relative to the sum, is below what one lost, doubled or exchanged chunk changes."""
import pytest
import torch

from sparseattentioninfer_amd import _lib, ops
from tests.chunk_reference import Ragged, attention, bounds_of, randn, select

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[chunk-long]", *msg, flush=True)


def _sparse_values(r):
    """Rewrites the values of the tokens that are there; other slots keep their NaN."""
    for b, n in enumerate(r.lens):
        for lb in range(-(-n // r.page)):
            j = torch.arange(lb * r.page, min(n, (lb + 1) * r.page))
            v = torch.zeros(len(j), r.D)
            v[torch.arange(len(j)), (j // 16) % r.D] = 1.0 + b % 7
            r.v_pages[r.table[b, lb].long(), :, :len(j)] = v.to(r.dtype)
    return r


def _bound(r, tol, want):
    """The accumulators add up to the keys' number of fp32 terms, all of one sign: that many half steps more at most."""
    return tol + 2 * max(r.lens) * 2.0 ** -24 * want.abs()


def _check(got, want, tol, live, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & live[:, None, None]
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {(err / tol)[live].max():.2f} of it"
    assert (got[~live] == 9.0).all(), f"{what}: rows of no sequence were written"


def _attend(r, q, **kw):
    out = torch.full_like(q, 9.0).cuda()
    ops.paged_chunk_attn(q.cuda(), *r.gpu("k_pages", "v_pages", "table", "cu", "kv_lens"), out=out, **kw)
    return out.cpu()


def _lists(r, rows, keep, seed):
    """Ascending random lists of ``keep`` of the pages, one for each list row and KV head."""
    g = torch.Generator().manual_seed(seed)
    pages = -(-max(r.lens) // r.page)
    sel = torch.stack([torch.stack([torch.randperm(pages, generator=g)[:keep].sort().values for _ in range(r.Hkv)])
                       for _ in range(rows)]).to(torch.int32)
    off = torch.tensor([0, keep], dtype=torch.int32).expand(rows, r.Hkv, 2).contiguous()
    return sel, off


# new tokens times the group of 4: 12 rows (narrow, four waves share the keys), 20 tokens (wide, all keys in one workgroup)
@pytest.mark.parametrize("t", [3, 20])
@pytest.mark.parametrize("keys,page,D,dtype", [(4095, 64, 128, BF), (4097, 64, 128, BF), (8300, 16, 64, HF), (8300, 64, 128, BF),
                                               (12345, 128, 64, BF)])
def test_more_key_tiles_than_a_window(keys, page, D, dtype, t):
    _say("windows", keys, page, D, dtype, t)
    r = _sparse_values(Ragged([t], [keys], page=page, Hkv=1, D=D, dtype=dtype, seed=500))
    q = randn(t, 4, D, seed=501, dtype=dtype)
    want, tol, live = attention(r, q)
    _check(_attend(r, q, num_splits=1), want, _bound(r, tol, want), live, "whole cache")
    pages = -(-keys // page)
    keep = pages - pages // 9
    assert keep * page > 64 * 64 or keys < 4200
    sel, off = _lists(r, 1 + t // 64, keep, seed=502)
    want, tol, live = attention(r, q, sel, off)
    _check(_attend(r, q, sel=sel.cuda(), sel_off=off.cuda(), num_splits=1), want, _bound(r, tol, want), live, "lists")


def _many(B):
    """0, 1, a few and many new tokens in turn, over lengths that differ; rows of no sequence behind them."""
    q_lens = [(1, 0, 3, 17, 1, 0, 2, 40)[b % 8] for b in range(B)]
    q_lens[B - 1] = 33
    q_lens[B // 2] = 70
    kv_lens = [t + (b * 37) % 331 + (700 if b % 13 == 5 else 0) for b, t in enumerate(q_lens)]
    return Ragged(q_lens, kv_lens, page=32, Hkv=2, D=64, dtype=BF, seed=510 + B, pad_rows=5)


_MANY = {}


def _many_case(B, selected):
    if (B, selected) not in _MANY:
        r = _sparse_values(_many(B))
        q = randn(r.N, 4, 64, seed=520 + B)
        lists = None
        if selected:
            lists = select(r, q, bounds_of(r), top_k=4, sink=1, recent=1, tokens=False)
        want, tol, live = attention(r, q, *(lists or ()))
        _MANY[B, selected] = r, q, lists, want, _bound(r, tol, want), live
    return _MANY[B, selected]


@pytest.mark.parametrize("splits", [1, 0, 3])
@pytest.mark.parametrize("selected", [False, True])
@pytest.mark.parametrize("B", [64, 65, 130])
def test_more_sequences_than_lanes(B, selected, splits):
    _say("sequences", B, "selected", selected, "splits", splits)
    r, q, lists, want, tol, live = _many_case(B, selected)
    kw = dict(sel=lists[0].cuda(), sel_off=lists[1].cuda()) if selected else {}
    _check(_attend(r, q, num_splits=splits, **kw), want, tol, live, f"{B} sequences")


@pytest.mark.parametrize("B", [64, 65, 130])
def test_selection_for_more_sequences_than_lanes(B):
    _say("selection", B)
    r, q, lists = _many_case(B, True)[:3]
    got = ops.paged_block_select(q.cuda(), bounds_of(r).cuda(), *r.gpu("table", "kv_lens"), page=32, top_k=4, sink=1,
                                 recent=1, cu_seqlens=r.cu.cuda())
    assert torch.equal(got[0].cpu(), lists[0]) and torch.equal(got[1].cpu(), lists[1])


# Lengths that the plan divides: few rows over many keys.
PLANNED = [  # q_lens, kv_lens, page, Hq, Hkv, D, dtype
    ([1], [6000], 64, 8, 2, 128, BF),
    ([4, 4, 1], [3000, 5001, 1700], 16, 8, 2, 64, HF),
    ([80], [3333], 64, 4, 1, 128, BF),
    ([30, 2, 0, 90], [4001, 2500, 9, 90], 128, 6, 2, 64, BF),
]


def _planned(r, q, keys, **kw):
    """Attention with a workspace of the size asked for; also whether partial results were left in it."""
    need = _lib.load().sa_paged_chunk_workspace_bytes(r.N, len(r.lens), q.size(1), r.Hkv, r.D, keys, 0)
    assert need > 0
    ws = torch.full((need,), 0xA5, dtype=torch.uint8, device="cuda")
    got = _attend(r, q, num_splits=0, workspace=ws, **kw)
    return got, bool((ws[(16 * len(r.lens) + 255) // 256 * 256:] != 0xA5).any())


@pytest.mark.parametrize("case", range(len(PLANNED)))
def test_planned_division(case):
    q_lens, kv_lens, page, Hq, Hkv, D, dtype = PLANNED[case]
    _say("planned", *PLANNED[case])
    r = _sparse_values(Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=540 + case, pad_rows=2))
    q = randn(r.N, Hq, D, seed=550 + case, dtype=dtype)
    want, tol, live = attention(r, q)
    got, divided = _planned(r, q, r.table.size(1) * page)
    _check(got, want, _bound(r, tol, want), live, "planned")
    assert divided


@pytest.mark.parametrize("case", range(len(PLANNED)))
def test_planned_division_over_lists(case):
    q_lens, kv_lens, page, Hq, Hkv, D, dtype = PLANNED[case]
    _say("planned lists", *PLANNED[case])
    r = _sparse_values(Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=560 + case, pad_rows=2, poison=False))
    q = randn(r.N, Hq, D, seed=570 + case, dtype=dtype)
    keep = 1280 // page          # 20 key tiles
    sel, off = select(r, q, bounds_of(r), top_k=keep, sink=1, recent=1, tokens=False)
    want, tol, live = attention(r, q, sel, off)
    got, divided = _planned(r, q, min(sel.size(2), r.table.size(1)) * page, sel=sel.cuda(), sel_off=off.cuda())
    _check(got, want, _bound(r, tol, want), live, "planned lists")
    assert divided
