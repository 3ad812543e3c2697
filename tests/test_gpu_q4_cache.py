"""The 4-bit paged cache written (``paged_append_q4``) and read back (``paged_read_q4``) against its definition in float64: bytes
of values and of keys that are stored as they are, bounds of normed and rotated ones, the places of what is written."""
import math

import pytest
import torch

from sparseattentioninfer_amd import ops
from tests.chunk_reference import assert_rotated, randn, rotate
from tests.q4_reference import Q4Ragged, codes_of, pack, quantise, stats_of, unpack, value_of

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[q4-cache]", *msg, flush=True)


def _inv(D, theta=1e6):
    return (1.0 / theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).float()


def _gpu(t):
    return None if t is None else t.cuda()


def _rows_of(pool, r, b, p, values):
    """(codes, scale, minimum) of positions p of sequence b, heads second."""
    phys, slot = r.table[b, p // r.page].long(), p % r.page
    s, m = stats_of(pool, r.page, r.D, r.dtype)
    return tuple(x[phys, :, slot] for x in (codes_of(pool, r.page, r.D, values), s, m))


# ---- reading back ------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (128, HF), (64, BF)])
def test_read_ragged(page, D, dtype):
    """The last tokens of each sequence: none, one, whole sequences, starts inside a chunk of 16; rows of no sequence stay."""
    _say("read", page, D, dtype)
    r = Q4Ragged([130, 0, 1, 77, 16, 300, 3], [130, 40, 90, 200, 16, 431, 66], page=page, Hkv=3, D=D, dtype=dtype, seed=page,
                 pad_rows=5, offset=0.5)
    out = [torch.full((r.N, 3, D), 7.0, dtype=dtype, device="cuda") for _ in "kv"]
    got = ops.paged_read_q4(*r.gpu("k4", "v4", "table", "cu", "kv_lens"), rows=r.N, head_dim=D, dtype=dtype, k_out=out[0],
                            v_out=out[1])
    assert got[0] is out[0] and got[1] is out[1]
    for g, pages in zip(got, (r.k_pages, r.v_pages)):
        g = g.cpu()
        for b, at, t, n in r.rows():
            want = r.cached(pages, b, n)[:, n - t:].transpose(0, 1).float().to(dtype)
            assert torch.equal(g[at:at + t], want), (b, t, n)
        assert (g[sum(r.q_lens):] == 7.0).all()


def test_read_strided_outputs_and_missing_pages():
    """Outputs inside a wider tensor; ids outside the pool and tokens past the table read as zeros."""
    _say("read strided, missing pages")
    r = Q4Ragged([70, 64], [70, 100], page=32, Hkv=2, D=128, seed=3, extra_cols=0)
    r.table[0, 1] = -1
    r.table[1, 2] = 99
    wide = torch.full((r.N, 2, 3, 128), 5.0, dtype=BF, device="cuda")
    lens = torch.tensor([70, 200], dtype=torch.int32)        # the second reaches past the table's 4 columns
    k, v = ops.paged_read_q4(*r.gpu("k4", "v4", "table", "cu"), lens.cuda(), rows=r.N, head_dim=128, dtype=BF,
                             k_out=wide[:, :, 0], v_out=wide[:, :, 2])
    assert (wide[:, :, 1] == 5.0).all()
    for b, at, t, _ in r.rows():
        n = int(lens[b])
        for i in range(t):
            p = n - t + i
            lb = p // 32
            pg = int(r.table[b, lb]) if lb < r.table.size(1) else -1
            for g, pages in ((k, r.k_pages), (v, r.v_pages)):
                want = pages[pg, :, p % 32].float().to(BF) if 0 <= pg < r.k4.size(0) else torch.zeros(2, 128, dtype=BF)
                want = torch.zeros(2, 128, dtype=BF) if not 0 <= pg < r.k4.size(0) else want
                assert torch.equal(g[at + i].cpu().nan_to_num(9.0), want.nan_to_num(9.0)), (b, i)


# ---- writing -----------------------------------------------------------------------------------

def _append(q_lens, kv_lens, page, Hq, Hkv, D, dtype, *, norm, rope, bounds, pad=0, seed=10, scale=2.0, offset=0.0):
    r = Q4Ragged(q_lens, kv_lens, page=page, Hkv=Hkv, D=D, dtype=dtype, seed=seed, pad_rows=pad)
    before = r.k4.clone(), r.v4.clone()
    row = randn(r.N, (Hq + 2 * Hkv) * D, seed=seed + 3, dtype=dtype, scale=scale) + offset
    q, k, v = (x.unflatten(1, (-1, D)) for x in row.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    qw, kw = (randn(D, seed=seed + s, dtype=dtype, scale=0.3) + 1 if norm else None for s in (4, 5))
    inv = _inv(D) if rope else None
    bd = randn(r.k4.size(0), Hkv, 2, D, seed=seed + 6, dtype=dtype).sort(dim=2).values if bounds else None
    kp, vp, gb, grow = _gpu(r.k4), _gpu(r.v4), _gpu(bd), row.cuda()
    gq, gk, gv = (x.unflatten(1, (-1, D)) for x in grow.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    q_out = torch.full((r.N, Hq, D), 7.0, dtype=dtype, device="cuda")
    ops.paged_append_q4(gk, gv, kp, vp, *r.gpu("table", "cu", "kv_lens"), inv_freq=_gpu(inv), k_weight=_gpu(kw), eps=EPS,
                        k_bounds=gb, q=gq, q_weight=_gpu(qw), q_out=q_out)
    kp, vp, q_out = kp.cpu(), vp.cpu(), q_out.cpu()
    back = unpack(kp, page, D, dtype, False)
    written = torch.zeros(kp.size(0), page, dtype=torch.bool)
    new_lo = torch.full((kp.size(0), Hkv, D), math.inf, dtype=torch.float64)
    new_hi, fresh = -new_lo, torch.zeros(kp.size(0), dtype=torch.bool)
    for b, at, t, n in r.rows():
        p = torch.arange(n - t, n)
        ok = p >= 0
        want, terms = rotate(q[at:at + t], qw, p, inv, EPS)
        assert_rotated(q_out[at:at + t], want, terms, f"q of sequence {b}")
        p = p[ok]
        phys, slot = r.table[b, p // page].long(), p % page
        # values: bit for bit
        code, s, m = quantise(v[at:at + t][ok])
        got = _rows_of(vp, r, b, p, True)
        assert torch.equal(got[0], code) and torch.equal(got[1], s) and torch.equal(got[2], m), f"v of sequence {b}"
        got = _rows_of(kp, r, b, p, False)
        if not norm and not rope:
            code, s, m = quantise(k[at:at + t][ok])
            assert torch.equal(got[0], code) and torch.equal(got[1], s) and torch.equal(got[2], m), f"k of sequence {b}"
        else:
            # The key before quantisation is off by at most `tol` (assert_rotated's bound), the minimum by the largest of
            # its group; the quantised value by half a step of the stored scale more.
            want, terms = rotate(k[at:at + t][ok], kw, p, inv, EPS)
            h = torch.finfo(dtype).eps / 2
            tol = (h * want.abs() + 2.0 ** -20 * terms) * (1 + h) + torch.finfo(torch.float16).tiny * 2.0 ** -10
            in_groups = lambda x: x.unflatten(-1, (-1, 32))
            worst = in_groups(tol).amax(-1)
            s, m = got[1].double(), got[2].double()
            assert ((m - in_groups(want).amin(-1)).abs() <= worst).all(), f"minima of sequence {b}"
            true = (in_groups(want).amax(-1) - in_groups(want).amin(-1)) / 15
            assert (s <= true + 2 * worst / 15).all() and (s >= (true - 2 * worst / 15) * (1 - 2 * h)).all(), f"scales of {b}"
            err = in_groups((value_of(*got) - want).abs())
            assert (err <= (s[..., None] / 2) * (1 + 2.0 ** -18) + in_groups(tol)).all(), f"k of sequence {b}"
        written[phys, slot] = True
        for pg in phys.unique().tolist():
            kk = back[pg][:, slot[phys == pg]]
            new_lo[pg], new_hi[pg] = kk.amin(1), kk.amax(1)
            fresh[pg] = bool((slot[phys == pg] == 0).any())
    assert (q_out[sum(q_lens):] == 7.0).all()          # rows of no sequence
    # every byte of other slots is as it was
    for pool, old, values in ((kp, before[0], False), (vp, before[1], True)):
        keep = ~written[:, None, :, None]
        a, o = (codes_of(x, page, D, values) for x in (pool, old))
        assert torch.equal(a.masked_select(keep), o.masked_select(keep))
        for x, y in zip(stats_of(pool, page, D, dtype), stats_of(old, page, D, dtype)):
            assert torch.equal(x.view(torch.int16).masked_select(keep), y.view(torch.int16).masked_select(keep))
    if bounds:
        touched = written.any(1)
        lo, hi = new_lo.float().to(dtype), new_hi.float().to(dtype)
        merge = (~fresh)[:, None, None]
        lo = torch.where(merge, torch.minimum(lo, bd[:, :, 0]), lo)
        hi = torch.where(merge, torch.maximum(hi, bd[:, :, 1]), hi)
        got = gb.cpu()
        assert torch.equal(got[touched], torch.stack([lo, hi], 2)[touched]) and torch.equal(got[~touched], bd[~touched])


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (128, HF), (64, BF)])
def test_append_ragged(page, D, dtype):
    _say("append", page, D, dtype)
    _append([130, 0, 1, 77, 16, 300, 3], [130, 40, 90, 200, 16, 431, 66], page, 6, 2, D, dtype, norm=True, rope=True,
            bounds=True, pad=5)


@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (128, HF), (64, BF)])
@pytest.mark.parametrize("offset", [0.0, 20.0])
def test_append_as_they_are(D, dtype, offset):
    """No norm, no rotation: keys bit for bit too, also where a group's range is small against its values."""
    _say("append plain", D, dtype, offset)
    _append([50, 1, 200], [50, 64, 333], 64, 4, 4, D, dtype, norm=False, rope=False, bounds=True, offset=offset)


@pytest.mark.parametrize("B", [1, 64, 65, 130])
def test_append_single_tokens(B):
    _say("append tokens", B)
    lens = [(1, 64, 65, 1000, 128, 7)[b % 6] for b in range(B)]
    _append([1] * B, lens, 64, 8, 2, 128, BF, norm=True, rope=True, bounds=B % 2 == 0)


def test_append_token_by_token_equals_one_chunk():
    """The bytes of a sequence do not depend on how its tokens came."""
    _say("append token by token")
    for D, dtype in ((128, BF), (64, HF)):
        N, Hkv, page = 37, 2, 16
        k, v = (randn(N, Hkv, D, seed=s, dtype=dtype).cuda() for s in (1, 2))
        table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
        pools = []
        for steps in ([N], [1] * N, [5, 2, 9, 1, 20]):
            kp, vp = (torch.zeros(4, Hkv, ops.q4_block_bytes(page, D), dtype=torch.uint8, device="cuda") for _ in "kv")
            at = 0
            for t in steps:
                ops.paged_append_q4(k[at:at + t], v[at:at + t], kp, vp, table, torch.tensor([0, t], dtype=torch.int32).cuda(),
                                    torch.tensor([at + t], dtype=torch.int32).cuda(), inv_freq=_inv(D).cuda())
                at += t
            pools.append((kp, vp))
        for kp, vp in pools[1:]:
            assert torch.equal(kp, pools[0][0]) and torch.equal(vp, pools[0][1])


def test_append_extremes():
    """Groups of equal values, of the type's largest, of one outlier, of zeros; NaN and infinities make their group NaN."""
    _say("append extremes")
    for dtype in (BF, HF):
        top = torch.finfo(dtype).max
        x = randn(16, 2, 128, seed=5, dtype=dtype)
        x[0] = 1.5
        x[1] = 0.0
        x[2, :, ::2], x[2, :, 1::2] = top, -top
        x[3, :, 7] = 300.0
        x[4] = 3.0 * torch.finfo(dtype).tiny
        x[4, 0, 5] = 4.0 * torch.finfo(dtype).tiny
        x[5, 0, 40] = math.nan
        x[5, 1, 100] = math.inf
        x[6, 0, 0] = -math.inf
        x[7] = torch.arange(128).to(dtype)[None] / 2                        # ties
        kp, vp = (torch.zeros(1, 2, ops.q4_block_bytes(16, 128), dtype=torch.uint8, device="cuda") for _ in "kv")
        one = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")
        ops.paged_append_q4(x.cuda(), x.cuda(), kp, vp, one(0)[None], one(0, 16), one(16))
        back = ops.paged_read_q4(kp, vp, one(0)[None], one(0, 16), one(16), rows=16, head_dim=128, dtype=dtype)
        code, s, m = quantise(x)
        want = value_of(code, s, m).float().to(dtype)
        assert want.isnan().sum() == 3 * 32
        for g in back:
            g = g.cpu()
            assert torch.equal(g.isnan(), want.isnan())
            assert torch.equal(g.nan_to_num(1.0, math.inf, -math.inf), want.nan_to_num(1.0, math.inf, -math.inf))
            assert g[2].isfinite().all()
        assert torch.equal(kp.cpu()[:, :, :1024][0, :, :].unflatten(-1, (16, 64))[:, :5], pack(x.transpose(0, 1), False)[:, :1024].unflatten(-1, (16, 64))[:, :5])


def test_append_places_without_pages_are_not_written():
    _say("append missing pages")
    kp, vp = (torch.full((3, 1, ops.q4_block_bytes(16, 64)), 3, dtype=torch.uint8, device="cuda") for _ in "kv")
    x = randn(60, 1, 64, seed=1, dtype=HF).cuda()
    table = torch.tensor([[1, -1, 7]], dtype=torch.int32, device="cuda")    # tokens 48.. are past the table
    ops.paged_append_q4(x, x, kp, vp, table, torch.tensor([0, 60], dtype=torch.int32, device="cuda"),
                        torch.tensor([60], dtype=torch.int32, device="cuda"))
    want = pack(x.cpu()[None, :16].transpose(1, 2), False)[0]
    assert torch.equal(kp.cpu()[1], want) and (kp[[0, 2]] == 3).all() and (vp[[0, 2]] == 3).all()
