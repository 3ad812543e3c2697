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
