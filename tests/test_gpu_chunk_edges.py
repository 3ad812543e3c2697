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
