"""Attention over the 4-bit cache within bounds that reject other outputs (tests/test_q4_bounds_host.py): keys and values far from
0, far from 1, scores far apart."""
import pytest
import torch

from sparseattentioninfer_amd import _lib, ops
from tests.chunk_reference import randn
from tests.q4_bounds import CHUNKS, DECODES, VALUES, cache_of, forms, good_rows

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _say(*msg):
    print("[q4-bounds]", *msg, flush=True)


def _assert(got, bounds, what):
    good = good_rows(got, bounds)
    over = min((((got.double().cpu() - want).abs() - tol).max().item() for want, tol, _ in bounds))
    assert good.all(), f"{what}: {int((~good).sum())} of {good.numel()} rows, worst {over:.3e} past the bound"


@pytest.mark.parametrize("values", VALUES, ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (128, HF), (64, BF)])
def test_decode(D, dtype, values):
    for lens in DECODES:
        r = cache_of([1] * len(lens), lens, page=32, Hkv=2, D=D, dtype=dtype, seed=4, **values)
        q = randn(len(lens), 8, D, seed=9, dtype=dtype)
        bounds = [forms(r, q, codes=True)]
        for splits in (0, 1, 5):
            _say("decode", D, dtype, values, lens, splits)
            out = ops.paged_sparse_decode_q4(q.cuda(), *r.gpu("k4", "v4", "table", "kv_lens"), num_splits=splits)
            _assert(out, bounds, f"{values} {lens} {splits}")


@pytest.mark.parametrize("values", VALUES, ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_chunk(D, dtype, values):
    for q_lens, kv_lens in CHUNKS:
        r = cache_of(q_lens, kv_lens, page=32, Hkv=2, D=D, dtype=dtype, seed=5, **values)
        q = randn(r.N, 8, D, seed=9, dtype=dtype)
        bounds = [forms(r, q, codes=True), forms(r, q, codes=False)]
        for splits in (0, 1, 3):
            _say("chunk", D, dtype, values, kv_lens, splits)
            out = ops.paged_chunk_attn_q4(q.cuda(), *r.gpu("k4", "v4", "table", "cu", "kv_lens"), num_splits=splits)
            _assert(out, bounds, f"{values} {q_lens} {kv_lens} {splits}")


def test_chunk_workspaces():
    """A workspace of a call's own, its contents arbitrary, on another stream; one that is too small or not 16-byte aligned is
    refused."""
    _say("chunk workspace")
    r = cache_of([3, 70], [300, 900], page=32, Hkv=2, D=128, dtype=BF, seed=5)
    q = randn(r.N, 8, 128, seed=9)
    args = (q.cuda(), *r.gpu("k4", "v4", "table", "cu", "kv_lens"))
    want = ops.paged_chunk_attn_q4(*args, num_splits=3)
    need = _lib.load().sa_paged_chunk_workspace_bytes(r.N, 2, 8, 2, 128, r.table.size(1) * 32, 3)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.paged_chunk_attn_q4(*args, num_splits=3, workspace=ws[:need])
    s.synchronize()
    assert torch.equal(got, want) and (ws[need:] == 255).all()
    _assert(got, [forms(r, q, codes=True), forms(r, q, codes=False)], "workspace")
    with pytest.raises(AssertionError, match="workspace"):
        ops.paged_chunk_attn_q4(*args, num_splits=3, workspace=ws[:need - 16])
    with pytest.raises(RuntimeError, match="aligned"):
        ops.paged_chunk_attn_q4(*args, num_splits=3, workspace=ws[8:need + 8])
