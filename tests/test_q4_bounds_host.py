"""The bounds of attention over a 4-bit cache pass the result and no other output: in every case of the GPU tests that use them."""
import pytest
import torch

from tests.chunk_reference import randn
from tests.q4_bounds import CHUNKS, DECODES, VALUES, cache_of, forms, good_rows, wrong_outputs

BF, HF = torch.bfloat16, torch.float16


def _check(r, q, bounds, what):
    assert good_rows(bounds[0][0].to(q.dtype), bounds)[bounds[0][2] > 0].all(), what
    many = bounds[0][2] > 8                      # a row of a few keys may well be like its neighbour
    assert many.any()
    for name, out in wrong_outputs(r, bounds).items():
        passed = good_rows(out, bounds) & many
        assert not passed.any(), f"{what}: {int(passed.sum())} rows of {name} pass"


@pytest.mark.parametrize("values", VALUES, ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF), (128, HF), (64, BF)])
def test_decode_bounds_pass_the_result_only(D, dtype, values):
    for lens in DECODES:
        r = cache_of([1] * len(lens), lens, page=32, Hkv=2, D=D, dtype=dtype, seed=4, **values)
        q = randn(len(lens), 8, D, seed=9, dtype=dtype)
        _check(r, q, [forms(r, q, codes=True)], f"{values} {lens}")


@pytest.mark.parametrize("values", VALUES, ids=str)
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, HF)])
def test_chunk_bounds_pass_the_result_only(D, dtype, values):
    for q_lens, kv_lens in CHUNKS:
        r = cache_of(q_lens, kv_lens, page=32, Hkv=2, D=D, dtype=dtype, seed=5, **values)
        q = randn(r.N, 8, D, seed=9, dtype=dtype)
        _check(r, q, [forms(r, q, codes=True), forms(r, q, codes=False)], f"{values} {kv_lens}")
