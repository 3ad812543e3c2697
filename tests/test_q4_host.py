"""The 4-bit cache on the CPU: the byte form of its reference, and what the operators refuse before any device access."""
import pytest
import torch

from sparseattentioninfer_amd import _lib, ops
from tests.q4_reference import codes_of, pack, places, quantise, unpack, value_of


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,D", [(16, 64), (48, 128), (64, 128)])
def test_form(dtype, page, D):
    x = torch.randn(2, 3, page, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    code, s, m = quantise(x)
    for values in (False, True):
        byte, shift = places(page, D, values)
        assert sorted((byte * 8 + shift).flatten().tolist()) == list(range(0, page * D // 2 * 8, 4))   # every nibble once
        pool = pack(x, values)
        assert pool.shape == (2, 3, ops.q4_block_bytes(page, D))
        assert torch.equal(codes_of(pool, page, D, values), code)
        assert torch.equal(unpack(pool, page, D, dtype, values), value_of(code, s, m))
    err = (value_of(code, s, m) - x.double()).abs().unflatten(-1, (-1, 32))
    assert (err <= s.double()[..., None] / 2).all()
    assert (value_of(code, s, m).unflatten(-1, (-1, 32)).amax(-1) <= x.double().unflatten(-1, (-1, 32)).amax(-1)).all()


def test_block_bytes():
    assert ops.q4_block_bytes(64, 128) == 5120 and ops.q4_block_bytes(16, 64) == 640
    for page, D in ((8, 128), (40, 128), (144, 128), (64, 96)):
        with pytest.raises(AssertionError):
            ops.q4_block_bytes(page, D)


def test_calls_refuse_cpu_tensors():
    pool = torch.zeros(2, 1, 5120, dtype=torch.uint8)
    i = lambda *n: torch.tensor(n, dtype=torch.int32)
    x = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="on the GPU"):
        ops.paged_append_q4(x, x, pool, pool, i(0)[None], i(0, 1), i(1))
    with pytest.raises(AssertionError, match="on the GPU"):
        ops.paged_read_q4(pool, pool, i(0)[None], i(0, 1), i(1), rows=1, head_dim=128, dtype=torch.bfloat16)


FAKE = 1 << 12      # a 16-byte aligned stand-in address


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        from sparseattentioninfer_amd import _build
        _build.build(verbose=False)
    return _lib.load()


def _append(lib, **o):
    a = dict(dtype=0, k=FAKE, kp=FAKE, sp=10240, inv=FAKE, pos=None, pos_st=1, N=4, B=2, D=128, page=64, pages=8, mb=4, st=4,
             table=FAKE, Hkv=2, Hq=0, q=None)
    a.update(o)
    return lib.sa_paged_append_q4(a["dtype"], a["q"], 1024, 128, a["k"], 1024, 128, FAKE, 1024, 128, None, 0, 0, None, None,
                                  a["inv"], a["pos"], a["pos_st"], a["kp"], FAKE, a["sp"], 5120, a["pages"], None, 0, 0,
                                  a["table"], a["st"], a["mb"], FAKE, FAKE, a["N"], a["B"], a["Hq"], a["Hkv"], a["D"],
                                  a["page"], 1e-6, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=5), -1, b"dtype 5"), (dict(D=96), -3, b"head dim 96"), (dict(page=24), -4, b"page 24"),
    (dict(page=144), -4, b"page 144"), (dict(N=-1), -2, b"bad sizes"), (dict(mb=8), -2, b"8 columns"),
    (dict(k=None), -6, b"NULL"), (dict(kp=None), -6, b"NULL"), (dict(table=None), -6, b"NULL"), (dict(Hq=4), -6, b"NULL"),
    (dict(kp=FAKE + 8), -8, b"aligned"), (dict(sp=10248), -8, b"aligned"), (dict(k=FAKE + 2), -8, b"aligned"),
    (dict(pos=FAKE, inv=None), -6, b"inv_freq"), (dict(pos=FAKE, pos_st=-1), -2, b"stride -1")])
def test_append_refusals(lib, change, code, text):
    assert _append(lib, **change) == code and b"sa_paged_append_q4" in lib.sa_last_error() and text in lib.sa_last_error()


def test_append_nothing_to_do(lib):
    assert _append(lib, N=0, k=None) == 0 and _append(lib, B=0) == 0


def _read(lib, **o):
    a = dict(dtype=0, kp=FAKE, sp=10240, N=4, B=2, D=128, page=64, pages=8, mb=4, table=FAKE, Hkv=2, ko=FAKE, ko_st=256)
    a.update(o)
    return lib.sa_paged_read_q4(a["dtype"], a["kp"], FAKE, a["sp"], 5120, a["pages"], a["table"], 4, a["mb"], FAKE, FAKE,
                                a["ko"], a["ko_st"], 128, FAKE, 256, 128, a["N"], a["B"], a["Hkv"], a["D"], a["page"], None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), -1, b"dtype 2"), (dict(D=256), -3, b"head dim 256"), (dict(page=0), -4, b"page 0"),
    (dict(Hkv=0), -2, b"bad sizes"), (dict(mb=5), -2, b"5 columns"), (dict(kp=None), -6, b"NULL"),
    (dict(ko=None), -6, b"NULL"), (dict(table=None), -6, b"NULL"), (dict(kp=FAKE + 4), -8, b"aligned"),
    (dict(ko=FAKE + 2), -8, b"aligned"), (dict(ko_st=260), -8, b"aligned"), (dict(N=1 << 30, B=1 << 26), -2, b"too many")])
def test_read_refusals(lib, change, code, text):
    assert _read(lib, **change) == code and b"sa_paged_read_q4" in lib.sa_last_error() and text in lib.sa_last_error()


def test_read_nothing_to_do(lib):
    assert _read(lib, N=0, ko=None) == 0 and _read(lib, B=0) == 0


def _chunk(lib, **o):
    a = dict(dtype=0, kp=FAKE, sp=10240, pages=8, table=FAKE, mb=4, sel=None, rows=0, width=0, off=None, N=4, Hq=8, D=128, page=64,
             scale=0.1, splits=1, ws=None, q=FAKE)
    a.update(o)
    return lib.sa_paged_chunk_attn_q4(a["dtype"], a["q"], 1024, 128, a["kp"], a["kp"], a["sp"], 5120, a["pages"], a["table"],
                                      4, a["mb"], FAKE, FAKE, a["sel"], 8, 4, a["rows"], a["width"], a["off"], 8, 4, FAKE,
                                      1024, 128, a["N"], 2, a["Hq"], 2, a["D"], a["page"], a["scale"], a["splits"], a["ws"], 0,
                                      None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), -1, b"dtype 7"), (dict(D=80), -3, b"head dim 80"), (dict(page=20), -4, b"page 20"),
    (dict(Hq=9), -2, b"Hq=9"), (dict(mb=5), -2, b"5 columns"), (dict(splits=65), -2, b"65 splits"), (dict(scale=0.0), -2, b"scale"),
    (dict(q=None), -6, b"NULL"), (dict(kp=None), -6, b"NULL"), (dict(table=None), -6, b"NULL"),
    (dict(off=FAKE, rows=2, width=4), -6, b"NULL"), (dict(off=FAKE, rows=1, width=0), -2, b"selection"),
    (dict(sel=FAKE, rows=2, width=4), -2, b"selection"), (dict(kp=FAKE + 8), -8, b"aligned"), (dict(sp=10241), -8, b"aligned"),
    (dict(q=FAKE + 2), -8, b"aligned"), (dict(splits=2), -7, b"workspace")])
def test_chunk_refusals(lib, change, code, text):
    assert _chunk(lib, **change) == code and b"sa_paged_chunk_attn_q4" in lib.sa_last_error() and text in lib.sa_last_error()


def test_chunk_nothing_to_do(lib):
    assert _chunk(lib, N=0, q=None) == 0


def _decode(lib, **o):
    a = dict(dtype=0, kp=FAKE, sp=10240, pages=8, table=FAKE, mb=4, sel=None, rows=0, width=0, off=None, B=4, Hq=8, D=128, page=64,
             scale=0.1, splits=1, ws=None, q=FAKE, lens=FAKE)
    a.update(o)
    return lib.sa_decode_q4(a["dtype"], a["q"], 1024, 128, a["kp"], a["kp"], a["sp"], 5120, a["pages"], a["table"], 4, a["mb"],
                            a["lens"], a["sel"], 8, 4, a["width"], a["off"], 8, 4, a["rows"], FAKE, 1024, 128, a["B"], a["Hq"],
                            2, a["D"], a["page"], a["scale"], a["splits"], a["ws"], 0, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), -1, b"dtype 7"), (dict(D=32), -3, b"head dim 32"), (dict(page=136), -4, b"page 136"),
    (dict(Hq=9), -2, b"Hq=9"), (dict(mb=5), -2, b"5 columns"), (dict(splits=65), -2, b"65 splits"), (dict(splits=-1), -2, b"-1 splits"),
    (dict(scale=-1.0), -2, b"scale"), (dict(off=FAKE, sel=FAKE, rows=3, width=4), -5, b"sel_rows=3"),
    (dict(sel=FAKE), -2, b"selection"), (dict(off=FAKE, sel=FAKE, rows=2, width=-1), -2, b"selection"),
    (dict(off=FAKE, rows=2, width=4), -6, b"NULL"), (dict(lens=None), -6, b"NULL"), (dict(kp=None), -6, b"NULL"),
    (dict(kp=FAKE + 4), -8, b"aligned"), (dict(sp=8), -8, b"aligned"), (dict(splits=4), -7, b"workspace")])
def test_decode_refusals(lib, change, code, text):
    assert _decode(lib, **change) == code and b"sa_decode_q4" in lib.sa_last_error() and text in lib.sa_last_error()


def test_decode_nothing_to_do(lib):
    assert _decode(lib, B=0, q=None) == 0
    # 4 heads a workgroup at D = 128: 2 sequences, 2 lists, 3 shares; none in one share, nor of short lists
    assert lib.sa_decode_q4_workspace_bytes(2, 8, 2, 128, 6400, 0, 3) == 64 + 2 * 2 * 3 * 4 * 130 * 4
    assert lib.sa_decode_q4_workspace_bytes(2, 8, 2, 128, 6400, 0, 1) == 0
    assert lib.sa_decode_q4_workspace_bytes(2, 8, 2, 128, 512, 0, 0) == 0
    assert lib.sa_decode_q4_workspace_bytes(2, 8, 2, 128, 6400, 0, 0) > 0


def test_attention_refuses_cpu_tensors():
    pool = torch.zeros(2, 1, 5120, dtype=torch.uint8)
    i = lambda *n: torch.tensor(n, dtype=torch.int32)
    x = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="on the GPU"):
        ops.paged_chunk_attn_q4(x, pool, pool, i(0)[None], i(0, 1), i(1))
    with pytest.raises(AssertionError, match="on the GPU"):
        ops.paged_sparse_decode_q4(x, pool, pool, i(0)[None], i(1))


def test_stores_and_caches_of_4_bits_say_what_they_hold():
    from sparseattentioninfer_amd.models import PagedKVStore
    from sparseattentioninfer_amd.qwen3 import PagedKVCache
    with pytest.raises(ValueError, match="16 or 4 bits"):
        PagedKVStore(1, 1, 64, 64, device="cpu", bits=8)
    with pytest.raises(ValueError, match="GPU"):
        PagedKVStore(1, 1, 64, 64, device="cpu", bits=4)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        PagedKVStore(1, 1, 64, 64, device="cuda", bits=4, dtype=torch.float32)
    with pytest.raises(ValueError, match="64 or 128"):
        PagedKVStore(1, 1, 96, 64, device="cuda", bits=4)
    with pytest.raises(ValueError, match="16 or 4 bits"):
        PagedKVCache(1, 64, bits=2)
    assert PagedKVStore(1, 1, 64, 64, device="cpu").bits == 16 and PagedKVCache(2, 64, bits=4).layers[1].bits == 4
