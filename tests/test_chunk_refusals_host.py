"""Argument checks of the chunk operators' C entries beside those of their main forms: selections without entries, tables
and pools without any, appends at given positions.  Every call returns before any device access."""
import pytest

from sparseattentioninfer_amd import _lib

FAKE = 1 << 12      # a 16-byte aligned stand-in address


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        from sparseattentioninfer_amd import _build
        _build.build(verbose=False)
    return _lib.load()


def _chunk(lib, **o):
    a = dict(kp=FAKE, pages=8, table=FAKE, mb=4, sel=None, rows=0, width=0, off=None, N=4)
    a.update(o)
    return lib.sa_paged_chunk_attn(0, FAKE, 1024, 128, a["kp"], a["kp"], 16384, 8192, 128, a["pages"], a["table"], a["mb"],
                                   a["mb"], FAKE, FAKE, a["sel"], 8, 4, a["rows"], a["width"], a["off"], 8, 4, FAKE, 1024,
                                   128, a["N"], 2, 8, 2, 128, 64, 0.1, 1, None, 0, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(off=FAKE, rows=2, width=4), -6, b"NULL"), (dict(off=FAKE, rows=1, width=0), -2, b"selection"),
    (dict(sel=FAKE, rows=2, width=4), -2, b"selection"), (dict(off=FAKE, rows=2, width=-1), -2, b"selection")])
def test_chunk_selection_refusals(lib, change, code, text):
    assert _chunk(lib, **change) == code and text in lib.sa_last_error()


def _append_at(lib, **o):
    a = dict(dtype=0, k=FAKE, inv=FAKE, pos=FAKE, pos_st=1, N=4, B=2)
    a.update(o)
    return lib.sa_paged_append_at(a["dtype"], None, 0, 0, a["k"], 1024, 128, FAKE, 1024, 128, None, 0, 0, None, None,
                                  a["inv"], a["pos"], a["pos_st"], FAKE, FAKE, 16384, 8192, 128, 8, None, 0, 0, FAKE, 4, 4,
                                  FAKE, FAKE, a["N"], a["B"], 0, 2, 128, 64, 1e-6, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(pos=None), -6, b"positions"), (dict(inv=None), -6, b"inv_freq"), (dict(pos_st=-1), -2, b"stride -1"),
    (dict(dtype=5), -1, b"sa_paged_append_at: dtype 5"), (dict(k=FAKE + 2), -8, b"aligned")])
def test_append_at_refusals(lib, change, code, text):
    assert _append_at(lib, **change) == code and text in lib.sa_last_error()


def test_append_at_nothing_to_do(lib):
    assert _append_at(lib, N=0, k=None, pos=None) == 0 and _append_at(lib, B=0) == 0


@pytest.mark.parametrize("change,code,text", [
    (dict(kp=None), -6, b"NULL"), (dict(table=None), -6, b"NULL"), (dict(kp=None, table=None, mb=0), -6, b"NULL"),
    (dict(kp=None, table=None, pages=0), -6, b"NULL")])
def test_a_table_with_columns_and_a_pool_with_pages_are_needed(lib, change, code, text):
    assert _chunk(lib, **change) == code and text in lib.sa_last_error()
