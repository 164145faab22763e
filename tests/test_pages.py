"""Paged history, host side: sizes, workspace queries and the refusals of every entry point
before anything is launched."""
import ctypes

import pytest

import paged_reference as ref
from rta import _lib

FAKE = ctypes.c_void_p(0x100000)      # never dereferenced: every call below fails validation first
FAKE_ODD = ctypes.c_void_p(0x100002)
NULL, SHAPE, FORMAT, ALIGN, WS, RANGE = 1, 2, 3, 4, 5, 7


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def book(**change):
    d = dict(fmt=_lib.F16, kv_heads=4, head_dim=128, page=16, layers=2, n_pages=64, max_seqs=8, max_pages=20,
             pool=0x100000, table=0x100000, lengths=0x100000, refs=0x100000)
    d.update(change)
    return ctypes.byref(_lib.Pages(*(d[n] for n, _ in _lib.Pages._fields_)))


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
def test_page_bytes(lib, fmt):
    for hkv, hd, page in ((1, 64, 1), (8, 128, 16), (3, 256, 33), (1024, 256, 65536)):
        assert lib.rta_page_bytes(fmt, hkv, hd, page) == ref.page_bytes(fmt, hkv, hd, page)
    for bad in ((0, 128, 16), (8, 96, 16), (8, 128, 0), (1025, 128, 16), (8, 128, 65537)):
        assert lib.rta_page_bytes(fmt, *bad) == -1
    assert lib.rta_page_bytes(_lib.Q4_K, 8, 128, 16) == -1


def test_workspace_queries(lib):
    assert lib.rta_pages_workspace_bytes(book(), 8) > 0
    assert lib.rta_pages_workspace_bytes(book(), 0) == 0
    assert lib.rta_pages_workspace_bytes(book(fmt=_lib.F32), 8) == 0
    assert lib.rta_paged_attention_workspace_bytes(book(), 16, 4, 4, 1, 0, 0, 0) >= 0
    assert lib.rta_paged_attention_workspace_bytes(book(head_dim=96), 16, 4, 4, 1, 0, 0, 0) == 0


BAD_BOOKS = [(dict(pool=None), NULL), (dict(table=None), NULL), (dict(lengths=None), NULL), (dict(refs=None), NULL),
             (dict(fmt=_lib.Q4_K), FORMAT), (dict(fmt=_lib.F32), FORMAT), (dict(kv_heads=0), SHAPE),
             (dict(page=0), SHAPE), (dict(layers=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(max_seqs=0), SHAPE),
             (dict(max_pages=-1), SHAPE), (dict(head_dim=96), RANGE), (dict(kv_heads=1025), RANGE),
             (dict(n_pages=(1 << 20) + 1), RANGE), (dict(max_pages=1 << 28), RANGE), (dict(pool=0x100008), ALIGN),
             (dict(table=0x100002), ALIGN), (dict(lengths=0x100002), ALIGN), (dict(refs=0x100002), ALIGN)]


@pytest.mark.parametrize("change,code", BAD_BOOKS, ids=lambda x: str(x))
def test_a_bad_descriptor_is_refused_by_every_call(lib, change, code):
    b = book(**change)
    big = 1 << 30
    assert lib.rta_pages_init(b, None) == code
    assert lib.rta_pages_extend(b, FAKE, FAKE, 4, FAKE, big, None) == code
    assert lib.rta_pages_fork(b, FAKE, FAKE, 4, None) == code
    assert lib.rta_pages_free(b, FAKE, FAKE, FAKE, 4, None) == code
    assert lib.rta_pages_compact(b, FAKE, FAKE, big, None) == code
    assert lib.rta_paged_append(b, 0, FAKE, 1 << 20, FAKE, 1 << 20, 4, None, None, 4, None) == code
    assert lib.rta_paged_read(b, 0, 4, None, None, 4, FAKE, 1 << 20, FAKE, 1 << 20, None) == code
    assert lib.rta_paged_attention(b, 0, FAKE, 1 << 20, 4, 1024, None, None, 4, 1, 0, 0, 0, None, FAKE, None, None,
                                   FAKE, big, None) == code
    assert lib.rta_pages_init(None, None) == NULL


def test_list_refusals(lib):
    b, big = book(), 1 << 30
    assert lib.rta_pages_extend(b, FAKE, FAKE, 0, FAKE, big, None) == SHAPE
    assert lib.rta_pages_extend(b, FAKE_ODD, FAKE, 4, FAKE, big, None) == ALIGN
    assert lib.rta_pages_extend(b, FAKE, FAKE_ODD, 4, FAKE, big, None) == ALIGN
    assert lib.rta_pages_extend(b, FAKE, FAKE, 4, None, big, None) == WS
    assert lib.rta_pages_extend(b, FAKE, FAKE, 4, FAKE, 16, None) == WS
    assert lib.rta_pages_fork(b, None, FAKE, 4, None) == NULL
    assert lib.rta_pages_fork(b, FAKE, None, 4, None) == NULL
    assert lib.rta_pages_fork(b, FAKE, FAKE, 0, None) == SHAPE
    assert lib.rta_pages_fork(b, FAKE, FAKE_ODD, 1, None) == ALIGN
    assert lib.rta_pages_free(b, FAKE, FAKE, FAKE, -1, None) == SHAPE
    assert lib.rta_pages_free(b, FAKE, FAKE_ODD, FAKE, 1, None) == ALIGN
    assert lib.rta_pages_compact(b, FAKE, None, big, None) == WS
    assert lib.rta_pages_compact(b, FAKE_ODD, FAKE, big, None) == ALIGN


def test_row_refusals(lib):
    b = book()
    append = lambda layer=0, k=FAKE, ks=512, v=FAKE, vs=512, rows=4, seqs=None, cu=None, n=4: \
        lib.rta_paged_append(b, layer, k, ks, v, vs, rows, seqs, cu, n, None)   # noqa: E731
    assert append(layer=2) == RANGE and append(layer=-1) == RANGE
    assert append(k=None) == NULL and append(v=None) == NULL
    assert append(ks=511) == SHAPE and append(vs=1) == SHAPE
    assert append(rows=0) == SHAPE and append(n=3) == SHAPE and append(n=0, cu=FAKE) == SHAPE
    assert append(k=FAKE_ODD) == ALIGN and append(seqs=FAKE_ODD) == ALIGN and append(cu=FAKE_ODD) == ALIGN
    read = lambda k=FAKE, ks=512, v=FAKE, vs=512, rows=4: \
        lib.rta_paged_read(b, 1, rows, None, None, 4, k, ks, v, vs, None)   # noqa: E731
    assert read(k=None, v=None) == NULL and read(ks=5) == SHAPE and read(rows=5) == SHAPE and read(v=FAKE_ODD) == ALIGN


def test_attention_refusals(lib):
    b = book()

    def attention(layer=0, q=FAKE, stride=2048, rows=4, hq=16, cu=None, n=4, max_rows=1, max_len=0, window=0, sinks=0,
                  gate=None, out=FAKE, m=None, ws=FAKE, size=1 << 40):
        return lib.rta_paged_attention(b, layer, q, stride, rows, hq, None, cu, n, max_rows, max_len, window, sinks,
                                       gate, out, m, None, ws, size, None)
    assert attention(layer=2) == RANGE
    assert attention(q=None) == NULL and attention(out=None) == NULL
    assert attention(hq=18) == SHAPE and attention(hq=0) == SHAPE and attention(stride=2047) == SHAPE
    assert attention(rows=0) == SHAPE and attention(n=5) == SHAPE
    assert attention(max_rows=0) == SHAPE and attention(max_rows=5) == SHAPE and attention(max_len=-1) == SHAPE
    assert attention(window=-1) == RANGE and attention(sinks=-1) == RANGE
    assert attention(q=FAKE_ODD) == ALIGN and attention(gate=FAKE_ODD) == ALIGN and attention(m=FAKE_ODD) == ALIGN
