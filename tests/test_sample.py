"""The draw from logits, host side: its workspace and its refusals."""
import ctypes

import pytest

from rta import _lib

FAKE, FAKE_ODD = ctypes.c_void_p(0x100000), ctypes.c_void_p(0x100002)
NULL, SHAPE, ALIGN, WS, RANGE = 1, 2, 4, 5, 7


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_workspace(lib):
    need = lib.rta_sample_workspace_bytes
    assert need(1, 1) > 0 and need(1, 8192) == need(1, 1) and need(1, 8193) == 2 * need(1, 1) and need(7, 8192) == 7 * need(1, 1)
    assert need(1, 1 << 22) == 512 * need(1, 1)
    assert need(0, 10) == 0 and need(1, 0) == 0 and need(1, (1 << 22) + 1) == 0 and need(-1, 5) == 0


def test_refusals(lib):
    need = lib.rta_sample_workspace_bytes(4, 1000)

    def call(x=FAKE, stride=1000, rows=4, vocab=1000, t=None, k=None, p=None, m=None, u=FAKE, ids=FAKE, probs=None, ws=FAKE, size=16):
        return lib.rta_sample(x, stride, rows, vocab, t, k, p, m, u, ids, probs, ws, size, None)
    assert call(x=None) == NULL and call(u=None) == NULL and call(ids=None) == NULL
    assert call(rows=0) == SHAPE and call(vocab=0) == SHAPE and call(stride=999) == SHAPE and call(rows=-3) == SHAPE
    assert call(vocab=(1 << 22) + 1, stride=1 << 25) == RANGE and call(rows=1 << 22) == RANGE
    assert call(rows=1 << 13, vocab=1 << 22, stride=1 << 22) == RANGE
    for name in ("x", "t", "k", "p", "m", "u", "ids", "probs"):
        assert call(**{name: FAKE_ODD}) == ALIGN, name
    assert call() == WS and call(size=need - 1) == WS and call(ws=None, size=need) == WS
    assert call(ws=ctypes.c_void_p(0x100008), size=need) == WS
