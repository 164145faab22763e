"""4-bit pages, host side: sizes, and that the restatement that the GPU tests compare with holds what the
format promises (values within half a step, scales of six bits, products exact in binary16)."""
import ctypes

import numpy as np
import pytest

import paged_q4_reference as q4
from rta import _lib
from test_pages import book


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_page_bytes(lib):
    assert _lib.Q4_GROUP == q4.Q4_GROUP
    for hkv, hd, page in ((1, 64, 1), (8, 128, 16), (3, 256, 33), (1024, 256, 65536)):
        assert lib.rta_page_bytes(_lib.Q4_GROUP, hkv, hd, page) == q4.page_bytes(hkv, hd, page)
    for bad in ((0, 128, 16), (8, 96, 16), (8, 128, 0), (1025, 128, 16), (8, 128, 65537)):
        assert lib.rta_page_bytes(_lib.Q4_GROUP, *bad) == -1
    assert lib.rta_page_bytes(_lib.Q4_GROUP | _lib.TILED, 8, 128, 16) == -1
    assert lib.rta_pages_workspace_bytes(book(fmt=_lib.Q4_GROUP), 8) > 0
    assert lib.rta_pages_init(book(fmt=_lib.Q4_GROUP, pool=0x100008), None) == 4
    assert isinstance(ctypes.sizeof(_lib.Pages), int)


@pytest.mark.parametrize("scale", [1e-30, 1e-5, 1.0, 300.0, 4000.0])
def test_the_format_keeps_its_promises(scale):
    rng = np.random.default_rng(1)
    x = (scale * rng.standard_normal((500, 64))).astype(np.float32)
    x[:100] += np.float32(2 * scale)
    x[100:200] = np.abs(x[100:200])
    code, d, z = q4.encode(x)
    assert code.min() >= 0 and code.max() <= 15 and z.min() >= 0 and z.max() <= 15 and np.isfinite(d).all()
    half = d.astype(np.float16)
    assert np.array_equal(half.astype(np.float64), d) and not (half.view(np.uint16) & 31).any()
    # within half a step (code 15's end: the step is rounded up, so the range fits up to fp32's own rounding)
    off = np.abs(q4.values(code, d, z) - x).reshape(500, 2, 32)
    assert np.all(off <= d[..., None] * (0.5 + 2.0**-19))
    # the scale is at most 1/32 and 2^-19 above the range's fifteenth
    g = x.reshape(500, 2, 32).astype(np.float64)
    f = (np.maximum(g.max(-1), 0) - np.minimum(g.min(-1), 0)) / 15
    assert np.all(d <= f * (1 + 2.0**-5 + 2.0**-22) + 2.0**-19) and np.all(d >= f * (1 - 2.0**-22))


def test_every_value_is_exact_in_binary16():
    """scale * (code - zero) and both terms of scale * (16 + code) - scale * (16 + zero), for every word."""
    words = np.arange(1 << 16, dtype=np.uint32)
    d = (words & 0xFFE0).astype(np.uint16).view(np.float16).astype(np.float64)
    d = np.unique(d[np.isfinite(d) & (np.abs(d) <= q4.MOST)])
    for n in range(-15, 32):
        p = d * n
        assert np.array_equal(p.astype(np.float16).astype(np.float64), p)


def test_codes_lie_where_the_layout_says():
    for hd in (64, 128, 256):
        byte, shift = q4.places(hd)
        assert sorted(zip(byte.tolist(), shift.tolist())) == [(b, s) for b in range(hd // 2) for s in (0, 4)]
