"""Rotary positions, host side: the frequencies of every scaling and the refusals."""
import ctypes

import numpy as np
import pytest

import rotary_reference as ref
from rta import _lib, rotary
from test_pages import FAKE, FAKE_ODD, book

NULL, SHAPE, ALIGN, RANGE = 1, 2, 4, 7
FAKE_4 = ctypes.c_void_p(0x100004)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def turn(layout=0, head_dim=128, dims=128, amplitude=1.0, turns=0x100000):
    return ctypes.byref(_lib.Rotary(layout, head_dim, dims, amplitude, turns))


@pytest.mark.parametrize("dims", [2, 4, 6, 64, 128, 250])
@pytest.mark.parametrize("theta", [10.0, 1e4, 5e6])
@pytest.mark.parametrize("scaling,how", [("plain", {}), ("linear", dict(factor=4.0)), ("base", dict(factor=8.0)),
                                         ("ramp", dict(factor=16.0, original=4096)),
                                         ("ramp", dict(factor=1.0, original=2, low=0.5, high=0.6)),
                                         ("ramp", dict(factor=40.0, original=32768, low=1.0, high=64.0)),
                                         ("bands", dict(factor=8.0, original=8192, low=1.0, high=4.0))])
def test_turns(dims, theta, scaling, how):
    got, amplitude = rotary.turns(dims, theta, scaling, **how)
    want = ref.turns(dims, theta, scaling, **how)
    # exponentials of up to 20 logarithms, each with a few roundings of 2^-53
    assert np.all(np.abs(got.numpy() - want) <= 2.0**-46 * want)
    assert abs(amplitude - (0.1 * np.log(how["factor"]) + 1 if scaling == "ramp" and how["factor"] > 1 else 1.0)) < 1e-15


def test_turns_refusals(lib):
    room = (ctypes.c_double * 64)()
    turns = lambda dims=128, theta=1e6, scaling=3, factor=2.0, original=100.0, low=1.0, high=32.0, out=room: \
        lib.rta_rotary_turns(dims, theta, scaling, factor, original, low, high, out, None)   # noqa: E731
    assert turns() == 0
    assert turns(out=None) == NULL and turns(dims=0) == SHAPE and turns(dims=7) == SHAPE and turns(dims=-2) == SHAPE
    nan, inf = float("nan"), float("inf")
    for change in (dict(theta=0.0), dict(theta=-1.0), dict(theta=nan), dict(theta=inf), dict(theta=1.0), dict(scaling=5),
                   dict(scaling=-1), dict(factor=0.0), dict(factor=nan), dict(factor=inf), dict(original=0.0),
                   dict(original=nan), dict(low=0.0), dict(low=32.0), dict(high=inf), dict(high=nan), dict(low=nan)):
        assert turns(**change) == RANGE, change
    assert turns(theta=0.5, scaling=0, factor=nan, original=nan) == 0   # what plain frequencies do not read
    with pytest.raises(ValueError):
        rotary.turns(128, scaling="other")
    with pytest.raises(ValueError):
        rotary.Rotary(128, 130)
    with pytest.raises(ValueError):
        rotary.Rotary(128, layout="thirds")


BAD_TURNS = [(dict(turns=None), NULL), (dict(head_dim=0), SHAPE), (dict(dims=0), SHAPE), (dict(dims=5), SHAPE),
             (dict(dims=130), SHAPE), (dict(layout=2), RANGE), (dict(layout=-1), RANGE), (dict(head_dim=514), RANGE),
             (dict(amplitude=float("nan")), RANGE), (dict(amplitude=float("inf")), RANGE), (dict(turns=0x100004), ALIGN)]


@pytest.mark.parametrize("change,code", BAD_TURNS, ids=lambda x: str(x))
def test_a_bad_rotation_is_refused_by_every_call(lib, change, code):
    r = turn(**change)
    assert lib.rta_rotate(r, FAKE, 1 << 20, 4, 4, FAKE, FAKE, 1 << 20, None) == code
    assert lib.rta_paged_append_rotary(book(), 0, r, FAKE, 512, FAKE, 512, None, 0, 0, None, 0, 4, None, None, 4,
                                       None) == code
    assert lib.rta_rotate(None, FAKE, 1 << 20, 4, 4, FAKE, FAKE, 1 << 20, None) == NULL


def test_rotate_refusals(lib):
    r = turn()
    call = lambda x=FAKE, xs=512, rows=4, heads=4, p=FAKE, y=FAKE, ys=512: \
        lib.rta_rotate(r, x, xs, rows, heads, p, y, ys, None)   # noqa: E731
    assert call(x=None) == NULL and call(p=None) == NULL and call(y=None) == NULL
    assert call(xs=511) == SHAPE and call(ys=511) == SHAPE and call(rows=0) == SHAPE and call(heads=-1) == SHAPE
    assert call(rows=1 << 24) == RANGE and call(heads=65536, xs=1 << 40, ys=1 << 40) == RANGE
    assert call(x=FAKE_ODD) == ALIGN and call(y=FAKE_ODD) == ALIGN and call(p=FAKE_4) == ALIGN
    assert call(xs=600) == RANGE   # in place at another stride


def test_append_refusals(lib):
    r, b = turn(), book()
    call = lambda b=b, r=r, layer=0, k=FAKE, ks=512, v=FAKE, vs=512, q=FAKE_4, qs=1024, hq=8, o=FAKE, os=1024, rows=4, \
        seqs=None, cu=None, n=4: lib.rta_paged_append_rotary(b, layer, r, k, ks, v, vs, q, qs, hq, o, os, rows, seqs,
                                                             cu, n, None)   # noqa: E731
    assert call(layer=2) == RANGE and call(layer=-1) == RANGE and call(b=None) == NULL and call(r=None) == NULL
    assert call(b=book(fmt=_lib.Q4_K)) == 3
    assert call(k=None) == NULL and call(v=None) == NULL and call(q=None) == NULL and call(o=None) == NULL
    assert call(ks=511) == SHAPE and call(vs=0) == SHAPE and call(qs=1023) == SHAPE and call(os=1) == SHAPE
    assert call(hq=0) == SHAPE and call(hq=-4) == SHAPE and call(r=turn(head_dim=64, dims=64)) == SHAPE
    assert call(rows=0) == SHAPE and call(n=3) == SHAPE and call(n=0, cu=FAKE) == SHAPE and call(rows=1 << 24, n=1 << 24) == RANGE
    assert call(hq=65536, qs=1 << 40, os=1 << 40) == RANGE and call(q=FAKE, o=FAKE, qs=2000) == RANGE
    assert call(k=FAKE_ODD) == ALIGN and call(v=FAKE_ODD) == ALIGN and call(q=FAKE_ODD) == ALIGN and call(o=FAKE_ODD) == ALIGN
    assert call(seqs=FAKE_ODD) == ALIGN and call(cu=FAKE_ODD) == ALIGN
