"""Attention over the paged history at the ends of its ranges: value scales, values and scores far
apart or near the end of fp32, and what rows may not see, against 64-bit results.

The tolerance of a head is `bound` of paged_reference.attend (the relative error of every weight)
times sum p |v| of the head's worst dim, doubled: errors of the terms add up to no more."""
import numpy as np
import pytest

import paged_reference as ref
from rta import _lib, ops
from test_gpu_paged_attention import rows_of
from test_gpu_pages import env, ints  # noqa: F401

pytestmark = pytest.mark.gpu

ALL = [ref.F16, ref.BF16, ref.Q8_ROW]


def holding(env, fmt, hkv, hd, page, k, v):
    """A cache whose only sequence holds k and v [length, hkv * hd]."""
    torch, pages, dev = env
    n = -(-len(k) // page)
    c = pages.PagedCache(fmt, hkv, hd, page, n_pages=n + 2, max_seqs=2, max_pages=n + 1)
    c.pool.fill_(255)
    c.extend(ints(torch, [0], dev), ints(torch, [len(k)], dev))
    c.append(k.to(dev), v.to(dev), seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, len(k)], dev))
    return c


def newest(env, c, q, **how):
    """Attention of the rows q as the newest positions of sequence 0."""
    torch, _, dev = env
    return c.attention(q, seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, len(q)], dev), max_rows=len(q), **how)


def check_terms(c, q, got, rows=None, window=0, sinks=0):
    out, m, z = (t.cpu().double().numpy() for t in got)
    k, v, held = ref.dense(c, 0, 0)
    x = q.cpu().double().numpy()
    for r in range(len(q)) if rows is None else rows:
        t = len(k) - len(q) + r
        wo, wm, wz, bound, _ = ref.attend(x[r], k, v, held, t, window, sinks)
        terms = ref.attend(x[r], k, np.abs(v), held, t, window, sinks)[0]
        err = np.abs(out[r] - wo).max(1)
        assert np.all(err <= 2 * bound * terms.max(1)), (r, float((err / terms.max(1)).max()), float(bound.max()))
        assert np.all(np.abs(m[r] - wm) <= bound) and np.all(np.abs(z[r] - wz) <= (bound + 2.0**-21) * wz), r


def normal(env, seed, *shape):
    torch = env[0]
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------ value scales far apart ----
@pytest.mark.parametrize("spread", [12, 30, 45, 100])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,hq,hkv,window", [(4, 4, 1, 0), (8, 4, 1, 5), (90, 8, 2, 0), (90, 8, 2, 24)])
def test_a_large_value_scale_out_of_sight(env, spread, hd, rows, hq, hkv, window):
    """A value 2^spread times the others at a position in the middle of the new rows: rows before it,
    and rows whose window has passed it, keep their precision; the others get it as it is."""
    length = 130
    k, v = normal(env, 1, length, hkv * hd), normal(env, 2, length, hkv * hd)
    v[length - rows + rows // 2] *= 2.0**spread
    c = holding(env, ref.Q8_ROW, hkv, hd, 16, k, v)
    q = rows_of(env[0], env[2], rows, hq, hd, 3)
    check_terms(c, q, newest(env, c, q, window=window), window=window)
    assert ops.device_error() == 0


@pytest.mark.parametrize("spread", [8, 16, 24, 40, 90])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 2, 5, 40])
def test_a_large_value_scale_of_no_weight(env, spread, hd, rows):
    """The largest value scale at a visible position whose weight is e^-90 of the largest, early and
    late in a history of several tiles and chunks: the other positions' sum stays whole."""
    torch, _, dev = env
    length = 700
    q = rows_of(torch, dev, rows, 4, hd, 4, 0.01) + 0.5
    k, v = 0.1 * normal(env, 5, length, hd), normal(env, 6, length, hd)
    for p in (9, 400):
        k[p] = -90 * hd**0.5 / (0.5 * hd)   # q . k / sqrt(hd) = -90 for q = 0.5 in every dim
        v[p] *= 2.0**spread
    c = holding(env, ref.Q8_ROW, 1, hd, 16, k, v)
    check_terms(c, q, newest(env, c, q))
    assert ops.device_error() == 0


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_value_scales_of_every_size(env, hd, rows):
    """Scales spread log-normally over some 2^+-30, and some heads' values zero."""
    length = 500
    k, v = normal(env, 7, length, hd), normal(env, 8, length, hd)
    v *= (8 * normal(env, 9, length, 1)).exp()
    v[::7] = 0.0
    c = holding(env, ref.Q8_ROW, 1, hd, 8, k, v)
    q = rows_of(env[0], env[2], rows, 4, hd, 10, 4.0)
    check_terms(c, q, newest(env, c, q))
    assert ops.device_error() == 0


# ------------------------------------------------------------------ values near the end ----
@pytest.mark.parametrize("fmt", [ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("size", [1e30, 1e36, 3e38])
def test_values_near_the_end_of_fp32(env, fmt, hd, rows, size):
    """A mean of finite values is finite: 1500 positions of about the same weight, all of one sign,
    whose plain sum would overflow."""
    length = 1500
    k = normal(env, 11, length, hd)
    v = size * (1 - 0.5 * normal(env, 12, length, hd).abs().clamp(max=1))
    c = holding(env, fmt, 1, hd, 64, k, v)
    q = rows_of(env[0], env[2], rows, 4, hd, 13, 0.1)
    check_terms(c, q, newest(env, c, q))
    assert ops.device_error() == 0


# ------------------------------------------------------------------ what a row may not see ----
@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_a_missing_page_is_not_scored(env, fmt, hd, rows):
    """Where a page is missing nothing is read for it: infinite keys in page 0 (another sequence's)
    report nothing."""
    torch, pages, dev = env
    length = 100
    c = pages.PagedCache(fmt, 1, hd, 16, n_pages=20, max_seqs=2, max_pages=8)
    c.extend(ints(torch, [1, 0], dev), ints(torch, [16, length], dev))
    assert c.table[1, 0].item() == 0
    k, v = normal(env, 14, length + 16, hd), normal(env, 15, length + 16, hd)
    c.append(k.to(dev), v.to(dev), seqs=ints(torch, [1, 0], dev), cu_rows=ints(torch, [0, 16, 16 + length], dev))
    if fmt == ref.Q8_ROW:
        c.pool[0, 0, : 16 * hd] = 0
        c.pool[0, 0, : 16 * hd].view(16, hd)[:, 0] = 1
        c.pool[0, 0, 2 * 16 * hd :][: 16 * 4] = torch.full((16,), 3e38, device=dev).view(torch.uint8)
    else:
        kv = c.pool[0, 0].view(torch.float16 if fmt == ref.F16 else torch.bfloat16)
        kv[: 16 * hd] = 0
        kv[: 16 * hd].view(16, hd)[:, 0] = float("inf")
    c.table[0, 2] = -1
    q = rows_of(torch, dev, rows, 4, hd, 16)
    q[:, :, 0] = -8.0    # a score of -inf wherever page 0 is looked at
    got = newest(env, c, q)
    assert ops.device_error() == _lib.DEVERR_PAGES
    k, v, held = ref.dense(c, 0, 0, missing_ok=True)
    want = [ref.attend(q[r].cpu().double().numpy(), np.where(held[:, None, None], k, 0), v, held, length - rows + r)
            for r in range(rows)]
    ref.check_rows(got, want)


@pytest.mark.parametrize("fmt", [ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [4, 40])
def test_a_score_out_of_sight_reports_nothing(env, fmt, hd, rows):
    """A later position's key would overflow the scores of rows before it (and only theirs)."""
    length = 90
    k, v = normal(env, 17, length, hd), normal(env, 18, length, hd)
    p = length - rows // 2
    k[p] = 0.0
    k[p, 0] = 3e38
    c = holding(env, fmt, 1, hd, 16, k, v)
    q = rows_of(env[0], env[2], rows, 4, hd, 19)
    q[: rows - rows // 2, :, 0] = -100.0
    q[rows - rows // 2 :, :, 0] = 0.0
    got = newest(env, c, q)
    assert ops.device_error() == 0
    check_terms(c, q, got, rows=range(rows - rows // 2))
    assert all(bool(t.isfinite().all()) for t in got)


@pytest.mark.parametrize("fmt", [ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,length", [(1, 64), (1, 70), (4, 70), (40, 70), (40, 300)])
def test_a_score_of_minus_infinity_in_sight_is_reported(env, fmt, hd, rows, length):
    """In the newest position (seen by the last row alone) and in the oldest (seen by all).  (A binary16
    key is below 2^16 and a query is taken by its head's power of two, so there is no such product.)"""
    torch = env[0]
    q = rows_of(torch, env[2], rows, 4, hd, 24)
    q[:, :, 0] = -1e10
    for p in (length - 1, 0):
        k, v = normal(env, 25, length, hd), normal(env, 26, length, hd)
        k[:, 0] = 0.0
        k[p, 0] = 3e38
        c = holding(env, fmt, 1, hd, 16, k, v)
        out = newest(env, c, q)[0]
        assert ops.device_error() == _lib.DEVERR_DETECTOR
        if p:   # rows that do not see it keep theirs
            assert bool(out[: rows - 1].isfinite().all())


# ------------------------------------------------------------------ large scores ----
@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e8, 1e9, 1e12, 1e20])
def test_scores_of_any_finite_size(env, fmt, hd, rows, size):
    """Far apart as they are, one position takes all: out is its value, z is 1.  A score's error is
    below sqrt(hd) roundings of 2^-22 of sum |q k|, so heads whose two largest are further apart than
    2^-14 of that are told apart."""
    length = 400
    k, v = normal(env, 20, length, hd), normal(env, 21, length, hd)
    c = holding(env, fmt, 1, hd, 16, k, v)
    q = rows_of(env[0], env[2], rows, 4, hd, 22, size)
    out, m, z = (t.cpu().double().numpy() for t in newest(env, c, q))
    assert ops.device_error() == 0
    k, v, _ = ref.dense(c, 0, 0)
    told = 0
    for r in range(rows):
        n = length - rows + r + 1
        for h in range(4):
            x = q[r, h].cpu().double().numpy()
            s = k[:n, 0] @ x / hd**0.5
            a, b = np.argsort(s)[-2:][::-1]
            most = (np.abs(k[:n, 0]) @ np.abs(x)).max() / hd**0.5
            if s[a] - s[b] <= 2.0**-14 * most + 30:
                continue
            told += 1
            assert np.abs(out[r, h] - v[a, 0]).max() <= 2.0**-20 * np.abs(v[a, 0]).max(), (r, h)
            assert abs(m[r, h] - s[a]) <= hd**0.5 * 2.0**-22 * most and abs(z[r, h] - 1) <= 2.0**-20, (r, h, z[r, h])
    assert told >= rows


# ------------------------------------------------------------------ small values ----
@pytest.mark.parametrize("fmt", [ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("size", [1e-20, 2.0**-98])
def test_values_near_zero(env, fmt, hd, rows, size):
    length = 700
    k, v = normal(env, 27, length, hd), size * normal(env, 28, length, hd)
    c = holding(env, fmt, 1, hd, 64, k, v)
    q = rows_of(env[0], env[2], rows, 4, hd, 29)
    check_terms(c, q, newest(env, c, q))
    assert ops.device_error() == 0
