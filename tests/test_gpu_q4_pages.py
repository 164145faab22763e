"""4-bit pages on the GPU: rows in and out bit by bit against their restatement in fp32, and attention over
them against 64-bit attention of the values they stand for, over the sizes, masks and bad entries of the
other formats' tests."""
import numpy as np
import pytest

import paged_q4_reference as q4
import paged_reference as ref
import test_gpu_paged_attention as base
from rta import _lib, ops
from test_gpu_pages import env, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu
Q4 = q4.Q4_GROUP


@pytest.fixture(autouse=True)
def knows_q4(monkeypatch):
    monkeypatch.setattr(ref, "decode", q4.decode)


def hard_rows(rng, rows, heads, hd):
    """Rows whose groups are of every kind: ordinary, zero, of one sign, tiny, large, at the format's ends."""
    x = rng.standard_normal((rows, heads, hd // 32, 32)).astype(np.float32)
    kind = rng.integers(0, 12, (rows, heads, hd // 32))
    x[kind == 0] = 0.0
    x[kind == 1] = np.abs(x[kind == 1])
    x[kind == 2] = -np.abs(x[kind == 2]) - 1
    x[kind == 3] *= np.float32(1e-6)
    x[kind == 4] *= np.float32(1e-40)
    x[kind == 5] *= np.float32(5000)
    x[kind == 6] = np.round(x[kind == 6])          # halves of steps, ties
    x[kind == 7] += np.float32(31000)              # near the largest range
    x[kind == 8] = np.float32(2.5)
    return x.reshape(rows, heads, hd)


@pytest.mark.parametrize("hkv,hd,page", [(1, 64, 1), (2, 64, 16), (8, 128, 16), (3, 128, 7), (2, 256, 33), (34, 64, 5)])
def test_append_and_read(env, hkv, hd, page):
    torch, _, dev = env
    lens, counts = [37, 5, 0, 64, 1], [37, 3, 0, 20, 1]
    c = filled(env, Q4, hkv, hd, page, lens, layers=2)
    c.pool.random_(0, 256)
    before = c.pool.clone()
    cu = np.concatenate([[0], np.cumsum(counts)])
    rng = np.random.default_rng(5)
    k, v = hard_rows(rng, cu[-1], hkv, hd), hard_rows(rng, cu[-1], hkv, hd)
    v[3, 0, 5], v[4, 0, 40], k[6, 0, 1] = np.nan, np.inf, -np.inf
    k[7, 0, 0], k[7, 0, 1] = 16000.0, -16000.0    # too far apart
    up = lambda x: torch.from_numpy(x.reshape(len(x), -1)).to(dev)   # noqa: E731
    c.append(up(k), up(v), layer=1, cu_rows=ints(torch, cu, dev))
    got = [x.cpu().numpy().reshape(k.shape) for x in c.read(int(cu[-1]), layer=1, cu_rows=ints(torch, cu, dev))]
    for x, y in ((k, got[0]), (v, got[1])):
        code, scale, zero = q4.encode(x)
        want = q4.values(code, scale, zero)
        assert np.array_equal(np.isnan(y), np.isnan(want))
        assert np.array_equal(np.nan_to_num(y), np.nan_to_num(want).astype(np.float32))
    assert np.isnan(got[1][3, 0, :32]).all() and np.isnan(got[1][4, 0, 32:64]).all() and np.isnan(got[0][7, 0, :32]).all()
    assert not np.isnan(got[0][7, :, 32:]).any()
    # the bytes themselves, and nothing else's
    assert torch.equal(c.pool[0], before[0])
    for s, n in enumerate(counts):
        for j in range(n):
            p = lens[s] - n + j
            raw = c.pool[1][int(c.table[s, p // page])].cpu()
            code, word = q4.split(hkv, hd, page, raw)
            for which, x in ((0, k), (1, v)):
                wc, ws, wz = q4.encode(x[cu[s] + j])
                bad = np.isnan(ws)
                assert np.array_equal(code[which, :, p % page], wc)
                want = np.where(bad, q4.NAN_WORD, np.nan_to_num(ws).astype(np.float16).view(np.uint16).astype(np.int64) | wz)
                assert np.array_equal(word[which, :, p % page], want)
    changed = int((c.pool != before).sum())
    assert changed <= cu[-1] * 2 * hkv * (hd // 2 + hd // 16)
    assert ops.device_error() == 0


def test_strides_and_addresses(env):
    torch, _, dev = env
    lens = [50, 9]
    c = filled(env, Q4, 2, 128, 16, lens)
    cu = ints(torch, [0, 50, 59], dev)
    k, v = (torch.randn(59, 256, generator=torch.Generator(device=dev).manual_seed(i), device=dev) for i in (1, 2))
    c.append(k, v, cu_rows=cu)
    want = c.read(59, cu_rows=cu)
    for shift in (1, 2, 3):
        flat = torch.zeros(2, 59 * 261 + 8, device=dev)
        a, b = (flat[i, shift : shift + 59 * (257 + shift)].view(59, 257 + shift)[:, :256] for i in (0, 1))
        a.copy_(k), b.copy_(v)
        c.pool.zero_()
        c.append(a, b, cu_rows=cu)
        a.fill_(7), b.fill_(7)
        got = c.read(59, cu_rows=cu, k=a, v=b)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert ops.device_error() == 0


@pytest.mark.parametrize("hq,hkv,hd,page", [(8, 8, 128, 16), (32, 8, 128, 64), (12, 2, 64, 7), (8, 1, 256, 1),
                                            (16, 1, 64, 32), (34, 2, 128, 24), (9, 3, 256, 100)])
def test_one_row_per_sequence(env, hq, hkv, hd, page):
    base.test_one_row_per_sequence(env, Q4, hq, hkv, hd, page)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (32, 4), (100, 3), (129, 500), (5000, 7), (0, 9)])
@pytest.mark.parametrize("page", [16, 3])
def test_windows_and_first_tokens(env, page, window, sinks):
    base.test_windows_and_first_tokens(env, Q4, page, window, sinks)


@pytest.mark.parametrize("hq,hkv,hd,page,window,sinks", [(8, 2, 128, 16, 0, 0), (32, 8, 128, 64, 40, 4),
                                                         (12, 1, 64, 5, 0, 0), (6, 3, 256, 33, 64, 70),
                                                         (16, 16, 128, 128, 1, 2), (20, 1, 128, 8, 0, 0)])
def test_several_rows_per_sequence(env, hq, hkv, hd, page, window, sinks):
    base.test_several_rows_per_sequence(env, Q4, hq, hkv, hd, page, window, sinks)


@pytest.mark.parametrize("hq,hkv,hd,page,window,sinks", [(8, 2, 128, 16, 0, 0), (32, 4, 128, 64, 40, 4),
                                                         (12, 2, 64, 5, 0, 0), (6, 3, 256, 33, 64, 70),
                                                         (40, 2, 256, 64, 0, 0), (20, 1, 64, 8, 3, 1)])
def test_a_few_rows_per_sequence(env, hq, hkv, hd, page, window, sinks):
    base.test_a_few_rows_per_sequence(env, Q4, hq, hkv, hd, page, window, sinks)


@pytest.mark.parametrize("length", [2048, 60000])
def test_long_histories_keep_fp32_precision(env, length):
    base.test_long_histories_keep_fp32_precision(env, Q4, length)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1, 1], [5, 3], [80, 41]])
def test_tensors_at_any_multiple_of_four_bytes(env, hd, counts):
    base.test_tensors_at_any_multiple_of_four_bytes(env, Q4, hd, counts)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_a_serving_loop(env, window, sinks):
    base.test_a_serving_loop(env, Q4, window, sinks)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,hq,hkv,window", [(1, 4, 2, 0), (4, 4, 1, 0), (8, 4, 1, 5), (90, 8, 2, 0), (90, 8, 2, 24)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(env, hd, rows, hq, hkv, window):
    """Groups of the keys and values of two positions are NaN and inf."""
    torch, _, dev = env
    length, page = 130, 16
    c = filled(env, Q4, hkv, hd, page, [length])
    c.pool.fill_(255)   # what lies past the length is NaN
    base.fill(env, c, [length], 36)
    q = base.rows_of(torch, dev, rows, hq, hd, 37)
    p0 = length - rows
    odd = sorted({p0 + 2, p0 + rows // 2}) if rows > 1 else [p0 - 60, p0 - 3]
    words = c.pool[0].view(torch.int16)
    for p in odd:
        for which in (0, 1):
            at = hkv * page * hd // 2 + (which * hkv * page + p % page) * (hd // 32)
            n = int(c.table[0, p // page])
            words[n, at], words[n, at + hd // 32 - 1] = q4.NAN_WORD, 0x7C00 + 3
    if rows == 1:
        # one row: in sight, and behind the window
        out, m, z = c.attention(q, max_len=length)
        assert ops.device_error() & _lib.DEVERR_DETECTOR
        clean = c.attention(q, max_len=length, window=3)
        ref.check_rows(clean, base.want_rows(c, q, [(0, 0, 1)], window=3))
        assert ops.device_error() == 0
        return
    out, m, z = c.attention(q, cu_rows=ints(torch, [0, rows], dev), max_rows=rows, window=window)
    assert ops.device_error() & _lib.DEVERR_DETECTOR
    k, v, held = ref.dense(c, 0, 0)
    k, v = (np.nan_to_num(x, nan=1.0, posinf=1.0, neginf=1.0) for x in (k, v))
    clean = 0
    for r in range(rows):
        t = p0 + r
        sees = any(p <= t and (not window or p > t - window) for p in odd)
        clean += not sees
        heads = slice(hq // hkv if sees else 0, hq)   # kv head 0 holds them
        want = ref.attend(q[r].cpu().double().numpy(), k, v, held, t, window)
        if heads.start < hq:
            ref.check_rows([x[r : r + 1, heads] for x in (out, m, z)], [tuple(w[heads] for w in want)], r)
    assert clean >= 2


def test_large_scales_and_tiny_values(env):
    torch, _, dev = env
    lens = [300, 300]
    for scale in (2e-4, 900.0):
        c = filled(env, Q4, 2, 128, 16, lens)
        gen = torch.Generator(device=dev).manual_seed(19)
        k, v = (scale * torch.randn(600, 256, generator=gen, device=dev) for _ in range(2))
        c.append(k, v, cu_rows=ints(torch, [0, 300, 600], dev))
        q = base.rows_of(torch, dev, 2, 8, 128, 20) / scale
        got = c.attention(q, max_len=300)
        ref.check_rows(got, base.want_rows(c, q, [(s, s, 1) for s in range(2)]), scale)
        several = c.attention(q, seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, 2], dev))
        ref.check_rows(several, base.want_rows(c, q, [(0, 0, 2)]), scale)
    assert ops.device_error() == 0


def test_bad_entries_read_as_nothing(env):
    torch, _, dev = env
    lens = [40, 500, 10, 100]
    c = filled(env, Q4, 2, 64, 16, lens)
    base.fill(env, c, lens, 14)
    q = base.rows_of(torch, dev, 4, 4, 64, 15)
    c.table[3, 2], c.table[3, 4] = -1, 10**8
    out, m, z = c.attention(q, seqs=ints(torch, [9, 1, 2, 3], dev), max_len=400)
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert not out[:2].any() and not z[:2].any() and (m[:2] == -np.inf).all()
    ref.check_rows([t[2:] for t in (out, m, z)], base.want_rows(c, q, [(2, 2, 1), (3, 3, 1)], missing_ok=True))
    q = base.rows_of(torch, dev, 70, 4, 64, 16)
    got = c.attention(q, seqs=ints(torch, [3], dev), cu_rows=ints(torch, [0, 70], dev), max_rows=70)
    assert ops.device_error() == _lib.DEVERR_PAGES
    ref.check_rows(got, base.want_rows(c, q, [(3, 0, 70)], missing_ok=True))


def test_pages_move_whole(env):
    """Copies on write and compaction carry codes and words alike."""
    torch, pages, dev = env
    c = pages.PagedCache(Q4, 3, 64, 5, n_pages=40, max_seqs=6, max_pages=10, layers=2)
    c.pool.fill_(255)
    c.extend(ints(torch, [0, 1], dev), ints(torch, [13, 22], dev))
    cu = ints(torch, [0, 13, 35], dev)
    x = torch.randn(35, 192, generator=torch.Generator(device=dev).manual_seed(3), device=dev)
    for layer in (0, 1):
        c.append(x, 2 * x, layer=layer, seqs=ints(torch, [0, 1], dev), cu_rows=cu)
    want = c.read(35, layer=1, seqs=ints(torch, [0, 1], dev), cu_rows=cu)
    c.fork(ints(torch, [0], dev), ints(torch, [4], dev))
    c.extend(ints(torch, [4], dev))
    c.free(ints(torch, [1], dev))
    c.compact()
    assert c.lengths.tolist() == [13, 0, 0, 0, 14, 0]
    got = c.read(13, layer=1, seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, 13], dev))
    assert all(torch.equal(a, b[:13]) for a, b in zip(got, want))
    k, v, _ = ref.dense(c, 1, 4)
    assert np.array_equal(k[:13].reshape(13, -1), want[0][:13].cpu().double().numpy())
    assert np.array_equal(v[:13].reshape(13, -1), want[1][:13].cpu().double().numpy())
    assert ops.device_error() == 0


def test_a_captured_step_replays(env):
    torch, _, dev = env
    eager, graph = base.Loop(env, Q4, 0, 0, 26), base.Loop(env, Q4, 0, 0, 26)
    for x in (eager, graph):
        x.prompt([40, 7, 16])
        x.new_rows()
        x.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graph.step()
    for i in range(5):
        for x in (eager, graph):
            x.new_rows()
        eager.step()
        g.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(eager.out[layer], graph.out[layer]), (i, layer)
    assert ops.device_error() == 0


def test_pools_past_four_gigabytes(env):
    torch, pages, dev = env
    page = 1024
    pb = pages.page_bytes(Q4, 4, 128, page)
    n_pages = (5 << 30) // pb
    pool = torch.empty(1, n_pages, pb, dtype=torch.uint8, device=dev)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    table = torch.full((1, 4), -1, dtype=torch.int32, device=dev)
    names = [n_pages - 1, n_pages - 3, 0]
    table[0, :3] = ints(torch, names, dev)
    refs[names] = 1
    lens = [2 * page + 77]
    c = pages.PagedCache(Q4, 4, 128, page, pool=pool, table=table, lengths=ints(torch, lens, dev), refs=refs)
    base.fill(env, c, lens, 21)
    for hq, rows in ((8, 1), (24, 1), (8, 3), (8, 40)):   # each of the kernels
        q = base.rows_of(torch, dev, rows, hq, 128, 22)
        got = c.attention(q, cu_rows=ints(torch, [0, rows], dev), max_rows=rows)
        ref.check_rows(got, base.want_rows(c, q, [(0, 0, rows)]))
    assert ops.device_error() == 0


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (3, 1), (10, 2)])
def test_lengths_around_the_cut(env, hd, hq, hkv):
    """Calls of up to 512 positions in one piece, longer ones in chunks; tiles and chunks that end early."""
    torch, _, dev = env
    lens = [511, 512, 513, 31, 33, 127, 640, 1025]
    c = filled(env, Q4, hkv, hd, 24, lens)
    base.fill(env, c, lens, 41)
    q = base.rows_of(torch, dev, len(lens), hq, hd, 42)
    want = base.want_rows(c, q, [(s, s, 1) for s in range(len(lens))])
    ref.check_rows(c.attention(q, max_len=1025), want)
    few = [1, 3, 4, 5]
    ref.check_rows(c.attention(q[few].contiguous(), seqs=ints(torch, few, dev), max_len=512), [want[s] for s in few])
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW, Q4])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (6, 2), (12, 1)])
def test_what_lies_in_other_pages_does_not_matter_where_one_is_missing(env, fmt, hd, hq, hkv):
    """Positions without a page beside positions with one, page 0 free and full of NaN: the rows, and the score
    of every other position, are those of the positions that have a page."""
    torch, pages, dev = env
    page, lens = 16, [100, 33, 700]
    c = pages.PagedCache(fmt, hkv, hd, page, n_pages=60, max_seqs=3, max_pages=50)
    c.pool.fill_(255)   # NaN in every format's elements or scales
    at = 1
    for s, n in enumerate(lens):
        held = -(-n // page)
        c.table[s, :held] = torch.arange(at, at + held, dtype=torch.int32, device=dev)
        c.refs[at : at + held] = 1
        at += held
    c.lengths[:] = ints(torch, lens, dev)
    base.fill(env, c, lens, 43)
    # pages behind a window given back (of either half of a tile of 32, and whole tiles), an entry past the pool
    c.free(ints(torch, [0, 2], dev), ints(torch, [16, 64], dev), ints(torch, [48, 144], dev))
    assert ops.device_error() == 0
    c.table[0, 4], c.table[1, 1], c.table[2, 20] = 10**8, -1, -(2**31)
    assert int(c.refs[0]) == 0
    q = base.rows_of(torch, dev, 3, hq, hd, 44)
    got = c.attention(q, max_len=700)
    assert ops.device_error() == _lib.DEVERR_PAGES
    ref.check_rows(got, base.want_rows(c, q, [(s, s, 1) for s in range(3)], missing_ok=True))
    for rows in (2, 90):   # few rows and many
        q = base.rows_of(torch, dev, rows, hq, hd, 45)
        for s in (0, 2):
            got = c.attention(q, seqs=ints(torch, [s], dev), cu_rows=ints(torch, [0, rows], dev), max_rows=rows)
            assert ops.device_error() == _lib.DEVERR_PAGES
            ref.check_rows(got, base.want_rows(c, q, [(s, 0, rows)], missing_ok=True), (rows, s))
