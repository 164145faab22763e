"""Paged history on the GPU: the book against its plain restatement, call by call and over random
sequences of calls, page copies byte for byte, rows in and out against their roundings."""
import numpy as np
import pytest

import paged_reference as ref
from rta import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from rta import pages
    ops.device_error(clear=True)
    return torch, pages, torch.device("cuda:0")


def ints(torch, v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


def make(env, page=16, n_pages=64, max_seqs=12, max_pages=10, fmt=ref.F16, hkv=2, hd=64, layers=2):
    torch, pages, dev = env
    c = pages.PagedCache(fmt, hkv, hd, page, n_pages=n_pages, max_seqs=max_seqs, max_pages=max_pages, layers=layers)
    c.pool.random_(0, 256)
    return c, ref.Book(page, n_pages, max_seqs, max_pages)


def test_reset_empties_the_book(env):
    c, b = make(env)
    b.check(c)


def test_extend_takes_the_lowest_free_pages_in_list_order(env):
    torch, _, dev = env
    c, b = make(env)
    seqs, add = [3, 0, 7], [17, 0, 40]
    c.extend(ints(torch, seqs, dev), ints(torch, add, dev))
    b.extend(seqs, add)
    b.check(c)
    c.extend(n=4)   # the first four sequences, one position each
    b.extend([0, 1, 2, 3], [1] * 4)
    b.check(c)
    assert ops.device_error() == 0


def test_extend_refuses_bad_entries_and_leaves_the_rest(env):
    torch, _, dev = env
    c, b = make(env, max_pages=4)
    seqs, add = [1, -1, 12, 1, 2, 5, 6], [5, 5, 5, 9, -3, 65, 64]
    c.extend(ints(torch, seqs, dev), ints(torch, add, dev))
    b.extend(seqs, add)
    b.check(c)
    assert b.lengths[1] == 5 and b.lengths[5] == 0 and b.lengths[6] == 64
    assert ops.device_error() == _lib.DEVERR_PAGES


def test_extend_stops_where_the_pages_run_out(env):
    torch, _, dev = env
    c, b = make(env, n_pages=5)
    seqs, add = [0, 1, 2, 3], [33, 40, 1, 0]   # 3 pages, 3 that do not fit, then nothing
    c.extend(ints(torch, seqs, dev), ints(torch, add, dev))
    b.extend(seqs, add)
    assert b.lengths[:4] == [33, 0, 0, 0]
    b.check(c)
    assert ops.device_error() == _lib.DEVERR_PAGES


@pytest.mark.parametrize("page", [1, 5, 16])
def test_fork_copies_on_write(env, page):
    torch, _, dev = env
    c, b = make(env, page=page, n_pages=200, max_pages=40)
    c.extend(ints(torch, [0, 1], dev), ints(torch, [37, 32], dev))
    b.extend([0, 1], [37, 32])
    src, dst = [0, 0, 1, 0], [4, 5, 6, 9]
    c.fork(ints(torch, src, dev), ints(torch, dst, dev))
    b.fork(src, dst)
    b.check(c)
    before = c.pool.clone()
    every = [4, 5, 6, 9, 0, 1]
    c.extend(ints(torch, every, dev))
    pairs = b.extend(every, [1] * 6)
    b.check(c)
    assert ops.device_error() == 0
    after = before.clone()
    for a, z in pairs:
        after[:, z] = before[:, a]
    assert torch.equal(c.pool, after)
    # one sharer alone copies, the others keep the page
    c.fork(ints(torch, [0], dev), ints(torch, [11], dev))
    b.fork([0], [11])
    c.extend(ints(torch, [11], dev))
    b.extend([11], [1])
    b.check(c)


def test_fork_refusals(env):
    torch, _, dev = env
    c, b = make(env)
    c.extend(ints(torch, [0, 1, 2], dev), ints(torch, [20, 5, 0], dev))
    b.extend([0, 1, 2], [20, 5, 0])
    # onto one that holds something, onto itself, twice onto one, a chain, outside
    src, dst = [0, 2, 0, 1, 4, 0, 12, 0], [1, 2, 4, 4, 5, 6, 7, -1]
    c.fork(ints(torch, src, dev), ints(torch, dst, dev))
    b.fork(src, dst)
    b.check(c)
    assert b.lengths[6] == 20 and b.lengths[4] == 0
    assert ops.device_error() == _lib.DEVERR_PAGES


def test_free_whole_end_and_middle(env):
    torch, _, dev = env
    c, b = make(env, n_pages=100)
    c.extend(ints(torch, range(5), dev), ints(torch, [100, 33, 160, 16, 7], dev))
    b.extend(list(range(5)), [100, 33, 160, 16, 7])
    c.fork(ints(torch, [0], dev), ints(torch, [8], dev))
    b.fork([0], [8])
    big = 2**31 - 1
    #  all of 0, the end of 1 from 20 on, the middle of 2, a page-aligned end, nothing, twice, outside
    seqs, first, last = [0, 1, 2, 3, 4, 1, 99], [0, 20, 10, 16, 7, 0, 0], [big, big, 90, big, big, big, big]
    c.free(ints(torch, seqs, dev), ints(torch, first, dev), ints(torch, last, dev))
    b.free(seqs, first, last)
    b.check(c)
    assert b.lengths[:5] == [0, 20, 160, 16, 7] and b.table[2][:6].count(-1) == 4
    assert ops.device_error() == _lib.DEVERR_PAGES
    c.extend(ints(torch, [2, 1], dev), ints(torch, [0, 30], dev))
    b.extend([2, 1], [0, 30])
    b.check(c)
    c.free()
    b.free(list(range(12)))
    b.check(c)
    assert not any(b.refs) and ops.device_error() == 0


def test_a_freed_last_page_is_replaced(env):
    torch, _, dev = env
    c, b = make(env)
    c.extend(ints(torch, [0], dev), ints(torch, [20], dev))
    b.extend([0], [20])
    c.free(ints(torch, [0], dev), ints(torch, [16], dev), ints(torch, [19], dev))   # not the whole held part
    b.free([0], [16], [19])
    b.check(c)
    c.table[0, 1] = -1      # a caller's hole
    c.refs[1] = 0
    b.table[0][1], b.refs[1] = -1, 0
    c.extend(ints(torch, [0], dev), ints(torch, [2], dev))
    b.extend([0], [2])
    b.check(c)
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt,page", [(ref.F16, 16), (ref.Q8_ROW, 3)])
def test_compact_moves_pages_and_tables(env, fmt, page):
    torch, _, dev = env
    c, b = make(env, page=page, n_pages=60, max_pages=12, fmt=fmt)
    add = [page * 3 + 1, page * 5, 1, page * 2, page * 7 + 2]
    c.extend(ints(torch, range(5), dev), ints(torch, add, dev))
    b.extend(list(range(5)), add)
    c.fork(ints(torch, [4], dev), ints(torch, [7], dev))
    b.fork([4], [7])
    c.free(ints(torch, [0, 2], dev))
    b.free([0, 2])
    want = [ref.dense(c, layer, s)[:2] for layer in range(2) for s in (1, 3, 4, 7)]
    used = c.compact()
    n, pairs = b.compact()
    assert pairs and used.tolist() == [n]
    b.check(c)
    assert max(p for row in b.table for p in row) == n - 1
    got = [ref.dense(c, layer, s)[:2] for layer in range(2) for s in (1, 3, 4, 7)]
    assert all(np.array_equal(x, y, equal_nan=True) for a, z in zip(want, got) for x, y in zip(a, z))
    assert c.compact().tolist() == [n]   # closed up already
    b.check(c)
    c.free()
    assert c.compact().tolist() == [0]
    assert ops.device_error() == 0


@pytest.mark.parametrize("seed,page,n_pages,max_seqs", [(1, 4, 90, 9), (2, 1, 300, 20), (3, 7, 5000, 1500),
                                                        (4, 64, 20000, 40)])
def test_random_calls_match_the_plain_book(env, seed, page, n_pages, max_seqs):
    torch, _, dev = env
    rng = np.random.default_rng(seed)
    max_pages = 60
    c, b = make(env, page=page, n_pages=n_pages, max_seqs=max_seqs, max_pages=max_pages, hkv=1, layers=1)
    for step in range(25):
        kind = rng.choice(["extend", "extend", "fork", "free", "compact"])
        n = int(rng.integers(1, max_seqs + 1))
        seqs = rng.permutation(max_seqs)[:n].tolist()
        if kind == "extend":
            add = rng.integers(0, 1 + rng.choice([1, 3 * page, max_pages * page // 3]), n).tolist()
            before = c.pool.clone()
            c.extend(ints(torch, seqs, dev), ints(torch, add, dev))
            for a, z in b.extend(seqs, add):
                before[:, z] = before[:, a]
            assert torch.equal(c.pool, before), step
        elif kind == "fork":
            dst = rng.permutation(max_seqs)[:n].tolist()
            c.fork(ints(torch, seqs, dev), ints(torch, dst, dev))
            b.fork(seqs, dst)
        elif kind == "free":
            first = (rng.integers(0, max_pages * page, n) * rng.integers(0, 2, n)).tolist()
            last = [int(x) if rng.random() < 0.4 else 2**31 - 1 for x in rng.integers(0, max_pages * page, n)]
            c.free(ints(torch, seqs, dev), ints(torch, first, dev), ints(torch, last, dev))
            b.free(seqs, first, last)
        else:
            before = c.pool.clone()
            assert c.compact().tolist()[0] == (got := b.compact())[0]
            for a, z in got[1]:
                before[:, z] = before[:, a]
            assert torch.equal(c.pool, before), step
        b.check(c)
    ops.device_error()


# ------------------------------------------------------------------ rows ----
def filled(env, fmt, hkv, hd, page, lens, layers=1, extra=0):
    """A cache whose sequences hold `lens` positions in scattered pages, everything NaN or worst codes."""
    torch, pages, dev = env
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + 5
    c = pages.PagedCache(fmt, hkv, hd, page, n_pages=n_pages, max_seqs=len(lens) + extra, max_pages=max(held + [1]) + 1,
                         layers=layers)
    c.pool.fill_(255)   # NaN in every format's elements or scales
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    at = 0
    for s, h in enumerate(held):
        c.table[s, :h] = order[at : at + h].to(dev)
        c.refs[order[at : at + h].long().to(dev)] = 1
        at += h
    c.lengths[: len(lens)] = ints(torch, lens, dev)
    return c


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hkv,hd,page", [(2, 64, 16), (8, 128, 7), (3, 256, 1), (1, 128, 64)])
def test_append_and_read(env, fmt, hkv, hd, page):
    torch, _, dev = env
    rng = np.random.default_rng(hkv)
    lens, cu = [40, 3, 0, 19, 130], [0, 7, 10, 10, 11, 61]   # new rows 7, 3 (all), none, 1, 50
    c = filled(env, fmt, hkv, hd, page, lens, layers=3)
    rows = cu[-1] + 4   # four rows behind the last entry
    w = hkv * hd
    big = torch.from_numpy((rng.standard_normal((rows, 2 * w + 5)) * np.exp(rng.normal(0, 2, (rows, 1)))).astype(
        np.float32)).to(dev)
    big[0, :hd] = 0.0   # a head of zeros
    k, v = big[:, :w], big[:, w + 5 :]
    before = c.pool.clone()
    c.append(k, v, layer=1, cu_rows=ints(torch, cu, dev))
    assert torch.equal(c.pool[0], before[0]) and torch.equal(c.pool[2], before[2])
    out = [torch.full((rows, w), 7.0, device=dev) for _ in range(2)]
    gk, gv = c.read(rows, layer=1, cu_rows=ints(torch, cu, dev), k=out[0], v=out[1])
    assert ops.device_error() == 0
    for x, g, which in ((k, gk, 0), (v, gv, 1)):
        x, g = x.cpu().double().numpy().reshape(rows, hkv, hd), g.cpu().double().numpy().reshape(rows, hkv, hd)
        assert (g[cu[-1]:] == 7.0).all()   # rows of no entry
        x, g = x[: cu[-1]], g[: cu[-1]]
        if fmt == ref.Q8_ROW:   # half a step of max / 127, and the roundings of scale and product
            top = np.abs(x).max(-1, keepdims=True)
            assert np.all(np.abs(g - x) <= top / 127 * 0.5 * (1 + 2.0**-16) + 2.0**-22 * top)
        else:
            # (below fp16's normal range the half step is 2^-25)
            assert np.all(np.abs(g - x) <= ref.EPS[fmt] * np.abs(x) + 2.0**-25)
        for s in range(len(lens)):   # and the bytes lie where the table says
            n = cu[s + 1] - cu[s]
            kv = ref.dense(c, 1, s)[which]   # (q8: the exact product, which the read rounds to fp32 once)
            assert np.array_equal(kv[lens[s] - n:].astype(np.float32), g[cu[s]:cu[s + 1]].astype(np.float32)), s
            assert not np.isfinite(kv[: lens[s] - n]).any()   # the positions before are untouched
    # nothing else was written: as many elements changed as rows went in
    changed = int((c.pool[1] != before[1]).sum())
    assert changed <= cu[-1] * 2 * hkv * (hd * (1 if fmt == ref.Q8_ROW else 2) + 4)


def test_rounding_is_to_nearest_even(env):
    torch, _, dev = env
    for fmt, t in ((ref.F16, torch.float16), (ref.BF16, torch.bfloat16)):
        c = filled(env, fmt, 1, 64, 4, [1])
        bits = torch.tensor([0x3f800000, 0x3f808000, 0x3f818000, 0x3f801000, 0x3f803000, 0x7f7fffff, 0x7f800000,
                             0xff800000 - 2**32, 0x00000001, 0x33000000, 0x33000001, 0x80000000 - 2**32],
                            dtype=torch.int64).to(torch.int32)
        x = torch.zeros(1, 64)
        x[0, : len(bits)] = bits.view(torch.float32)
        x[0, 40] = float("nan")
        k, v = x.to(dev), torch.flip(x, [1]).to(dev)
        c.append(k, v)
        gk, gv = c.read(1)
        for a, g in ((k, gk), (v, gv)):
            want = a.cpu().to(t).float()
            assert torch.equal(torch.isnan(want), torch.isnan(g.cpu()))
            assert torch.equal(torch.nan_to_num(want, nan=1.0), torch.nan_to_num(g.cpu(), nan=1.0))


def test_q8_rows_that_are_not_finite_or_tiny(env):
    torch, _, dev = env
    c = filled(env, ref.Q8_ROW, 4, 64, 4, [1])
    k = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1))
    k[0, 1, 5], k[0, 2, 6] = float("nan"), float("-inf")
    k[0, 3] = torch.arange(64) * 1.4e-45 * 3   # subnormal
    c.append(k.view(1, -1).to(dev), k.view(1, -1).to(dev))
    g = c.read(1)[0].cpu().view(4, 64)
    assert torch.isfinite(g[0]).all() and torch.isnan(g[1]).all() and torch.isnan(g[2]).all()
    assert (g[3] - k[0, 3]).abs().max() <= 64 * 1.5e-45 + 1.5e-45 * 63   # half a step of code 127 and of the scale
    assert ops.device_error() == 0


def test_rows_of_bad_entries(env):
    torch, _, dev = env
    c = filled(env, ref.F16, 2, 64, 4, [9, 6, 2], extra=1)
    c.table[1, 1] = -1
    c.table[0, 2] = 10**6
    k = torch.ones(5, 128, device=dev)
    before = c.pool.clone()
    #  a position without a page, a page past the pool, a sequence outside, rows before the start
    seqs, cu = ints(torch, [1, 0, 7, 2], dev), ints(torch, [0, 1, 2, 2, 5], dev)
    c.append(k, k, seqs=seqs, cu_rows=cu)
    assert ops.device_error() == _lib.DEVERR_PAGES
    gk, gv = c.read(5, seqs=seqs, cu_rows=cu)
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert gk.tolist() == [[0.0] * 128] * 3 + [[1.0] * 128] * 2 and torch.equal(gk, gv)
    assert int((c.pool != before).sum()) <= 2 * 2 * 128 * 2
    c.append(k[:1], k[:1], seqs=ints(torch, [-3], dev))
    assert ops.device_error() == _lib.DEVERR_PAGES


def test_a_workspace_elsewhere_is_refused(env):
    torch, pages, dev = env
    c, _ = make(env)
    need = c.workspace_bytes(1)
    with pytest.raises(TypeError):
        c.extend(n=1, workspace=torch.empty(need, dtype=torch.uint8))
    with pytest.raises(TypeError):
        c.compact(workspace=np.empty(need, np.uint8))
    with pytest.raises(ValueError):
        c.extend(n=1, workspace=torch.empty(need, 2, dtype=torch.uint8, device=dev)[:, 0])
    with pytest.raises(_lib.RtaError):
        c.extend(n=1, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))
    c.extend(n=1, workspace=torch.empty(need, dtype=torch.uint8, device=dev))
    assert c.lengths.tolist()[0] == 1 and ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
def test_rows_at_any_multiple_of_four_bytes(env, fmt):
    """append and read at strides and addresses that are no multiple of 16 bytes."""
    torch, pages, dev = env
    gen = torch.Generator(device=dev).manual_seed(5)
    got = []
    for shift, pitch in ((0, 128), (1, 131), (3, 129)):
        c = filled(env, fmt, 2, 64, 5, [7, 3])
        gen.manual_seed(5)
        rows = torch.randn(10, 2, 128, generator=gen, device=dev)
        flat = torch.zeros(2, 10 * pitch + 4, device=dev)
        k, v = (flat[i, shift : shift + 10 * pitch].view(10, pitch)[:, :128] for i in (0, 1))
        k.copy_(rows[:, 0])
        v.copy_(rows[:, 1])
        cu = ints(torch, [0, 7, 10], dev)
        c.append(k, v, cu_rows=cu)
        back = torch.full((2, 10 * pitch + 4), 7.0, device=dev)
        kb, vb = (back[i, shift : shift + 10 * pitch].view(10, pitch)[:, :128] for i in (0, 1))
        c.read(10, cu_rows=cu, k=kb, v=vb)
        outside = torch.ones_like(back, dtype=torch.bool)
        for i in (0, 1):
            outside[i, shift : shift + 10 * pitch].view(10, pitch)[:, :128] = False
        assert torch.all(back[outside] == 7.0)
        got.append((kb.clone(), vb.clone()))
    for kb, vb in got[1:]:
        assert torch.equal(kb, got[0][0]) and torch.equal(vb, got[0][1])
    assert ops.device_error() == 0


def test_python_refusals(env):
    torch, pages, dev = env
    with pytest.raises(ValueError):
        pages.PagedCache(_lib.Q4_K, 2, 64, 16, n_pages=4, max_seqs=2, max_pages=2)
    with pytest.raises(ValueError):
        pages.PagedCache(_lib.F16, 2, 64, 16, n_pages=4)
    c, _ = make(env)
    with pytest.raises(ValueError):
        pages.PagedCache(_lib.F16, 2, 64, 16, pool=c.pool)
    with pytest.raises(ValueError):
        pages.PagedCache(_lib.F16, 2, 64, 32, pool=c.pool, table=c.table, lengths=c.lengths, refs=c.refs)
    with pytest.raises(TypeError):
        c.extend(torch.zeros(3, dtype=torch.int64, device=dev))
    with pytest.raises(TypeError):
        c.extend(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        c.extend(ints(torch, [1, 2], dev), ints(torch, [1], dev))
    with pytest.raises(_lib.RtaError):
        c.extend(n=0)
    with pytest.raises(_lib.RtaError):
        c.extend(ints(torch, [1], dev), workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    with pytest.raises(TypeError):
        c.fork(None, ints(torch, [1], dev))
    with pytest.raises(ValueError):
        c.append(torch.zeros(13, 128, device=dev), torch.zeros(13, 128, device=dev))   # 13 entries, 12 sequences
    with pytest.raises(TypeError):
        c.append(torch.zeros(2, 128, device=dev).half(), torch.zeros(2, 128, device=dev).half())
    with pytest.raises(_lib.RtaError):
        c.append(torch.zeros(2, 128, device=dev), torch.zeros(2, 128, device=dev), layer=2)
    with pytest.raises(ValueError):
        c.attention(torch.zeros(2, 4, 128, device=dev))
    with pytest.raises(_lib.RtaError):
        c.attention(torch.zeros(2, 3, 64, device=dev))
    with pytest.raises(ValueError):
        c.attention(torch.zeros(2, 4, 64, device=dev), gate=torch.zeros(2, 2, 64, device=dev))
    assert ops.device_error() == 0
