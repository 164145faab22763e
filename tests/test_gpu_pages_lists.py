"""Lists and books that the paged history's calls refuse on the device: the entry is left undone,
RTA_DEVERR_PAGES is raised, and the others come out as they should."""
import numpy as np
import pytest

import paged_reference as ref
from rta import _lib, ops
from test_gpu_paged_attention import fill, rows_of, want_rows
from test_gpu_pages import env, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu

LENS = [1500, 40, 700]
# row offsets over nine rows and three entries, and the entries that are good
LISTS = [([-3, 2, 5, 9], [1, 2]), ([0, 2, 5, 12], [0, 1]), ([0, 2, 5, 2**31 - 1], [0, 1]), ([4, 9, 12, 20], [0]),
         ([12, 13, 14, 15], []), ([-9, -5, -2, 0], []), ([-2**31, 0, 4, 9], [1, 2])]
# where a list falls, a row has two entries (whose parts of it may mix) or is not found by the offsets around it:
# a row of one entry comes out as that has it, or stays as it was
FALLING = [([0, 4, 3, 9], [0, 2]), ([3, 3, 1, 6], [0, 2])]


def rows_left(cu, good):
    """(entries with rows as (entry, first row, count), rows that no good entry has)."""
    held = np.zeros(9, int)
    for i in good:
        held[cu[i] : cu[i + 1]] += 1
    return [(i, cu[i], cu[i + 1] - cu[i]) for i in good], np.flatnonzero(held == 0)


# ------------------------------------------------------------------ row lists ----
@pytest.mark.parametrize("fmt", [ref.F16, ref.Q8_ROW])
@pytest.mark.parametrize("hq", [4, 16])   # few columns, and more
@pytest.mark.parametrize("cu,good", LISTS + FALLING, ids=str)
def test_attention_leaves_bad_rows(env, fmt, hq, cu, good):
    torch, _, dev = env
    c = filled(env, fmt, 1, 64, 16, LENS)
    fill(env, c, LENS, 3)
    q = rows_of(torch, dev, 9, hq, 64, 4)
    out = torch.full((9, hq, 64), 7.0, device=dev)
    m, z = torch.full((9, hq), 7.0, device=dev), torch.full((9, hq), 7.0, device=dev)
    how = dict(cu_rows=ints(torch, cu, dev), max_rows=6, max_len=1500)
    assert c.attention_workspace_bytes(hq, 9, 3, 6, 1500) > 0   # cut into chunks, so there is a merge
    # what an earlier call left in the workspace must not come out
    ws = torch.full((c.attention_workspace_bytes(hq, 9, 3, 6, 1500),), 63, dtype=torch.uint8, device=dev)
    c.attention(q, out=out, m=m, z=z, workspace=ws, **how)
    assert ops.device_error() == _lib.DEVERR_PAGES
    entries, left = rows_left(cu, good)
    for t in (out, m, z):
        assert all((t[r] == 7.0).all() for r in left)
    if (cu, good) not in FALLING:
        for i, first, count in entries:
            ref.check_rows([t[first : first + count] for t in (out, m, z)], want_rows(c, q, [(i, first, count)]), (cu, i))
        return
    for r in set(range(9)) - set(left.tolist()):
        of = [(i, first, count) for i, first, count in entries if first <= r < first + count]
        if len(of) == 1 and not (out[r] == 7.0).all():
            ref.check_rows([t[r : r + 1] for t in (out, m, z)], [want_rows(c, q, of)[r - of[0][1]]], r)


@pytest.mark.parametrize("cu,good", [([-1, 1, 2, 3], [1, 2]), ([0, 1, 2, 4], [0, 1]), ([3, 4, 5, 6], [])], ids=str)
@pytest.mark.parametrize("max_len", [1500, 100])
def test_single_rows_of_bad_lists(env, cu, good, max_len):
    torch, _, dev = env
    lens = [min(n, max_len) for n in LENS]
    c = filled(env, ref.F16, 1, 64, 16, lens)
    fill(env, c, lens, 5)
    q = rows_of(torch, dev, 3, 4, 64, 6)
    out = torch.full((3, 4, 64), 7.0, device=dev)
    _, m, z = c.attention(q, cu_rows=ints(torch, cu, dev), max_rows=1, max_len=max_len, out=out)
    assert ops.device_error() == _lib.DEVERR_PAGES
    for r in range(3):
        i = [i for i in good if cu[i] == r]
        if i:
            ref.check_rows([t[r : r + 1] for t in (out, m, z)], want_rows(c, q, [(i[0], r, 1)]))
        else:
            assert (out[r] == 7.0).all()


@pytest.mark.parametrize("cu,good", LISTS, ids=str)
def test_rows_in_and_out_of_bad_lists(env, cu, good):
    torch, _, dev = env
    c, d = (filled(env, ref.BF16, 2, 64, 16, LENS) for _ in range(2))
    d.pool.copy_(c.pool)
    entries, left = rows_left(cu, good)
    x = torch.randn(9, 2, 128, generator=torch.Generator().manual_seed(7)).to(dev)
    c.append(x[:, 0], x[:, 1], cu_rows=ints(torch, cu, dev))
    assert ops.device_error() == _lib.DEVERR_PAGES
    for i, first, count in entries:   # the same rows by lists of their own
        rows = x[first : first + count]
        d.append(rows[:, 0], rows[:, 1], seqs=ints(torch, [i], dev), cu_rows=ints(torch, [0, count], dev))
    assert ops.device_error() == 0
    assert torch.equal(c.pool, d.pool)
    back = [torch.full((9, 128), 7.0, device=dev) for _ in range(2)]
    d.read(9, cu_rows=ints(torch, cu, dev), k=back[0], v=back[1])
    assert ops.device_error() == _lib.DEVERR_PAGES
    want = x.bfloat16().float()
    want[left.tolist()] = 7.0
    assert torch.equal(back[0], want[:, 0]) and torch.equal(back[1], want[:, 1])


@pytest.mark.parametrize("cu,good", FALLING, ids=str)
def test_rows_in_and_out_of_falling_lists(env, cu, good):
    torch, _, dev = env
    c = filled(env, ref.BF16, 2, 64, 16, LENS)
    before = c.pool.clone()
    _, left = rows_left(cu, good)
    x = torch.ones(9, 128, device=dev)
    c.append(x, x, cu_rows=ints(torch, cu, dev))
    assert ops.device_error() == _lib.DEVERR_PAGES
    changed = c.pool.view(torch.bfloat16)[c.pool.view(torch.bfloat16).view(torch.int16) != before.view(torch.int16)]
    assert bool((changed == 1.0).all())
    back = torch.full((9, 128), 7.0, device=dev)
    c.read(9, cu_rows=ints(torch, cu, dev), k=back, v=back.clone())
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert all((back[r] == 7.0).all() for r in left)


# ------------------------------------------------------------------ compaction ----
@pytest.mark.parametrize("page", [1, 4])
def test_compact_leaves_entries_of_free_pages(env, page):
    """Table entries that name pages outside the pool or that the counts call free, below and past the
    pages in use, stay as they are; the others follow their pages."""
    torch, pages, dev = env
    c = pages.PagedCache(ref.F16, 1, 64, page, n_pages=600, max_seqs=6, max_pages=200)
    b = ref.Book(page, 600, 6, 200)
    add = [100 * page, 60 * page, 120 * page]
    c.extend(ints(torch, range(3), dev), ints(torch, add, dev))
    b.extend([0, 1, 2], add)
    c.free(ints(torch, [1], dev))
    b.free([1])
    # sequences 4 and 5 (empty in the book): a hole below the pages in use, free ones past them, a page in use, outside
    odd = {(4, 0): 130, (4, 1): 590, (4, 7): 279 + 1, (5, 0): 600, (5, 3): -2, (5, 4): 2**31 - 1, (5, 5): 270}
    for (s, e), p in odd.items():
        c.table[s, e] = b.table[s][e] = p
    ws = torch.full((c.workspace_bytes(),), 1, dtype=torch.uint8, device=dev)   # (numbers that are no answer)
    used = c.compact(workspace=ws)
    n, pairs = b.compact()
    assert pairs and used.tolist() == [n] and b.table[5][5] != 270
    b.check(c)
    assert ops.device_error() == _lib.DEVERR_PAGES


# ------------------------------------------------------------------ lengths and pages outside ----
def grown(env):
    """Four sequences of 20, 33, 64 and 16 positions, pages of 16, at most 4 each; the book beside it."""
    torch, pages, dev = env
    c = pages.PagedCache(ref.F16, 1, 64, 16, n_pages=40, max_seqs=8, max_pages=4)
    b = ref.Book(16, 40, 8, 4)
    c.extend(ints(torch, range(4), dev), ints(torch, [20, 33, 64, 16], dev))
    b.extend([0, 1, 2, 3], [20, 33, 64, 16])
    return c, b


@pytest.mark.parametrize("length", [65, 2**31 - 1, -1, -2**31])
def test_lengths_that_the_table_cannot_hold(env, length):
    """A caller's length of sequence 2: forks of it, frees (whole, its end, its middle) and extends are
    left undone, the other entries are done."""
    torch, _, dev = env
    for what in ("fork", "whole", "end", "middle", "extend"):
        c, b = grown(env)
        c.lengths[2] = b.lengths[2] = length
        if what == "fork":
            c.fork(ints(torch, [2, 1], dev), ints(torch, [5, 6], dev))
            b.fork([1], [6])
        elif what == "extend":
            c.extend(ints(torch, [2, 1], dev))
            b.extend([1], [1])
        else:
            first, last = {"whole": (None, None), "end": ([16, 16], None), "middle": ([16, 16], [32, 32])}[what]
            c.free(ints(torch, [2, 1], dev), None if first is None else ints(torch, first, dev),
                   None if last is None else ints(torch, last, dev))
            b.free([1], first and first[:1], last and last[:1])
        b.check(c)
        assert ops.device_error() == _lib.DEVERR_PAGES, what


@pytest.mark.parametrize("page", [40, 2**31 - 1, -2, -2**31])
def test_pages_outside_the_pool(env, page):
    """A caller's table entry that is neither a page nor -1: what would copy, free or replace it is left
    undone; what does not touch it is done."""
    torch, _, dev = env
    for what in ("fork", "free", "before", "extend"):
        c, b = grown(env)
        c.table[1, 2] = b.table[1][2] = page   # the third, partly filled page of sequence 1
        if what == "fork":
            c.fork(ints(torch, [1, 0], dev), ints(torch, [5, 6], dev))
            b.fork([0], [6])
        elif what == "free":
            c.free(ints(torch, [1, 0], dev))
            b.free([0])
        elif what == "extend":
            c.extend(ints(torch, [1, 0], dev))
            b.extend([0], [1])
        else:   # the first two pages of it
            c.free(ints(torch, [1], dev), None, ints(torch, [32], dev))
            b.free([1], None, [32])
        b.check(c)
        assert ops.device_error() == (0 if what == "before" else _lib.DEVERR_PAGES), what


def test_holes_are_forked_and_freed(env):
    """-1 is no bad page: a sequence whose window has passed its first pages goes on like any other."""
    torch, _, dev = env
    c, b = grown(env)
    c.free(ints(torch, [2], dev), None, ints(torch, [40], dev))
    b.free([2], None, [40])
    c.fork(ints(torch, [2], dev), ints(torch, [7], dev))
    b.fork([2], [7])
    c.free(ints(torch, [2], dev))
    b.free([2])
    b.check(c)
    assert b.table[7] == [-1, -1] + b.table[7][2:] and ops.device_error() == 0


# ------------------------------------------------------------------ arguments ----
def test_queries_of_one_head_at_any_stride(env):
    """A head's stride says nothing where there is one head."""
    torch, _, dev = env
    lens = [30, 70, 5]
    c = filled(env, ref.F16, 1, 64, 16, lens)
    fill(env, c, lens, 8)
    q = rows_of(torch, dev, 3, 1, 64, 9)
    turned = torch.empty(1, 3, 64, device=dev).transpose(0, 1).copy_(q)
    assert turned.stride(1) != 64
    got, want = c.attention(turned, max_len=70), c.attention(q, max_len=70)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and ops.device_error() == 0


def test_lists_that_are_no_tensors(env):
    torch, _, dev = env
    c, _ = grown(env)
    for call in (lambda: c.extend([1, 2]), lambda: c.free([1]), lambda: c.fork([0], ints(torch, [5], dev)),
                 lambda: c.fork(ints(torch, [0], dev), [5]), lambda: c.attention(torch.zeros(1, 1, 64, device=dev), seqs=[0])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: c.extend(ints(torch, [[1, 2]], dev)), lambda: c.append([1.0], [2.0])):
        with pytest.raises(ValueError):
            call()
    assert c.lengths.tolist()[:4] == [20, 33, 64, 16] and ops.device_error() == 0
