"""Attention over the paged history against 64-bit attention of the pages' own values: formats,
head layouts, page sizes, lengths from nothing to long, windows and first tokens, several rows per
sequence, bad entries, and a whole serving loop, eager and captured in a graph."""
import numpy as np
import pytest

import paged_reference as ref
from rta import _lib, ops
from test_gpu_pages import env, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def fill(env, c, lens, seed):
    """Random values at the sequences' held positions of every layer; all else stays as it was."""
    torch, _, dev = env
    gen = torch.Generator(device=dev).manual_seed(seed)
    w = c.kv_heads * c.head_dim
    cu = np.concatenate([[0], np.cumsum(lens)])
    for layer in range(c.pool.shape[0]):
        k = torch.randn(int(cu[-1]), w, generator=gen, device=dev)
        v = torch.randn(int(cu[-1]), w, generator=gen, device=dev) + 0.3
        if cu[-1]:
            c.append(k, v, layer=layer, seqs=ints(torch, range(len(lens)), dev), cu_rows=ints(torch, cu, dev))


def rows_of(torch, dev, n, hq, hd, seed, scale=1.5, pad=0):
    x = scale * torch.randn(n, hq * hd + pad, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)
    return x[:, : hq * hd].unflatten(1, (hq, hd))


def want_rows(c, q, entries, layer=0, window=0, sinks=0, gate=None, missing_ok=False):
    """entries: (sequence, first row, count); rows in order."""
    q = q.cpu().double().numpy()
    gate = None if gate is None else gate.cpu().double().numpy()
    got = []
    for s, first, count in entries:
        k, v, held = ref.dense(c, layer, s, missing_ok)
        for j in range(count):
            r = first + j
            got.append(ref.attend(q[r], k, v, held, len(k) - count + j, window, sinks,
                                  None if gate is None else gate[r]))
    return got


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hq,hkv,hd,page", [(8, 8, 128, 16), (32, 8, 128, 64), (12, 2, 64, 7), (8, 1, 256, 1),
                                            (16, 1, 64, 32), (34, 2, 128, 24), (9, 3, 256, 100)])
def test_one_row_per_sequence(env, fmt, hq, hkv, hd, page):
    torch, _, dev = env
    lens = [1, 0, 31, 32, 33, 64, 129, 700, 257]
    c = filled(env, fmt, hkv, hd, page, lens)
    fill(env, c, lens, 3)
    q = rows_of(torch, dev, len(lens), hq, hd, 4, pad=64)
    got = c.attention(q, max_len=700)
    ref.check_rows(got, want_rows(c, q, [(s, s, 1) for s in range(len(lens))]), (fmt, hq, hkv, hd, page))
    assert ops.device_error() == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (32, 4), (100, 3), (128, 64), (129, 500), (5000, 7), (0, 9)])
@pytest.mark.parametrize("fmt,page", [(ref.F16, 16), (ref.Q8_ROW, 3)])
def test_windows_and_first_tokens(env, fmt, page, window, sinks):
    torch, _, dev = env
    lens = [1, 2, 0, 100, 101, 132, 133, 134, 999]
    c = filled(env, fmt, 2, 128, page, lens)
    fill(env, c, lens, 5)
    q = rows_of(torch, dev, len(lens), 8, 128, 6)
    got = c.attention(q, max_len=999, window=window, sinks=sinks)
    want = want_rows(c, q, [(s, s, 1) for s in range(len(lens))], window=window, sinks=sinks)
    ref.check_rows(got, want, (window, sinks))
    if window:   # the pages that the window has left behind may be freed
        first = ints(torch, [sinks] * len(lens), dev)
        last = ints(torch, [max(0, n - window) for n in lens], dev)
        c.free(ints(torch, range(len(lens)), dev), first, last)
        ref.check_rows(c.attention(q, max_len=999, window=window, sinks=sinks), want, "freed")
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hq,hkv,hd,page,window,sinks", [(8, 2, 128, 16, 0, 0), (32, 8, 128, 64, 40, 4),
                                                         (12, 1, 64, 5, 0, 0), (6, 3, 256, 33, 64, 70),
                                                         (16, 16, 128, 128, 1, 2), (20, 1, 128, 8, 0, 0)])
def test_several_rows_per_sequence(env, fmt, hq, hkv, hd, page, window, sinks):
    torch, _, dev = env
    lens = [5, 300, 64, 0, 129, 1, 97]
    counts = [5, 3, 64, 0, 70, 1, 33]     # a prompt from nothing, drafts, none, chunks, a single token
    c = filled(env, fmt, hkv, hd, page, lens, layers=2)
    fill(env, c, lens, 7)
    cu = np.concatenate([[2], 2 + np.cumsum(counts)])   # two rows in front and three behind are nobody's
    rows = int(cu[-1]) + 3
    q = rows_of(torch, dev, rows, hq, hd, 8, pad=4)
    seqs = [4, 1, 0, 3, 2, 6, 5]
    order = [seqs.index(s) for s in range(7)]   # entry of each sequence
    cnt = [counts[s] for s in seqs]
    cu = np.concatenate([[2], 2 + np.cumsum(cnt)])
    out = torch.full((rows, hq, hd), 7.0, device=dev)
    m, z = torch.full((rows, hq), 7.0, device=dev), torch.full((rows, hq), 7.0, device=dev)
    c.attention(q, layer=1, seqs=ints(torch, seqs, dev), cu_rows=ints(torch, cu, dev), max_rows=70, max_len=300,
                window=window, sinks=sinks, out=out, m=m, z=z)
    for t in (out, m, z):
        assert (t[:2] == 7.0).all() and (t[-3:] == 7.0).all()
    entries = [(s, int(cu[i]), cnt[i]) for i, s in enumerate(seqs)]
    want = want_rows(c, q, entries, layer=1, window=window, sinks=sinks)
    ref.check_rows([t[2:-3] for t in (out, m, z)], want, (fmt, hq, hkv, hd, page))
    assert ops.device_error() == 0 and len(order) == 7


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hq,hkv,hd,page,window,sinks", [(8, 2, 128, 16, 0, 0), (32, 4, 128, 64, 40, 4),
                                                         (12, 2, 64, 5, 0, 0), (6, 3, 256, 33, 64, 70),
                                                         (40, 2, 256, 64, 0, 0), (20, 1, 64, 8, 3, 1)])
def test_a_few_rows_per_sequence(env, fmt, hq, hkv, hd, page, window, sinks):
    torch, _, dev = env
    lens, counts = [3, 300, 64, 0, 129, 1, 1200], [3, 2, 3, 0, 1, 1, 3]
    c = filled(env, fmt, hkv, hd, page, lens)
    fill(env, c, lens, 31)
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = rows_of(torch, dev, int(cu[-1]), hq, hd, 32)
    gate = rows_of(torch, dev, int(cu[-1]), hq, hd, 33).contiguous()
    for g, most in ((None, 3), (gate, 5)):   # the bound may be above the most there are
        got = c.attention(q, cu_rows=ints(torch, cu, dev), max_rows=most, max_len=1200, window=window, sinks=sinks, gate=g)
        want = want_rows(c, q, [(s, int(cu[s]), counts[s]) for s in range(7)], window=window, sinks=sinks, gate=g)
        ref.check_rows(got, want, (fmt, hq, hkv, hd, page))
    assert ops.device_error() == 0


@pytest.mark.parametrize("rows,length", [(2, 4000), (9, 2500), (200, 1500), (513, 513)])
def test_rows_split_over_long_histories(env, rows, length):
    torch, _, dev = env
    c = filled(env, ref.F16, 1, 128, 64, [length, 40])
    fill(env, c, [length, 40], 9)
    q = rows_of(torch, dev, rows + 1, 4, 128, 10)
    got = c.attention(q, cu_rows=ints(torch, [0, rows, rows + 1], dev), max_rows=rows, max_len=length)
    ref.check_rows(got, want_rows(c, q, [(0, 0, rows), (1, rows, 1)]), rows)
    assert ops.device_error() == 0


def test_gate_optional_outputs_and_repeats(env):
    torch, _, dev = env
    lens = [50, 700]
    c = filled(env, ref.BF16, 2, 128, 16, lens)
    fill(env, c, lens, 11)
    q = rows_of(torch, dev, 4, 8, 128, 12)
    gate = rows_of(torch, dev, 4, 8, 128, 13, 3.0).contiguous()
    seqs = ints(torch, [1, 0, 1, 1], dev)   # a sequence may be read by several entries
    got = c.attention(q, seqs=seqs, max_len=700, gate=gate)
    ref.check_rows(got, want_rows(c, q, [(1, 0, 1), (0, 1, 1), (1, 2, 1), (1, 3, 1)], gate=gate))
    out = torch.empty_like(got[0])
    ws = torch.empty(max(16, c.attention_workspace_bytes(8, 4, max_len=700)), dtype=torch.uint8, device=dev)
    c._call("rta_paged_attention", 0, q.data_ptr(), q.stride(0), 4, 8, seqs.data_ptr(), None, 4, 1, 700, 0, 0,
            gate.data_ptr(), out.data_ptr(), None, None, ws.data_ptr(), ws.numel())
    assert torch.equal(out, got[0])


def test_bad_entries_read_as_nothing(env):
    torch, _, dev = env
    lens = [40, 500, 10, 100]
    c = filled(env, ref.F16, 2, 64, 16, lens)
    fill(env, c, lens, 14)
    q = rows_of(torch, dev, 4, 4, 64, 15)
    # outside, longer than max_len, in order, and with a page missing in the middle
    c.table[3, 2], c.table[3, 4] = -1, 10**8
    out, m, z = c.attention(q, seqs=ints(torch, [9, 1, 2, 3], dev), max_len=400)
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert not out[:2].any() and not z[:2].any() and (m[:2] == -np.inf).all()
    want = want_rows(c, q, [(2, 2, 1), (3, 3, 1)], missing_ok=True)
    ref.check_rows([t[2:] for t in (out, m, z)], want)
    # more rows than positions: the early ones see nothing; more than max_rows: left as they were
    q = rows_of(torch, dev, 20, 4, 64, 16)
    out = torch.full((20, 4, 64), 7.0, device=dev)
    got = c.attention(q, seqs=ints(torch, [2, 0], dev), cu_rows=ints(torch, [0, 12, 20], dev), max_rows=12, out=out)
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert not out[:2].any()
    ref.check_rows([t[2:] for t in got], want_rows(c, q, [(2, 0, 12), (0, 12, 8)])[2:])
    out = torch.full((20, 4, 64), 7.0, device=dev)
    got = c.attention(q, seqs=ints(torch, [0, 3], dev), cu_rows=ints(torch, [0, 15, 20], dev), max_rows=12, out=out)
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert (out[12:15] == 7.0).all()
    want = want_rows(c, q, [(0, 0, 15), (3, 15, 5)], missing_ok=True)
    ref.check_rows([t[:12] for t in got], want[:12])
    ref.check_rows([t[15:] for t in got], want[15:])
    # every visible position without a page
    c.table[2] = -1
    for cu in (None, ints(torch, [0, 3], dev)):
        n = 1 if cu is None else 3
        out, m, z = c.attention(q[:n], seqs=ints(torch, [2], dev), cu_rows=cu)
        assert not out.any() and not z.any() and (m == -np.inf).all()
        assert ops.device_error() == _lib.DEVERR_PAGES


def test_a_visible_value_that_is_not_finite_is_reported(env):
    torch, _, dev = env
    c = filled(env, ref.F16, 1, 64, 8, [20])
    fill(env, c, [20], 17)
    q = rows_of(torch, dev, 1, 2, 64, 18)
    kv = c.pool.view(torch.float16)
    kv[0, c.table[0, 1].long(), 3] = float("inf")   # key of position 11
    c.attention(q)
    assert ops.device_error() & _lib.DEVERR_DETECTOR
    c.attention(q, window=9)   # not seen any more
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,hq,hkv,window", [(4, 4, 1, 0), (8, 4, 1, 5), (90, 8, 2, 0), (90, 8, 2, 24)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(env, fmt, hd, rows, hq, hkv, window):
    """Keys and values of two positions are inf and NaN: rows before them, and rows whose window has
    passed them, come out as if those positions held anything else."""
    torch, _, dev = env
    length = 130
    c = filled(env, fmt, hkv, hd, 16, [length])
    fill(env, c, [length], 36)
    q = rows_of(torch, dev, rows, hq, hd, 37)
    cu = ints(torch, [0, rows], dev)
    p0 = length - rows
    odd = sorted({p0 + 2, p0 + rows // 2})
    for p in odd:
        for which in (0, 1):
            page = int(c.table[0, p // 16])
            if fmt == ref.Q8_ROW:
                at = (which * hkv * 16 + p % 16) * 4 + 2 * hkv * 16 * hd
                c.pool[0, page, at : at + 4] = torch.tensor([float("inf")], device=dev).view(torch.uint8)
            else:
                e = c.pool[0, page].view(torch.float16 if fmt == ref.F16 else torch.bfloat16)
                at = (which * hkv * 16 + p % 16) * hd
                e[at + 3], e[at + 5] = float("nan"), float("-inf")
    out, m, z = c.attention(q, cu_rows=cu, max_rows=rows, window=window)
    assert ops.device_error() & _lib.DEVERR_DETECTOR
    # the oracle sees finite numbers there: rows that may not look at them do not change
    k, v, held = ref.dense(c, 0, 0)
    k, v = np.nan_to_num(k, nan=1.0, posinf=1.0, neginf=1.0), np.nan_to_num(v, nan=1.0, posinf=1.0, neginf=1.0)
    per = hq // hkv
    clean = seen = 0
    for r in range(rows):
        t = p0 + r
        sees = any(p <= t and (not window or p > t - window) for p in odd)
        if sees:
            seen += 1
            heads = slice(per, hq)   # kv head 0 holds them: its values mean nothing
        else:
            clean += 1
            heads = slice(0, hq)
        want = ref.attend(q[r].cpu().double().numpy(), k, v, held, t, window)
        if heads.start < hq:
            ref.check_rows([x[r : r + 1, heads] for x in (out, m, z)], [tuple(w[heads] for w in want)], r)
    assert clean >= 2 and seen >= 2


def test_large_scores_and_tiny_queries(env):
    torch, _, dev = env
    lens = [300, 300, 300]
    for fmt in (ref.F16, ref.BF16, ref.Q8_ROW):
        c = filled(env, fmt, 2, 128, 16, lens)
        fill(env, c, lens, 19)
        q = rows_of(torch, dev, 3, 8, 128, 20)
        q[0] *= 40.0        # scores of some hundreds: one position takes nearly all
        q[1] *= 1e-30       # all alike
        q[2, :, 5:] = 0.0
        q[2, 3] = 0.0
        got = c.attention(q, max_len=300)
        ref.check_rows(got, want_rows(c, q, [(s, s, 1) for s in range(3)]), fmt)
        several = c.attention(q, seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, 3], dev))
        ref.check_rows(several, want_rows(c, q, [(0, 0, 3)]), fmt)
    assert ops.device_error() == 0


def test_pools_past_four_gigabytes(env):
    torch, pages, dev = env
    page = 1024
    pb = pages.page_bytes(ref.F16, 4, 128, page)
    n_pages = (5 << 30) // pb
    pool = torch.empty(1, n_pages, pb, dtype=torch.uint8, device=dev)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    table = torch.full((1, 4), -1, dtype=torch.int32, device=dev)
    names = [n_pages - 1, n_pages - 3, 0]
    table[0, :3] = ints(torch, names, dev)
    refs[names] = 1
    lens = [2 * page + 77]
    c = pages.PagedCache(ref.F16, 4, 128, page, pool=pool, table=table, lengths=ints(torch, lens, dev), refs=refs)
    fill(env, c, lens, 21)
    q = rows_of(torch, dev, 1, 8, 128, 22)
    ref.check_rows(c.attention(q), want_rows(c, q, [(0, 0, 1)]))
    kv = [ref.dense(c, 0, 0)[i] for i in (0, 1)]
    assert c.compact().tolist() == [3] and sorted(c.table[0, :3].tolist()) == [0, 1, 2]
    assert all(np.array_equal(a, b) for a, b in zip(kv, ref.dense(c, 0, 0)))
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("length", [2048, 60000])
def test_long_histories_keep_fp32_precision(env, fmt, length):
    """Over a long history nearly all of the sum lies in weights far below the largest, and values
    around zero leave nothing of it but the weights' own errors.  Bound: every weight carries the
    roundings of its score (up to 16 in log2 units: half a step 2^-21) and of its parts (2^-22),
    all of them independent: 2^-20 of a head's result, doubled."""
    torch, _, dev = env
    c = filled(env, fmt, 1, 128, 256, [length])
    gen = torch.Generator(device=dev).manual_seed(34)
    k, v = (torch.randn(length, 128, generator=gen, device=dev) for _ in range(2))
    c.append(k, v, cu_rows=ints(torch, [0, length], dev))
    q = rows_of(torch, dev, 5, 8, 128, 35, 1.5)
    k, v, _ = ref.dense(c, 0, 0)
    p = np.exp(q.cpu().double().numpy() @ k[:, 0].T / np.sqrt(128))   # [5, 8, length]
    for n in (1, 2, 5):   # one row, and two and five in 16 and 32 columns of the kernel of a few
        got = c.attention(q[:n], cu_rows=ints(torch, [0, n], dev), max_rows=n)[0]
        for r in range(n):
            w = p[r][:, : length - n + 1 + r]
            want = w @ v[: w.shape[1], 0] / w.sum(1, keepdims=True)
            err = np.linalg.norm(got[r].cpu().double().numpy() - want, axis=1)
            assert np.all(err <= 2 * 2.0**-20 * np.linalg.norm(want, axis=1)), (n, r, err / np.linalg.norm(want, axis=1))


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("counts", [[1, 1], [5, 3], [80, 41]])
def test_tensors_at_any_multiple_of_four_bytes(env, fmt, hd, counts):
    """Queries of an odd row stride, and out, gate, m and z at addresses that are no multiple of 16."""
    torch, _, dev = env
    lens, hq = [600, 41], 4
    c = filled(env, fmt, 2, hd, 16, lens)
    fill(env, c, lens, 38)
    rows = sum(counts)
    q, gate = rows_of(torch, dev, rows, hq, hd, 39), rows_of(torch, dev, rows, hq, hd, 40)
    cu = None if max(counts) == 1 else ints(torch, np.concatenate([[0], np.cumsum(counts)]), dev)
    how = dict(cu_rows=cu, max_rows=max(counts), max_len=600, window=300, sinks=2)
    want = c.attention(q, gate=gate, **how)

    def odd(t, shift, pitch):
        flat = torch.full((shift + rows * pitch + 8,), 7.0, device=dev)
        x = flat[shift : shift + rows * pitch].view(rows, pitch)[:, : t[0].numel()].view(t.shape)
        x.copy_(t)
        return flat, x

    n = hq * hd
    for shift in (1, 2, 3):
        _, q2 = odd(q, shift, n + shift)
        _, g2 = odd(gate, 4 - shift, n)
        flat, out = odd(torch.zeros_like(q), shift, n)
        _, m = odd(torch.zeros(rows, hq, device=dev), shift, hq)
        _, z = odd(torch.zeros(rows, hq, device=dev), 4 - shift, hq)
        c.attention(q2, gate=g2, out=out, m=m, z=z, **how)
        assert all(torch.equal(x, y) for x, y in zip((out, m, z), want)), shift
        assert torch.all(flat[:shift] == 7.0) and torch.all(flat[shift + rows * n :] == 7.0)
    assert ops.device_error() == 0


def test_tensors_on_another_stream(env):
    torch, _, dev = env
    lens = [200, 3]
    c = filled(env, ref.F16, 2, 128, 16, lens)
    fill(env, c, lens, 23)
    q = rows_of(torch, dev, 2, 8, 128, 24)
    want = c.attention(q, max_len=200)[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q2 = q * 1.0
        got = c.attention(q2, max_len=200)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


class Loop:
    """A serving loop over one cache: per step, one more position of `seqs` in every layer."""

    def __init__(self, env, fmt, window, sinks, seed):
        self.torch, pages, self.dev = env
        self.c = pages.PagedCache(fmt, 2, 128, 16, n_pages=120, max_seqs=8, max_pages=20, layers=2)
        self.c.pool.fill_(255)
        self.window, self.sinks = window, sinks
        self.gen = self.torch.Generator(device=self.dev).manual_seed(seed)
        self.seqs = ints(self.torch, [0, 2, 5], self.dev)
        self.q, self.k, self.v = (self.torch.zeros(3, 4 if i == 0 else 1, 256 if i else 128, device=self.dev).squeeze(1)
                                  for i in range(3))
        self.out = [self.torch.zeros(3, 4, 128, device=self.dev) for _ in range(2)]

    def new_rows(self):
        for t in (self.q, self.k, self.v):
            t.normal_(generator=self.gen)

    def prompt(self, counts):
        t, cu = self.torch, np.concatenate([[0], np.cumsum(counts)])
        n = int(cu[-1])
        cu = ints(t, cu, self.dev)
        self.c.extend(self.seqs, ints(t, counts, self.dev))
        got = []
        for layer in range(2):
            k, v = (t.randn(n, 256, generator=self.gen, device=self.dev) for _ in range(2))
            q = t.randn(n, 4, 128, generator=self.gen, device=self.dev)
            self.c.append(k, v, layer=layer, seqs=self.seqs, cu_rows=cu)
            got.append((q, self.c.attention(q, layer=layer, seqs=self.seqs, cu_rows=cu, max_rows=max(counts),
                                            window=self.window, sinks=self.sinks)))
        return got

    def step(self):
        self.c.extend(self.seqs)
        for layer in range(2):
            self.c.append(self.k, self.v, layer=layer, seqs=self.seqs)
            self.c.attention(self.q, layer=layer, seqs=self.seqs, max_len=320, window=self.window, sinks=self.sinks,
                             out=self.out[layer])


@pytest.mark.parametrize("fmt,window,sinks", [(ref.F16, 0, 0), (ref.BF16, 24, 2), (ref.Q8_ROW, 0, 0)])
def test_a_serving_loop(env, fmt, window, sinks):
    torch, _, dev = env
    a = Loop(env, fmt, window, sinks, 25)
    counts = [70, 1, 33]
    for layer, (q, got) in enumerate(a.prompt(counts)):
        want = want_rows(a.c, q, [(0, 0, 70), (2, 70, 1), (5, 71, 33)], layer=layer, window=window, sinks=sinks)
        ref.check_rows(got, want, "prompt")

    def check(what):
        for layer in range(2):
            want = want_rows(a.c, a.q, [(int(s), i, 1) for i, s in enumerate(a.seqs)], layer=layer, window=window,
                             sinks=sinks, missing_ok=True)
            err = np.abs(a.out[layer].cpu().double().numpy() - np.stack([w[0] for w in want]))
            assert np.all(err <= np.stack([(2 * w[3] * w[4])[:, None] for w in want])), (what, layer)

    for i in range(20):
        a.new_rows()
        a.step()
    check("steps")
    a.c.fork(ints(torch, [0, 0], dev), ints(torch, [1, 3], dev))   # two samples of sequence 0
    a.seqs.copy_(ints(torch, [1, 0, 3], dev))
    for i in range(3):
        a.new_rows()
        a.step()
        check("forked")
    if window:
        n = a.c.lengths
        every = ints(torch, [0, 1, 2, 3, 5], dev)
        a.c.free(every, torch.full_like(every, sinks), (n[every.long()] - window).clamp(min=0))
    a.c.free(ints(torch, [5], dev))
    used = a.c.compact()
    assert used.item() == int((a.c.refs > 0).sum()) and int(a.c.table.max()) < used.item()
    a.new_rows()
    a.step()
    check("closed up")
    assert ops.device_error() == 0


def test_a_captured_step_replays(env):
    torch, _, dev = env
    eager, graph = Loop(env, ref.F16, 0, 0, 26), Loop(env, ref.F16, 0, 0, 26)
    for x in (eager, graph):
        x.prompt([40, 7, 16])
        x.new_rows()
        x.step()   # (the first calls load the kernels)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        graph.step()
    for i in range(12):
        for x in (eager, graph):
            x.new_rows()
        eager.step()
        g.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(eager.out[layer], graph.out[layer]), (i, layer)
        for x, y in ((eager.c.table, graph.c.table), (eager.c.lengths, graph.c.lengths), (eager.c.refs, graph.c.refs)):
            assert torch.equal(x, y)
    assert ops.device_error() == 0


def test_two_captured_steps_of_one_cache(env):
    """Two graphs over one cache, each with its own workspace, replayed in turn."""
    torch, _, dev = env
    lens = [300, 77]
    c = filled(env, ref.BF16, 2, 128, 16, lens)
    fill(env, c, lens, 27)
    q = [rows_of(torch, dev, 2, 8, 128, 28 + i) for i in range(2)]
    want = [c.attention(x, max_len=300)[0].clone() for x in q]
    graphs, outs = [], []
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attention(x, max_len=300)[0])
        graphs.append(g)
    for i in range(4):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
        for o in outs:
            o.zero_()
