"""Attention over the paged history where the positions are cut into chunks and joined, against 64-bit
attention: chunk borders inside the list of first tokens and window, chunks that a row sees nothing of,
short sequences beside long ones."""
import numpy as np
import pytest

import paged_reference as ref
from rta import ops
from test_gpu_paged_attention import fill, rows_of, want_rows
from test_gpu_pages import env, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hq,hkv,hd,page", [(4, 1, 128, 64), (4, 2, 64, 7), (3, 1, 256, 33)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5), (1000, 300), (300, 2), (257, 0), (256, 300)])
@pytest.mark.parametrize("rows,length", [(3, 4000), (41, 1500), (130, 2100)])
def test_windows_cut_into_chunks(env, fmt, hq, hkv, hd, page, window, sinks, rows, length):
    torch, _, dev = env
    lens, counts = [40, length, 0, 300, length // 2], [7 if rows > 7 else 1, rows, 0, 2, 1]
    c = filled(env, fmt, hkv, hd, page, lens)
    fill(env, c, lens, 41)
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = rows_of(torch, dev, int(cu[-1]), hq, hd, 42)
    gate = rows_of(torch, dev, int(cu[-1]), hq, hd, 43).contiguous() if sinks else None
    how = dict(max_rows=rows, max_len=length, window=window, sinks=sinks)
    assert c.attention_workspace_bytes(hq, int(cu[-1]), 5, **how) > 0
    got = c.attention(q, cu_rows=ints(torch, cu, dev), gate=gate, **how)
    entries = [(s, int(cu[s]), counts[s]) for s in range(5)]
    ref.check_rows(got, want_rows(c, q, entries, window=window, sinks=sinks, gate=gate), (window, sinks, rows))
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.BF16, ref.Q8_ROW])
@pytest.mark.parametrize("hq,hkv,hd,page", [(4, 1, 128, 64), (20, 1, 64, 7), (3, 1, 256, 33)])
@pytest.mark.parametrize("window,sinks", [(700, 5), (1000, 300), (128, 1), (4000, 9)])
def test_single_windows_cut_into_chunks(env, fmt, hq, hkv, hd, page, window, sinks):
    torch, _, dev = env
    lens = [4100, 1, 699, 705, 129, 0, 1301, 2600]
    c = filled(env, fmt, hkv, hd, page, lens)
    fill(env, c, lens, 44)
    q = rows_of(torch, dev, 8, hq, hd, 45)
    how = dict(max_len=4100, window=window, sinks=sinks)
    assert c.attention_workspace_bytes(hq, 8, **how) > 0
    got = c.attention(q, **how)
    ref.check_rows(got, want_rows(c, q, [(s, s, 1) for s in range(8)], window=window, sinks=sinks))
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [ref.F16, ref.Q8_ROW])
def test_forked_sequences_listed_out_of_order(env, fmt):
    """A prompt's forks grow apart; drafts of all of them in one call, a sequence listed twice, with a gate."""
    torch, pages, dev = env
    c = pages.PagedCache(fmt, 2, 128, 16, n_pages=200, max_seqs=6, max_pages=60)
    gen = torch.Generator(device=dev).manual_seed(46)

    def grow(seqs, counts):
        n = sum(counts)
        cu = ints(torch, np.concatenate([[0], np.cumsum(counts)]), dev)
        c.extend(ints(torch, seqs, dev), ints(torch, counts, dev))
        k, v = (torch.randn(n, 256, generator=gen, device=dev) for _ in range(2))
        c.append(k, v, seqs=ints(torch, seqs, dev), cu_rows=cu)

    grow([3], [613])
    c.fork(ints(torch, [3, 3], dev), ints(torch, [0, 5], dev))
    grow([5, 3, 0], [4, 1, 70])
    seqs, counts = [5, 0, 3, 0], [4, 70, 1, 3]
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = rows_of(torch, dev, int(cu[-1]), 8, 128, 47)
    gate = rows_of(torch, dev, int(cu[-1]), 8, 128, 48).contiguous()
    got = c.attention(q, seqs=ints(torch, seqs, dev), cu_rows=ints(torch, cu, dev), max_rows=70, max_len=700, gate=gate)
    ref.check_rows(got, want_rows(c, q, [(s, int(cu[i]), counts[i]) for i, s in enumerate(seqs)], gate=gate))
    assert ops.device_error() == 0
