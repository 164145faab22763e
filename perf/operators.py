"""The paged history's operators as cases that can be timed and compared.

A paged history keeps the keys and values of many sequences in pages of `page` positions, each
sequence's pages named by its row of a table.  Kinds of case (sizes are those of the library's
own benchmark and tests, or generic):
  decode   attention of one new token per sequence over its pages, whole or through a sliding
           window with a few first tokens (sinks) that stay visible
  prompt   attention of several new rows per sequence (prompts, chunks of prompts, drafted
           tokens) over its pages, causal, with the same window and sinks
  append   the new rows' keys and values written into the pages, and read back
  fork     a round of sampling: last round's samples are freed, each parent is forked and every
           sequence takes one more position, which copies the pages that are shared
  compact  the used pages moved to the front of the pool

`own` chooses between the plain form (elementary torch operations) and the library's calls.
A page is [key, value][kv head][position][head_dim], with for q8 the fp32 scales
[key, value][kv head][position] behind the codes, rounded up to 128 bytes.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
LAST = 2**31 - 1
ELEMENT = {"f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}


def listed():
    return [
        # the smallest call: one short conversation, where the launch is all that counts
        decode("decode_f16_1seq", "f16", 1, 32, 8, 128, 16, 300, 300),
        # a continuous batch of ragged conversations, grouped heads
        decode("decode_bf16_32seq", "bf16", 32, 32, 8, 128, 64, 256, 8192),
        # a few very long documents, 8-bit rows: the largest history
        decode("decode_q8_long", "q8", 8, 32, 8, 128, 128, 60000, 131072),
        # endless streams of 64-wide heads that see their last 4096 tokens and the first 4
        decode("decode_f16_window", "f16", 64, 16, 4, 64, 32, 1, 40000, 4096, 4),
        # drafted tokens checked by the model: 5 rows each against long histories
        prompt("prompt_q8_draft5", "q8", 16, 32, 8, 128, 64, 500, 16384, 5, 5),
        # a prompt from nothing, the whole triangle
        prompt("prompt_bf16_4096", "bf16", 1, 32, 8, 128, 128, 0, 0, 4096, 4096),
        # chunks of streamed prompts behind a window, odd lengths
        prompt("prompt_f16_window", "f16", 4, 16, 4, 128, 64, 37, 6000, 701, 2048, 1024, 4),
        # the new keys and values of a decode batch
        append("append_f16_32rows", "f16", 32, 8, 128, 64, 256, 8192, 1, 1),
        # those of a few long prompts, into 8-bit rows
        append("append_q8_prompts", "q8", 4, 8, 128, 128, 0, 333, 1111, 4096),
        # 4 prompts sampled 3 times each, small pages
        fork("fork_bf16_4x3", "bf16", 4, 3, 8, 128, 16, 4, 100, 2000),
        # 16 prompts sampled 7 times each, large pages of 8 layers
        fork("fork_f16_16x7", "f16", 16, 7, 8, 128, 128, 8, 500, 8192),
        # half of 96 conversations have ended: the pool is closed up
        compact("compact_bf16_96", "bf16", 96, 8, 128, 64, 8, 100, 4096),
    ]


def _case(name, **c):
    return dict(c, name=name) if name else c


def decode(name, fmt, nseq, hq, hkv, hd, page, lo, hi, window=0, sinks=0):
    return _case(name, kind="decode", fmt=fmt, nseq=nseq, hq=hq, hkv=hkv, hd=hd, page=page, lo=lo, hi=hi,
                 window=window, sinks=sinks)


def prompt(name, fmt, nseq, hq, hkv, hd, page, lo, hi, rows_lo, rows_hi, window=0, sinks=0):
    return _case(name, kind="prompt", fmt=fmt, nseq=nseq, hq=hq, hkv=hkv, hd=hd, page=page, lo=lo, hi=hi,
                 rows_lo=rows_lo, rows_hi=rows_hi, window=window, sinks=sinks)


def append(name, fmt, nseq, hkv, hd, page, lo, hi, rows_lo, rows_hi):
    return _case(name, kind="append", fmt=fmt, nseq=nseq, hkv=hkv, hd=hd, page=page, lo=lo, hi=hi,
                 rows_lo=rows_lo, rows_hi=rows_hi)


def fork(name, fmt, parents, kids, hkv, hd, page, layers, lo, hi):
    return _case(name, kind="fork", fmt=fmt, nseq=parents * (1 + kids), parents=parents, hkv=hkv, hd=hd, page=page,
                 layers=layers, lo=lo, hi=hi)


def compact(name, fmt, nseq, hkv, hd, page, layers, lo, hi):
    return _case(name, kind="compact", fmt=fmt, nseq=nseq, hkv=hkv, hd=hd, page=page, layers=layers, lo=lo, hi=hi)


# ------------------------------------------------------------------ drawn cases ----
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "append", "fork", "compact"])
    fmt = rng.choice(["f16", "bf16", "q8"])
    hq, hkv = rng.choice([(32, 8), (16, 4), (8, 8), (24, 6), (16, 2), (16, 1), (4, 4), (20, 4), (12, 1)])
    hd = rng.choice([64, 128, 128, 128, 256])
    page = rng.choice([1, 8, 16, 24, 32, 64, 100, 128, 256])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 4096), rng.choice([0, 1, 4, 16, 100]))])
    if kind == "decode":
        nseq = _log_int(rng, 1, 128)
        hi = _log_int(rng, 2, min(131072, 330000000 // (hkv * hd * nseq)))   # at most 1.3 GB of history
        return decode(None, fmt, nseq, hq, hkv, hd, page, max(1, hi // rng.choice([1, 3, 50])), hi, window, sinks)
    if kind == "prompt":
        pairs = 32000000000 // (hq * hd)   # rows x positions of at most 128 GFLOP
        rows = _log_int(rng, 2, 2048)
        nseq = _log_int(rng, 1, max(1, min(32, 4096 // rows, pairs // (2 * rows * rows))))
        hi = _log_int(rng, 1, max(1, min(16384, pairs // (rows * nseq) - rows)))
        return prompt(None, fmt, nseq, hq, hkv, hd, page, hi // rng.choice([1, 4, 100]), hi,
                      max(1, rows // rng.choice([1, 3, 40])), rows, window, sinks)
    if kind == "append":
        rows = rng.choice([1, _log_int(rng, 1, 2048)])
        nseq = _log_int(rng, 1, max(1, min(128, 8192 // rows)))
        hi = _log_int(rng, 1, 4096)
        return append(None, fmt, nseq, hkv, hd, page, hi // rng.choice([1, 3, 50]), hi, max(1, rows // 3), rows)
    fmt = rng.choice(["f16", "bf16"])
    hkv = min(hkv, 8)
    page = max(page, 8)
    if kind == "fork":
        parents = _log_int(rng, 1, 12)
        hi = _log_int(rng, 2, 4096)
        return fork(None, fmt, parents, _log_int(rng, 1, 7), hkv, min(hd, 128), page, rng.choice([1, 3, 8]),
                    max(1, hi // rng.choice([1, 4, 50])), hi)
    hi = _log_int(rng, 2, 4096)
    return compact(None, fmt, _log_int(rng, 2, 64), hkv, min(hd, 128), page, rng.choice([1, 3, 8]),
                   max(1, hi // rng.choice([1, 4, 50])), hi)


# ------------------------------------------------------------------ sizes of a case ----
def _spread(n, lo, hi, phase):
    """n whole numbers from lo to hi (both there), spread over the logarithm, in no order."""
    if n == 1 or lo == hi:
        return [hi] * n
    at = [(i * 0.6180339887 + phase) % 1.0 for i in range(n)]
    rank = sorted(range(n), key=lambda i: at[i])
    got = [0] * n
    for k, i in enumerate(rank):
        got[i] = int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * k / (n - 1)))) - 1
    return got


def _sizes(c):
    """(positions before the new rows, new rows) of each sequence."""
    n = c["nseq"]
    if c["kind"] == "fork":
        p = c["parents"]
        return _spread(p, c["lo"], c["hi"], 0.3) + [0] * (n - p), [0] * n
    old = _spread(n, c["lo"], c["hi"], 0.3)
    new = [0] * n
    if c["kind"] == "decode":   # the newest of the positions is the query's
        old, new = [x - 1 for x in old], [1] * n
    elif "rows_hi" in c:
        new = _spread(n, c["rows_lo"], c["rows_hi"], 0.8)
    return old, new


def _visible(length, window, sinks):
    if window <= 0 or length <= window:
        return length
    return window + min(sinks, length - window)


def _row_bytes(c):
    """Bytes of one position's keys and values."""
    return 2 * c["hkv"] * (c["hd"] * (1 if c["fmt"] == "q8" else 2) + (4 if c["fmt"] == "q8" else 0))


def _page_bytes(c):
    return (_row_bytes(c) * c["page"] + 127) // 128 * 128


def _pages(length, page):
    return (length + page - 1) // page


def work(c):
    old, new = _sizes(c)
    if c["kind"] in ("decode", "prompt"):
        rows, hq, hd = sum(new), c["hq"], c["hd"]
        pairs = read = 0
        for o, r in zip(old, new):
            pairs += sum(_visible(o + i + 1, c["window"], c["sinks"]) for i in range(r))
            # positions that any of the rows sees: the sinks and all from the first row's window on
            first = o + 1 - c["window"] if c["window"] > 0 else 0
            read += o + r - max(0, first) + min(c["sinks"], max(0, first)) if c["window"] > 0 else o + r
        return {"bytes": read * _row_bytes(c) + 8 * rows * hq * (hd + 1), "flops": 4 * pairs * hq * hd}
    if c["kind"] == "append":
        rows, width = sum(new), 2 * c["hkv"] * c["hd"]
        return {"bytes": rows * (8 * width + 2 * _row_bytes(c)), "flops": 4 * rows * width}
    if c["kind"] == "fork":
        kids = c["nseq"] // c["parents"] - 1
        # a parent whose last page is not full: every sample of it copies that page
        copies = sum(kids for x in old[: c["parents"]] if x % c["page"])
        names = 4 * sum((1 + kids) * _pages(x + 1, c["page"]) for x in old[: c["parents"]])
        return {"bytes": 2 * copies * c["layers"] * _page_bytes(c) + 3 * names, "flops": 0}
    held = [_pages(x, c["page"]) for x in old]
    live = sum(held[1::2])
    # on the mean the share of the live pages that lies past their number
    moved = live * (1 - live / max(1, sum(held)))
    return {"bytes": 2 * moved * c["layers"] * _page_bytes(c) + 12 * sum(held), "flops": 0}


# ------------------------------------------------------------------ what the caller holds ----
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    old, new = _sizes(c)
    total = [o + r for o, r in zip(old, new)]
    n, page, layers = c["nseq"], c["page"], c.get("layers", 1)
    held = [_pages(x, page) for x in total]
    n_pages = sum(held) + 3 + (2 * n if c["kind"] == "fork" else 0)
    max_pages = max(held) + 2
    pb = _page_bytes(c)
    pool = _random_pool(c, layers * n_pages, gen).view(layers, n_pages, pb)
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((n, max_pages), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    at = 0
    for s in range(n):
        table[s, : held[s]] = order[at : at + held[s]]
        at += held[s]
    refs[order[:at].long()] = 1
    st = {"case": c, "pool": pool, "table": table, "refs": refs,
          "lengths": torch.tensor(total, dtype=torch.int32, device=DEV), "max_len": max(total)}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    if c["kind"] in ("prompt", "append"):
        cu = [0]
        for r in new:
            cu.append(cu[-1] + r)
        st["cu"] = ints(cu) if max(new) > 1 else None
        st["max_rows"] = max(new)
    rows = sum(new)
    if c["kind"] in ("decode", "prompt"):
        st["q"] = 1.5 * torch.randn(rows, c["hq"], c["hd"], generator=gen, device=DEV)
    elif c["kind"] == "append":
        width = c["hkv"] * c["hd"]
        st["k"] = 2.0 * torch.randn(rows, width, generator=gen, device=DEV)
        st["v"] = torch.randn(rows, width, generator=gen, device=DEV)
    elif c["kind"] == "fork":
        p = c["parents"]
        kids, sires = list(range(p, n)), list(range(p))
        each = n // p - 1
        st["every"] = ints(kids + sires)
        st["first"] = ints([0] * len(kids) + old[:p])
        st["last"] = ints([LAST] * n)
        st["src"], st["dst"] = ints([s for s in sires for _ in range(each)]), ints(kids)
        st["one"] = ints([1] * n)
    else:   # every other sequence has ended
        gone = table[0::2].clone()
        refs[gone[gone >= 0].long()] = 0
        table[0::2] = -1
        st["lengths"][0::2] = 0
        st["table0"], st["refs0"] = table.clone(), refs.clone()
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "ray-tracing-attention_amd"))
        from rta import _lib, pages
        fmt = {"f16": _lib.F16, "bf16": _lib.BF16, "q8": _lib.Q8_ROW}[c["fmt"]]
        st["cache"] = pages.PagedCache(fmt, c["hkv"], c["hd"], page, pool=pool, table=table, lengths=st["lengths"],
                                       refs=refs)
    return st


def _random_pool(c, count, gen):
    """Pages of N(0, 1) values (q8: codes up to the largest and scales to match)."""
    pb = _page_bytes(c)
    if c["fmt"] != "q8":
        return torch.randn(count * pb // 2, generator=gen, device=DEV, dtype=torch.float32).to(ELEMENT[c["fmt"]]).view(
            torch.uint8)
    raw = torch.randint(-(2**31), 2**31, (count * pb // 4,), dtype=torch.int32, generator=gen, device=DEV)
    raw = raw.view(torch.int8).clamp_(-127, 127).view(torch.uint8).view(count, pb)
    rows = 2 * c["hkv"] * c["page"]
    scales = (0.5 + torch.rand(count, rows, generator=gen, device=DEV)) / 73.0   # uniform codes: 73 on the root mean square
    raw[:, rows * c["hd"] : rows * (c["hd"] + 4)] = scales.view(torch.uint8)
    raw[:, rows * (c["hd"] + 4) :] = 0
    return raw.view(-1)


# ------------------------------------------------------------------ one pass ----
def run(st):
    return (_run_own if own else _run_plain)[st["case"]["kind"]](st)


def _own_decode(st):
    c = st["case"]
    out, m, z = st["cache"].attention(st["q"], window=c["window"], sinks=c["sinks"], max_len=st["max_len"])
    return {"out": out, "m": m, "z": z}


def _own_prompt(st):
    c = st["case"]
    out, m, z = st["cache"].attention(st["q"], cu_rows=st["cu"], max_rows=st["max_rows"], window=c["window"],
                                      sinks=c["sinks"], max_len=st["max_len"])
    return {"out": out, "m": m, "z": z}


def _own_append(st):
    st["cache"].append(st["k"], st["v"], cu_rows=st["cu"])
    k, v = st["cache"].read(st["k"].shape[0], cu_rows=st["cu"])
    return {"k": k, "v": v}


def _own_fork(st):
    cache = st["cache"]
    cache.free(st["every"], st["first"], st["last"])
    cache.fork(st["src"], st["dst"])
    cache.extend(st["every"], st["one"])
    return _book(st)


def _own_compact(st):
    _fragmented(st)
    used = st["cache"].compact()
    return dict(_book(st), used=used)


_run_own = {"decode": _own_decode, "prompt": _own_prompt, "append": _own_append, "fork": _own_fork,
            "compact": _own_compact}


def _book(st):
    """The table, the lengths, the references and every layer's pages (all of them the state's own)."""
    return {"table": st["table"], "lengths": st["lengths"], "refs": st["refs"],
            "pages": st["pool"].view(ELEMENT[st["case"]["fmt"]])}


def _fragmented(st):
    """The table and references as they were before a pass closed the pool up (what lies in the
    pages it moved from is still there), so that every pass has the same work."""
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])


# ---- the plain forms ----
def _rows_of(st):
    """(sequence, position) of each new row."""
    lengths = st["lengths"].long()
    if st.get("cu") is None:
        return torch.arange(len(lengths), device=DEV), lengths - 1
    cu = st["cu"].long()
    rows = (st["q"] if "q" in st else st["k"]).shape[0]
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:], r, right=True)
    return seq, lengths[seq] - cu[seq + 1] + r


def _views(c, pool):
    """One layer's elements [pages, 2, kv heads, page, head_dim] and (q8) scales [pages, 2, kv heads, page]."""
    rows = 2 * c["hkv"] * c["page"]
    size = rows * c["hd"] * (1 if c["fmt"] == "q8" else 2)
    e = pool[:, :size].view(ELEMENT[c["fmt"]]).unflatten(1, (2, c["hkv"], c["page"], c["hd"]))
    if c["fmt"] != "q8":
        return e, None
    return e, pool[:, size : size + 4 * rows].view(torch.float32).unflatten(1, (2, c["hkv"], c["page"]))


def _gather(c, pool, page, off, which):
    """fp32 values of `which` (0 key, 1 value) at (page, off): [..., kv heads, head_dim]."""
    e, scale = _views(c, pool)
    got = e[page, which, :, off].float()
    return got if scale is None else got * scale[page, which, :, off].unsqueeze(-1)


def _attend(st, q, pos, row_ok):
    """q [n, R, hq, hd] at positions pos [n, R] of sequence n, fp32: (out, m, z) of each row."""
    c = st["case"]
    n, R, hq, hd = q.shape
    hkv, window, sinks = c["hkv"], c["window"], c["sinks"]
    last = pos.amax(1)
    lo = ((pos.clamp(min=0) - window + 1).amin(1) if window > 0 else torch.zeros_like(last)).clamp(min=0)   # the first row's window
    head = torch.minimum(lo, torch.full_like(lo, sinks))
    most = st["max_len"] if window <= 0 else min(st["max_len"], window + R - 1 + sinks)
    j = torch.arange(most, device=DEV)
    p = torch.where(j < head[:, None], j, j + (lo - head)[:, None])
    held = p <= last[:, None]
    p = p.clamp(max=st["max_len"] - 1)
    page = st["table"].gather(1, p // c["page"]).long().clamp(min=0)
    off = p % c["page"]
    k = _gather(c, st["pool"][0], page, off, 0).permute(0, 2, 3, 1)   # [n, kv heads, hd, positions]
    v = _gather(c, st["pool"][0], page, off, 1).permute(0, 2, 1, 3)
    qg = q.view(n, R, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, hd)
    s = torch.matmul(qg, k.contiguous()).view(n, hkv, hq // hkv, R, most) / math.sqrt(hd)
    see = held[:, None] & (p[:, None] <= pos[:, :, None]) & row_ok[:, :, None]
    if window > 0:
        see &= (p[:, None] > pos[:, :, None] - window) | (p[:, None] < sinks)
    s = s.masked_fill_(~see[:, None, None], -math.inf)
    m = s.amax(-1)
    w = s.sub_(m.masked_fill(m == -math.inf, 0.0).unsqueeze(-1)).exp_()
    z = w.sum(-1)
    o = torch.matmul(w.view(n, hkv, -1, most), v.contiguous()).view(n, hkv, hq // hkv, R, hd)
    o = o / z.masked_fill(z == 0, 1.0).unsqueeze(-1)
    back = lambda t: t.permute(0, 3, 1, 2, *range(4, t.dim())).reshape(n, R, hq, *t.shape[4:])  # noqa: E731
    return back(o), back(m), back(z)


def _plain_decode(st):
    pos = st["lengths"].long()[:, None] - 1
    out, m, z = _attend(st, st["q"][:, None], pos, pos >= 0)
    return {"out": out[:, 0], "m": m[:, 0], "z": z[:, 0]}


def _plain_prompt(st):
    n, R = st["case"]["nseq"], st["max_rows"]
    if st["cu"] is None:
        return _plain_decode(st)
    cu = st["cu"].long()
    count = cu[1:] - cu[:-1]
    r = torch.arange(R, device=DEV)
    ok = r < count[:, None]
    q = st["q"][(cu[:-1, None] + r).clamp(max=st["q"].shape[0] - 1)]
    pos = torch.where(ok, st["lengths"].long()[:, None] - count[:, None] + r, st["lengths"].long()[:, None] - 1)
    out, m, z = _attend(st, q, pos, ok)
    seq, _ = _rows_of(st)
    at = torch.arange(st["q"].shape[0], device=DEV) - cu[seq]
    return {"out": out[seq, at], "m": m[seq, at], "z": z[seq, at]}


def _plain_append(st):
    c = st["case"]
    seq, pos = _rows_of(st)
    page, off = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    e, scale = _views(c, st["pool"][0])
    got = []
    for which, x in enumerate((st["k"], st["v"])):   # keys, values
        x = x.view(-1, c["hkv"], c["hd"])
        if scale is None:
            e[page, which, :, off] = x.to(e.dtype)
        else:
            d = x.abs().amax(-1) / 127.0
            e[page, which, :, off] = (x / torch.where(d > 0, d, 1.0).unsqueeze(-1)).round().to(torch.int8)
            scale[page, which, :, off] = d
        got.append(_gather(c, st["pool"][0], page, off, which).view(-1, c["hkv"] * c["hd"]))
    return {"k": got[0], "v": got[1]}


def _plain_free(st, seqs, first, last):
    page = st["case"]["page"]
    length, rows = st["lengths"][seqs], st["table"][seqs]
    at = torch.arange(rows.shape[1], device=DEV, dtype=torch.int32) * page
    end = torch.minimum(at + page, length[:, None])
    drop = (at < length[:, None]) & (at >= first[:, None]) & (end <= last[:, None])
    gone = (drop & (rows >= 0)).to(torch.int32)
    st["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), -gone.flatten())
    st["table"][seqs] = torch.where(drop, -1, rows)
    st["lengths"][seqs] = torch.where(last >= length, torch.minimum(first, length), length)


def _plain_fork_step(st, src, dst):
    page = st["case"]["page"]
    length, rows = st["lengths"][src], st["table"][src]
    at = torch.arange(rows.shape[1], device=DEV, dtype=torch.int32) * page
    rows = torch.where(at < length[:, None], rows, -1)
    st["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().to(torch.int32))
    st["table"][dst] = rows
    st["lengths"][dst] = length


def _plain_extend(st, seqs, add):
    page, refs = st["case"]["page"], st["refs"]
    length, rows, n = st["lengths"][seqs], st["table"][seqs], len(seqs)
    i = torch.arange(n, device=DEV, dtype=torch.int32)
    before, after = (length + page - 1) // page, (length + add + page - 1) // page
    tail = rows.gather(1, (length // page).long()[:, None])[:, 0].clamp(min=0).long()
    shared = (length % page > 0) & (add > 0) & (refs[tail] > 1)
    # of the listed sequences that share a page nobody else holds, the last one keeps it
    holders = torch.zeros_like(refs).index_add_(0, tail, shared.to(torch.int32))
    keeper = torch.full_like(refs, -1).scatter_reduce_(0, tail, torch.where(shared, i, -1), "amax")
    move = shared & ~((holders[tail] == refs[tail]) & (keeper[tail] == i))
    need = after - before + move.to(torch.int32)
    upto = need.cumsum(0)
    free = torch.sort((refs > 0).to(torch.int32), stable=True).indices   # free pages, lowest first
    begin = (upto - need)[:, None] + move.to(torch.int32)[:, None]
    e = torch.arange(rows.shape[1], device=DEV, dtype=torch.int32)
    fresh = (e >= before[:, None]) & (e < after[:, None])
    named = free[(begin + e - before[:, None]).clamp(0, len(refs) - 1)].to(torch.int32)
    rows = torch.where(fresh, named, rows)
    who = move.nonzero()[:, 0]
    to, source = free[(upto - need)[who]], tail[who]
    rows[who, (length // page)[who].long()] = to.to(torch.int32)
    st["pool"][:, to] = st["pool"][:, source]
    refs.index_add_(0, source, torch.full_like(source, -1, dtype=torch.int32))
    refs[to] = 1
    refs.index_add_(0, torch.where(fresh, named, 0).flatten().long(), fresh.flatten().to(torch.int32))
    st["table"][seqs] = rows
    st["lengths"][seqs] = length + add


def _plain_fork(st):
    every = st["every"].long()
    _plain_free(st, every, st["first"], st["last"])
    _plain_fork_step(st, st["src"].long(), st["dst"].long())
    _plain_extend(st, every, st["one"])
    return _book(st)


def _plain_compact(st):
    _fragmented(st)
    refs, table, pool = st["refs"], st["table"], st["pool"]
    used = refs > 0
    count = used.sum()
    at = torch.arange(len(refs), device=DEV)
    moved = used & (at >= count)
    holes = torch.sort((used | (at >= count)).to(torch.int32), stable=True).indices
    to = torch.where(moved, holes[(moved.cumsum(0) - 1).clamp(min=0)], at)
    who = moved.nonzero()[:, 0]
    pool[:, to[who]] = pool[:, who]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1))
    left = torch.where(moved, 0, refs)
    refs.copy_(left.index_add_(0, to, torch.where(moved, refs, 0)))
    return dict(_book(st), used=count.to(torch.int32).view(1))


_run_plain = {"decode": _plain_decode, "prompt": _plain_prompt, "append": _plain_append, "fork": _plain_fork,
              "compact": _plain_compact}


# ------------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    """Attention in 64 bits, a sequence and a kv head at a time; None for what is only moved or stored."""
    if case["kind"] not in ("decode", "prompt"):
        return None
    c = dict(case)
    st = prepare(c, seed)
    old, new = _sizes(c)
    hq, hkv, hd, page, window, sinks = (c[x] for x in ("hq", "hkv", "hd", "page", "window", "sinks"))
    rows, per = sum(new), hkv * page * hd
    out = torch.zeros(rows, hq, hd, dtype=torch.float64, device=DEV)
    m = torch.full((rows, hq), -math.inf, dtype=torch.float64, device=DEV)
    z = torch.zeros(rows, hq, dtype=torch.float64, device=DEV)
    at = 0
    for s, (o, r) in enumerate(zip(old, new)):
        length = o + r
        q = st["q"][at : at + r].double()
        if length:
            names = st["table"][s, : _pages(length, page)].long()
            raw = st["pool"][0][names]
            for h in range(hkv):
                kv = []
                for which in (0, 1):
                    first = (which * hkv + h) * page
                    if c["fmt"] == "q8":
                        code = raw[:, first * hd : (first + page) * hd].contiguous().view(torch.int8).double()
                        base = 2 * per + 4 * first
                        d = raw[:, base : base + 4 * page].contiguous().view(torch.float32).double()
                        x = code.view(-1, page, hd) * d.view(-1, page, 1)
                    else:
                        x = raw[:, 2 * first * hd : 2 * (first + page) * hd].contiguous().view(ELEMENT[c["fmt"]]).double()
                    kv.append(x.reshape(-1, hd)[:length])
                G = hq // hkv
                p = torch.arange(length, device=DEV)
                for lo in range(0, r, 512):   # rows in pieces, so that the scores fit
                    t = torch.arange(o + lo, o + min(r, lo + 512), device=DEV)
                    see = p[None] <= t[:, None]
                    if window > 0:
                        see = see & ((p[None] > t[:, None] - window) | (p[None] < sinks))
                    for g in range(h * G, (h + 1) * G):
                        x = q[lo : lo + 512, g] @ kv[0].t() * hd**-0.5
                        x = torch.where(see, x, -math.inf)
                        top = x.amax(1)
                        e = torch.exp(x - top[:, None])
                        total = e.sum(1)
                        a = at + lo
                        out[a : a + len(t), g] = e @ kv[1] / total[:, None]
                        m[a : a + len(t), g] = top
                        z[a : a + len(t), g] = total
        at += r
    return {"out": out, "m": m, "z": z}
