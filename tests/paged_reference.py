"""Plain 64-bit restatement of the paged history for the tests: the book as Python lists, the
pages decoded from their bytes, and attention row by row."""
import numpy as np
import torch

F16, BF16, Q8_ROW = 1, 30, 0x200
EPS = {F16: 2.0**-11, BF16: 2.0**-8}   # half a step, relative


def page_bytes(fmt, hkv, hd, page):
    n = 2 * hkv * page * (hd * (1 if fmt == Q8_ROW else 2) + (4 if fmt == Q8_ROW else 0))
    return -(-n // 128) * 128


class Book:
    """Tables, lengths and reference counts, call by call, as include/rta.h states them."""

    def __init__(self, page, n_pages, max_seqs, max_pages):
        self.page, self.max_pages = page, max_pages
        self.table = [[-1] * max_pages for _ in range(max_seqs)]
        self.lengths, self.refs = [0] * max_seqs, [0] * n_pages
        self.bad = False

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, seqs, add):
        """Returns the copied (from, to) pages."""
        seen, free = set(), [p for p, r in enumerate(self.refs) if r == 0]
        todo = []
        for i, (s, a) in enumerate(zip(seqs, add)):
            if not 0 <= s < len(self.lengths) or a < 0 or s in seen or \
                    self.lengths[s] + a > self.max_pages * self.page:
                self.bad = True
                seen.add(s)
                continue
            seen.add(s)
            e = self.lengths[s] // self.page
            tail = self.table[s][e] if a > 0 and self.lengths[s] % self.page else None
            todo.append((i, s, a, e, tail))
        holders = {}
        for i, s, a, e, tail in todo:
            if tail is not None and tail >= 0 and self.refs[tail] > 1:
                holders.setdefault(tail, []).append(i)
        refs, pairs, out = list(self.refs), [], False
        for i, s, a, e, tail in todo:
            old, new = self.pages(self.lengths[s]), self.pages(self.lengths[s] + a)
            kind = 0
            if tail is not None and tail < 0:
                kind = 2
            elif tail is not None and refs[tail] > 1 and not (len(holders[tail]) == refs[tail] and holders[tail][-1] == i):
                kind = 1
            need = new - old + (kind > 0)
            if out or need > len(free):
                out = self.bad = True
                continue
            if kind:
                p = free.pop(0)
                self.table[s][e] = p
                self.refs[p] = 1
                if kind == 1:
                    self.refs[tail] -= 1
                    pairs.append((tail, p))
            for j in range(old, new):
                p = free.pop(0)
                self.table[s][j] = p
                self.refs[p] = 1
            self.lengths[s] += a
        return pairs

    def fork(self, src, dst):
        lengths = list(self.lengths)
        for i, (s, d) in enumerate(zip(src, dst)):
            n = len(lengths)
            if not (0 <= s < n and 0 <= d < n) or d in dst[:i] or d in src or lengths[d]:
                self.bad = True
                continue
            for e in range(self.pages(lengths[s])):
                self.table[d][e] = p = self.table[s][e]
                if p >= 0:
                    self.refs[p] += 1
            self.lengths[d] = lengths[s]

    def free(self, seqs, first=None, last=None):
        for i, s in enumerate(seqs):
            lo = first[i] if first else 0
            if not 0 <= s < len(self.lengths) or s in seqs[:i] or lo < 0:
                self.bad = True
                continue
            n = self.lengths[s]
            hi = last[i] if last else n
            for e in range(self.pages(n)):
                if e * self.page >= lo and min((e + 1) * self.page, n) <= hi:
                    p, self.table[s][e] = self.table[s][e], -1
                    if p >= 0:
                        self.refs[p] -= 1
            if hi >= n and lo < n:
                self.lengths[s] = lo

    def compact(self):
        """Returns (used pages, [(from, to)])."""
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] <= 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return used, list(to.items())

    def check(self, cache):
        assert cache.lengths.tolist() == self.lengths
        assert cache.refs.tolist() == self.refs
        assert cache.table.tolist() == self.table


def decode(fmt, hkv, hd, page, raw):
    """[..., 2, kv heads, page, hd] float64 of page bytes [..., page_bytes] (a CPU tensor)."""
    rows = 2 * hkv * page
    lead = raw.shape[:-1]
    if fmt == Q8_ROW:
        x = raw[..., : rows * hd].contiguous().view(torch.int8).double().view(*lead, 2, hkv, page, hd)
        s = raw[..., rows * hd : rows * (hd + 4)].contiguous().view(torch.float32).double()
        return x * s.view(*lead, 2, hkv, page, 1)
    t = torch.float16 if fmt == F16 else torch.bfloat16
    return raw[..., : 2 * rows * hd].contiguous().view(t).double().view(*lead, 2, hkv, page, hd)


def dense(cache, layer, s, missing_ok=False):
    """(k, v, held) of sequence s: float64 [len, kv heads, hd] from the pool's bytes, and which
    positions have a page."""
    n = int(cache.lengths[s])
    names = cache.table[s, : -(-n // cache.page)].cpu().long()
    have = (names >= 0) & (names < cache.pool.shape[1])
    assert missing_ok or bool(have.all())
    raw = cache.pool[layer][names.clamp(0, cache.pool.shape[1] - 1).to(cache.device)].cpu()
    x = decode(cache.fmt, cache.kv_heads, cache.head_dim, cache.page, raw)   # [pages, 2, kv, page, hd]
    x = x.permute(1, 0, 3, 2, 4).reshape(2, -1, cache.kv_heads, cache.head_dim)[:, :n]
    held = have.repeat_interleave(cache.page)[:n]
    return x[0].numpy(), x[1].numpy(), held.numpy()


def attend(q, k, v, held, t, window=0, sinks=0, gate=None):
    """One row q [hq, hd] at position t: (out, m, z, bound), float64.  bound: how far an fp32
    result may be off per head, relative to max|v|: roundings of the products and sums of a score
    (sqrt(hd) of them, each 2^-24 of sum|q k|, twice for the split of q), of the weights' sums
    (sqrt(count)) and of exp and the final scaling (2^-21), four times their random walk."""
    hq, hd = q.shape
    G = hq // k.shape[1]
    p = np.arange(len(k))
    see = (p <= t) & held
    if window:
        see &= (p > t - window) | (p < sinks)
    out, m, z = np.zeros((hq, hd)), np.full(hq, -np.inf), np.zeros(hq)
    bound, top = np.zeros(hq), np.zeros(hq)
    n = int(see.sum())
    if n:
        for h in range(hq):
            kk, vv = k[see, h // G], v[see, h // G]
            s = kk @ q[h] / np.sqrt(hd)
            m[h] = s.max()
            w = np.exp(s - m[h])
            z[h] = w.sum()
            out[h] = w @ vv / z[h]
            most = (np.abs(kk) @ np.abs(q[h])).max() / np.sqrt(hd)
            bound[h] = 4 * (2 * np.sqrt(hd) * 2.0**-24 * most + np.sqrt(n) * 2.0**-24 + 2.0**-21)
            top[h] = np.abs(vv).max()
    if gate is not None:
        out /= 1 + np.exp(-gate)
    return out, m, z, bound, top


def check_rows(got, want, what=""):
    """(out, m, z) tensors of rows against a list of attend() results."""
    o, m, z = (t.cpu().double().numpy() for t in got)
    off = total = 0.0
    for r, (wo, wm, wz, bound, top) in enumerate(want):
        seen = np.isfinite(wm)
        assert np.array_equal(np.isfinite(m[r]), seen), (what, r, m[r])
        assert not z[r][~seen].any() and not o[r][~seen].any(), (what, r)
        assert np.all(np.abs(m[r][seen] - wm[seen]) <= bound[seen]), (what, r)
        assert np.all(np.abs(z[r] - wz) <= (bound + 2.0**-21) * wz), (what, r)
        err = np.abs(o[r] - wo)
        assert np.all(err <= (2 * bound * top)[:, None]), (what, r, float((err - (2 * bound * top)[:, None]).max()))
        off += float((err**2).sum())
        total += float((wo**2).sum())
    # fp32 results: as a whole within 1e-5, far below what one position too many or too few changes
    assert off**0.5 <= 1e-5 * total**0.5 + 1e-30, (what, (off / max(total, 1e-300)) ** 0.5)
