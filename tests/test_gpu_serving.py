"""A serving loop of the operators around the paged history, as a program runs them: embed, project, turn and
append, attend, read the vocabulary out, sample, and on with the new tokens; prompts of ragged lengths, forked
samples and ended sequences.  Every stage against its 64-bit restatement on the inputs that it had, and the same
loop captured in a graph against the eager one."""
import numpy as np
import pytest

import paged_q4_reference as q4
import paged_reference as ref
import rotary_reference
import sample_reference
from rta import _lib, ops, rotary
from test_gpu_pages import env, ints  # noqa: F401

pytestmark = pytest.mark.gpu
HQ, HKV, HD, VOCAB, SEQS = 6, 2, 64, 700, 6


@pytest.fixture(autouse=True)
def knows_q4(monkeypatch):
    monkeypatch.setattr(ref, "decode", q4.decode)


class Server:
    """One layer of a model with random weights, and its cache."""

    def __init__(self, env, fmt, layout, window=0, sinks=0):
        self.torch, pages, self.dev = env
        t, rng = self.torch, np.random.default_rng(1)
        w = lambda *s: t.tensor(rng.standard_normal(s) / np.sqrt(s[-1]), dtype=t.float32, device=self.dev)  # noqa: E731
        self.hidden = HQ * HD
        self.table = w(VOCAB, self.hidden) * np.sqrt(self.hidden).item()
        self.wq, self.wk, self.wv = w(HQ * HD, self.hidden), w(HKV * HD, self.hidden), w(HKV * HD, self.hidden)
        self.wo = 4 * w(VOCAB, HQ * HD)
        self.cache = pages.PagedCache(fmt, HKV, HD, 16, n_pages=80, max_seqs=SEQS, max_pages=16)
        self.cache.pool.fill_(255)
        self.rotary = rotary.Rotary(HD, 48, layout, theta=1e4, scaling="ramp", factor=8.0, original=64)
        self.how = dict(window=window, sinks=sinks)
        n = SEQS
        self.tokens = t.zeros(n, dtype=t.int32, device=self.dev)
        self.u = t.zeros(n, device=self.dev)
        self.rules = dict(temperature=t.tensor([0.0, 0.7, 1.0, 1.3, 1.0, 0.9], device=self.dev),
                          top_k=ints(t, [0, 50, 0, 7, 3, 0], self.dev), top_p=t.tensor([1, 0.9, 0.95, 1, 0.5, 1.0], device=self.dev),
                          min_p=t.tensor([0, 0, 0.02, 0, 0, 0.1], device=self.dev))
        self.seen = {}

    def project(self, w, x):
        return ops.gemv(_lib.F32, w, w.shape[0], w.shape[1], x)

    def rows(self, ids, n, seqs, cu, max_rows):
        """The layer's rows of new tokens: logits [rows, vocab]."""
        s = self.seen
        s["x"] = ops.embed(_lib.F32, self.table, VOCAB, self.hidden, ids)
        s["q"], s["k"], s["v"] = (self.project(w, s["x"]) for w in (self.wq, self.wk, self.wv))
        q = s["q"].view(-1, HQ, HD)
        s["turned"] = self.cache.append_rotary(self.rotary, s["k"], s["v"], q, seqs=seqs, cu_rows=cu)
        s["out"], s["m"], s["z"] = self.cache.attention(s["turned"], seqs=seqs, cu_rows=cu, max_rows=max_rows, max_len=256,
                                                        **self.how)
        s["logits"] = self.project(self.wo, s["out"].flatten(1))
        return s["logits"]

    def sample(self, logits, n):
        rules = {k: v[:n] for k, v in self.rules.items()}
        ids, self.seen["prob"] = ops.sample(logits, self.u[:n], **rules)
        return ids

    def prompt(self, lens, rng):
        t = self.torch
        n, cu = len(lens), np.concatenate([[0], np.cumsum(lens)])
        ids = ints(t, rng.integers(0, VOCAB, cu[-1]), self.dev)
        self.cache.extend(n=n, add=ints(t, lens, self.dev))
        cu_rows = ints(t, cu, self.dev)
        logits = self.rows(ids, n, None, cu_rows, int(max(lens)))
        last = logits[cu_rows[1:].long() - 1].contiguous()
        self.tokens[:n] = self.sample(last, n)
        return cu

    def step(self, n):
        self.cache.extend(n=n)
        logits = self.rows(self.tokens[:n], n, None, None, 1)
        self.tokens[:n] = self.sample(logits, n)


def check(s, entries, ids_before, n_ids):
    """The stages of the last call; entries: (sequence, first row, rows)."""
    seen = {k: v.cpu().double().numpy() for k, v in s.seen.items()}
    x = s.table.cpu().double().numpy()[ids_before]
    assert np.array_equal(seen["x"], x)
    pos = np.concatenate([np.arange(int(s.cache.lengths[q]) - c, int(s.cache.lengths[q])) for q, _, c in entries])
    want, bound = rotary_reference.rotate(seen["q"].reshape(-1, HQ, HD), pos, s.rotary.turns.cpu().numpy(), s.rotary.layout,
                                          s.rotary.amplitude)
    assert np.all(np.abs(seen["turned"] - want) <= bound)
    kt, kb = rotary_reference.rotate(seen["k"].reshape(-1, HKV, HD), pos, s.rotary.turns.cpu().numpy(), s.rotary.layout,
                                     s.rotary.amplitude)
    rows = []
    for q, first, c in entries:
        k, v, held = ref.dense(s.cache, 0, q, missing_ok=True)
        at = slice(first, first + c)
        off_k, off_v = np.abs(k[len(k) - c :] - kt[at]), np.abs(v[len(v) - c :] - seen["v"].reshape(-1, HKV, HD)[at])
        if s.cache.fmt == _lib.Q4_GROUP:   # half a step, at most the range's fifteenth and 1/32 of it
            lim = lambda y: np.repeat((np.maximum(y.reshape(-1, HKV, 2, 32).max(-1), 0) -   # noqa: E731
                                       np.minimum(y.reshape(-1, HKV, 2, 32).min(-1), 0)), 32, -1).reshape(y.shape) / 30 * (1 + 2.0**-4)
        else:
            lim = lambda y: np.abs(y) * 2.0**-11 + 2.0**-25   # noqa: E731
        assert np.all(off_k <= lim(kt[at]) + kb[at]) and np.all(off_v <= lim(seen["v"].reshape(-1, HKV, HD)[at]) + 1e-30)
        for j in range(c):
            rows.append(ref.attend(seen["turned"][first + j], k, v, held, len(k) - c + j, **s.how))
    ref.check_rows([s.seen[x] for x in ("out", "m", "z")], rows)
    last = [first + c - 1 for _, first, c in entries]
    ids, probs = s.tokens[: len(entries)].cpu().numpy(), seen["prob"]
    for r in range(n_ids):
        rule = [float(s.rules[k][r]) for k in ("temperature", "top_k", "top_p", "min_p")]
        i, share, near = sample_reference.draw(seen["logits"][last[r]], float(s.u[r]), *rule)
        assert near < 2.0**-32 or (ids[r] == i and abs(probs[r] - share) <= share * (2.0**-24 + 2.0**-36))


@pytest.mark.parametrize("fmt,layout,window,sinks", [(_lib.Q4_GROUP, "halves", 0, 0), (_lib.F16, "neighbours", 0, 0),
                                                     (_lib.Q4_GROUP, "neighbours", 24, 3)])
def test_a_serving_loop(env, fmt, layout, window, sinks):
    torch, _, dev = env
    s, rng = Server(env, fmt, layout, window, sinks), np.random.default_rng(2)
    lens = [40, 1, 17, 66]
    s.u[:4] = torch.tensor(rng.random(4), device=dev)
    state = rng.bit_generator.state
    cu = s.prompt(lens, rng)
    rng.bit_generator.state = state
    ids = rng.integers(0, VOCAB, cu[-1])
    check(s, [(q, int(cu[q]), lens[q]) for q in range(4)], ids, 4)
    s.cache.fork(ints(torch, [0, 0], dev), ints(torch, [4, 5], dev))   # two more samples of the first prompt
    s.tokens[4:] = s.tokens[0]
    for i in range(12):
        s.u.copy_(torch.tensor(rng.random(SEQS), device=dev))
        before = s.tokens.cpu().numpy().copy()
        s.step(SEQS)
        check(s, [(q, q, 1) for q in range(SEQS)], before, SEQS)
        if window and i == 8:   # what the windows have left behind, and the pool closed up
            n = s.cache.lengths
            s.cache.free(None, torch.full_like(n, sinks), (n - window).clamp(min=0))
            s.cache.compact()
    assert (s.tokens >= 0).all() and (s.tokens < VOCAB).all()
    assert s.cache.lengths.tolist() == [52, 13, 29, 78, 52, 52]
    assert ops.device_error() == 0


def test_a_captured_loop(env):
    torch, _, dev = env
    eager, graph = Server(env, _lib.Q4_GROUP, "halves"), Server(env, _lib.Q4_GROUP, "halves")
    for s in (eager, graph):
        rng = np.random.default_rng(3)
        s.u.fill_(0.4)
        s.prompt([20, 5, 1, 33, 2, 9], rng)
        s.step(SEQS)
    assert torch.equal(eager.tokens, graph.tokens)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graph.step(SEQS)
    rng = np.random.default_rng(4)
    for i in range(10):
        u = torch.tensor(rng.random(SEQS), dtype=torch.float32, device=dev)
        for s in (eager, graph):
            s.u.copy_(u)
        eager.step(SEQS)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.tokens, graph.tokens), i
        assert torch.equal(eager.seen["logits"], graph.seen["logits"])
        assert torch.equal(eager.cache.lengths, graph.cache.lengths) and torch.equal(eager.cache.table, graph.cache.table)
    assert ops.device_error() == 0
