"""The draw from rows of logits against its 64-bit restatement: rules alone and together, ties, masks,
sizes from one word to several hundred thousand, the ends of u, bad rows, streams and graphs.  A draw
has to be the restatement's word unless u, or a rule, is closer to a border than the weights' own
precision (2^-50 a word of up to 2^18, and 2^-45 of a scaled logit)."""
import numpy as np
import pytest

import sample_reference as ref
from rta import _lib, ops

pytestmark = pytest.mark.gpu
CLOSE = 2.0**-32


@pytest.fixture(scope="module")
def env():
    import torch
    ops.device_error(clear=True)
    return torch, torch.device("cuda:0")


def run(env, x, u, t=None, k=None, p=None, least=None):
    torch, dev = env
    up = lambda v, d: None if v is None else torch.tensor(np.asarray(v), dtype=d, device=dev)   # noqa: E731
    f = torch.float32
    x = x if isinstance(x, torch.Tensor) else up(x, f)
    return ops.sample(x, up(u, f), up(t, f), up(k, torch.int32), up(p, f), up(least, f))


def check(env, x, u, t=None, k=None, p=None, least=None, most_close=0):
    x, u = np.asarray(x, np.float32), np.asarray(u, np.float32)
    rows = len(x)
    ids, probs = (v.cpu().numpy() for v in run(env, x, u, t, k, p, least))
    pick = lambda v, r, off: off if v is None else np.asarray(v, np.float32 if off != 0 or v is not k else np.int64)[r]  # noqa: E731
    close = 0
    for r in range(rows):
        i, share, near = ref.draw(x[r], u[r], pick(t, r, 1.0), pick(k, r, 0), pick(p, r, 1.0), pick(least, r, 0.0))
        if near < CLOSE:
            close += 1
            continue
        assert ids[r] == i, (r, ids[r], i, share, near)
        # fp32's rounding, and the weights' 2^-45 of a scaled logit's bits
        assert abs(probs[r] - share) <= share * (2.0**-24 + 2.0**-40), r
    assert close <= most_close
    return ids


def logits(rng, rows, vocab, sigma=2.5, sure=6.0):
    x = sigma * rng.standard_normal((rows, vocab)).astype(np.float32)
    top = rng.integers(0, vocab, (rows, 20))
    for r in range(rows):
        x[r, top[r]] += np.float32(sure) * rng.random(20).astype(np.float32)
    return x


SIZES = [1, 2, 3, 5, 63, 64, 1000, 8191, 8192, 8193, 16385, 50001, 151936]
RULES = {"none": {}, "t": dict(t=(0.2, 2.0)), "k": dict(k=(1, 3000)), "p": dict(p=(0.05, 0.999)), "least": dict(least=(1e-4, 0.5)),
         "all": dict(t=(0.2, 2.0), k=(1, 200), p=(0.2, 0.99), least=(0.001, 0.3)),
         "wide": dict(t=(0.7, 3.0), k=(3000, 60000), p=(0.9, 0.9999), least=(1e-6, 1e-4)),
         "kp": dict(k=(1, 50), p=(0.1, 1.0)), "deep": dict(t=(0.7, 3.0), p=(0.9, 0.999), least=(0.01, 0.9)),
         "deep k": dict(k=(100, 9000), p=(0.5, 0.99), least=(0.05, 0.9)), "k least": dict(k=(1, 9000), least=(1e-5, 0.9))}


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("rules", sorted(RULES))
def test_rules(env, vocab, rules):
    rng = np.random.default_rng(vocab)
    rows = 9
    x, u = logits(rng, rows, vocab), rng.random(rows).astype(np.float32)
    how = {}
    for name, (lo, hi) in RULES[rules].items():
        how[name] = rng.integers(lo, hi + 1, rows) if name == "k" else np.exp(rng.uniform(np.log(lo), np.log(hi), rows))
    check(env, x, u, **how)
    assert ops.device_error() == 0


@pytest.mark.parametrize("vocab", [7, 900, 20000, 100003])
@pytest.mark.parametrize("step", [0.0, 0.25, 4.0])
def test_ties(env, vocab, step):
    """Few distinct logits (step 0: all alike, where every sum is a whole number): bins past the list's room."""
    rng = np.random.default_rng(vocab)
    rows = 12
    x = np.zeros((rows, vocab), np.float32) if step == 0 else \
        (np.round(2.0 * rng.standard_normal((rows, vocab)) / step) * step).astype(np.float32)
    x[3] *= -1.0   # zeros of both signs are equal
    x[3, ::2] = np.abs(x[3, ::2])
    u = rng.random(rows).astype(np.float32)
    check(env, x, u)
    check(env, x, u, k=rng.integers(1, vocab + 2, rows))
    if step:
        check(env, x, u, p=rng.uniform(0.05, 0.99, rows))
        check(env, x, u, t=rng.uniform(0.3, 3, rows), k=rng.integers(1, vocab + 2, rows), p=rng.uniform(0.05, 0.99, rows),
              least=rng.uniform(0, 0.2, rows))
        check(env, x, u, least=np.full(rows, 1.0))
        return
    # halves, quarters: p of the words exactly
    for p in (0.5, 0.25, 0.125):
        ids, probs = (v.cpu().numpy() for v in run(env, x, u, p=np.full(rows, p)))
        kept = int(np.ceil(vocab * p))
        assert np.array_equal(ids, np.floor(u.astype(np.float64) * kept)) and np.allclose(probs, 1 / kept, rtol=1e-6)
    ids = run(env, x, u, t=np.full(rows, np.inf))[0].cpu().numpy()
    assert np.array_equal(ids, np.floor(u.astype(np.float64) * vocab))


def test_every_word_has_its_share(env):
    """One row many times, u over a grid: the counts are the shares, word by word."""
    torch, dev = env
    rng = np.random.default_rng(3)
    x = logits(rng, 1, 9000)
    n = 3000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for how in ({}, dict(k=[40]), dict(p=[0.9]), dict(least=[0.01])):
        ids = run(env, torch.tensor(x, device=dev).expand(n, -1), u, **{a: np.repeat(v, n) for a, v in how.items()})[0].cpu().numpy()
        assert np.all(np.diff(ids) >= 0)   # in the order of index
        share = np.zeros(x.shape[1])
        w = np.exp(x[0].astype(np.float64) - x.max())
        order = np.argsort(-w, kind="stable")
        keep = len(w)
        if "k" in how:
            keep = 40
        if "p" in how:
            keep = int((np.cumsum(w[order]) < np.float32(0.9) * w.sum()).sum()) + 1
        if "least" in how:
            keep = int((w >= np.float32(0.01)).sum())
        share[order[:keep]] = w[order[:keep]] / w[order[:keep]].sum()
        counts = np.bincount(ids, minlength=len(share))
        assert np.all(np.abs(counts - n * share) <= 1.0 + n * 2.0**-24) and not counts[share == 0].any()


def test_masks(env):
    rng = np.random.default_rng(4)
    rows, vocab = 10, 30000
    x, u = logits(rng, rows, vocab), rng.random(rows).astype(np.float32)
    x[0, 1:] = -np.inf                      # one word left
    x[1, : vocab - 1] = -np.inf
    x[2, rng.random(vocab) < 0.999] = -np.inf
    x[3, 8192:16384] = -np.inf              # a whole chunk
    x[4, ::2] = np.finfo(np.float32).min    # the type's lowest value: words of no weight
    x[5] = np.finfo(np.float32).min         # nothing else: all alike
    x[6] = -1e30 + 0 * x[6]
    x[6, 77] = 1e30
    x[7] = np.finfo(np.float32).max
    for how in ({}, dict(k=np.full(rows, 5)), dict(p=np.full(rows, 0.7)), dict(least=np.full(rows, 0.1)),
                dict(k=np.full(rows, 20000), p=np.full(rows, 0.99)), dict(t=np.full(rows, 1e-30)), dict(t=np.full(rows, 1e30))):
        ids = check(env, x, u, **how)
        assert ids[0] == 0 and ids[1] == vocab - 1 and ids[4] % 2 == 1
    assert ops.device_error() == 0


def test_the_ends_of_u_and_of_the_rules(env):
    rng = np.random.default_rng(5)
    x = np.repeat(logits(rng, 1, 20000), 12, 0)
    u = np.array([0, -1, np.nan, 1, 2, np.inf, 1 - 2.0**-24, 1e-45, 0.5, 0.5, 0.5, 0.5], np.float32)
    ids = run(env, x, u)[0].cpu().numpy()
    w = np.exp(x[0].astype(np.float64) - x.max())
    first, last = np.nonzero(w)[0][[0, -1]]
    assert (ids[:3] == first).all() and (ids[3:6] == last).all() and ids[7] == first and ids[6] <= last
    largest = int(np.argmax(x[0]))
    for how in (dict(t=np.array([0, -1, np.nan] * 4)), dict(k=np.ones(12)), dict(p=np.array([0, -3, 1e-30] * 4)),
                dict(least=np.array([1, 2, np.inf] * 4)), dict(t=np.full(12, 1e-6))):
        ids, probs = (v.cpu().numpy() for v in run(env, x, u, **how))
        assert (ids == largest).all() and (probs == 1).all(), how
    plain = run(env, x, u)
    for how in (dict(k=np.array([0, -5, 20000, 2**31 - 1] * 3)), dict(p=np.array([1, 2, np.nan, np.inf] * 3)),
                dict(least=np.array([0, -1, np.nan, -np.inf] * 3)), dict(t=np.ones(12))):
        assert all((a == b).all() for a, b in zip(run(env, x, u, **how), plain)), how
    assert ops.device_error() == 0


def test_a_word_on_min_ps_border_alone_in_its_chunk(env):
    """One word that min-p just keeps or drops, in a chunk of its own behind more words than are ranked at
    once: with u = 1 it is the draw if it is kept, and the last of the largest words if it is not."""
    rng = np.random.default_rng(23)
    rows = 256
    x = np.full((rows, 20000), -np.inf, np.float32)
    t = rng.uniform(1e-3, 3, rows).astype(np.float32)
    least = (2.0 ** -(rng.integers(1, 300, rows) / 8)).astype(np.float32)   # (borders of the bins of eighths too)
    top = rng.uniform(-30, 30, rows).astype(np.float32)
    top[::3] = 0
    x[:, :8192] = top[:, None]
    word = (top + t.astype(np.float64) * np.log(least.astype(np.float64))).astype(np.float32)
    for r in range(rows):
        for _ in range(abs(r % 5 - 2)):
            word[r] = np.nextafter(word[r], np.float32(np.inf if r % 5 > 2 else -np.inf))
    x[np.arange(rows), 9000] = word
    ids = check(env, x, np.ones(rows), t=t, least=least, most_close=2)
    assert set(ids.tolist()) == {8191, 9000}
    assert ops.device_error() == 0


def test_an_infinite_temperature_makes_all_words_alike(env):
    rng = np.random.default_rng(11)
    rows, vocab = 6, 70001
    x, u = logits(rng, rows, vocab), rng.random(rows).astype(np.float32)
    x[1, ::3] = -np.inf
    t = np.full(rows, np.inf)
    for how in ({}, dict(k=rng.integers(1, vocab, rows)), dict(p=np.full(rows, 0.5)), dict(least=np.full(rows, 0.5)),
                dict(k=rng.integers(1, 100, rows), p=np.full(rows, 0.25))):
        ids, probs = (v.cpu().numpy() for v in run(env, x, u, t=t, **how))
        for r in range(rows):
            order = np.lexsort((np.arange(vocab), -x[r]))
            n = int((x[r] > -np.inf).sum())
            n = min(n, int(how["k"][r])) if "k" in how else n
            n = int(np.ceil(n * how["p"][r])) if "p" in how else n
            assert ids[r] == np.sort(order[:n])[int(np.floor(float(u[r]) * n))] and abs(probs[r] * n - 1) < 1e-6, (how, r)
    assert ops.device_error() == 0


def test_rows_past_two_to_the_31(env):
    torch, dev = env
    rng = np.random.default_rng(12)
    x, u = logits(rng, 2, 20000), rng.random(2).astype(np.float32)
    far = torch.empty((1 << 31) + 30000, device=dev)
    view = far.as_strided((2, 20000), (1 << 31, 1), 5)
    view.copy_(torch.tensor(x, device=dev))
    for how in ({}, dict(k=[40, 3000], p=[0.9, 0.5])):
        assert all(torch.equal(a, b) for a, b in zip(run(env, view, u, **how), run(env, x, u, **how)))


def test_bad_rows(env):
    torch, _ = env
    rng = np.random.default_rng(6)
    x = logits(rng, 8, 9001)
    x[1, 9000], x[3, 17], x[5] = np.nan, np.inf, -np.inf
    u = rng.random(8).astype(np.float32)
    for how in ({}, dict(t=np.zeros(8)), dict(k=np.full(8, 3))):
        ids, probs = (v.cpu().numpy() for v in run(env, x, u, **how))
        assert ops.device_error() == _lib.DEVERR_DETECTOR
        bad = np.array([1, 3, 5])
        assert (ids[bad] == -1).all() and (probs[bad] == 0).all()
        good = np.array([0, 2, 4, 6, 7])
        want = [v.cpu().numpy() for v in run(env, x[good], u[good], **{a: v[good] for a, v in how.items()})]
        assert np.array_equal(ids[good], want[0]) and np.array_equal(probs[good], want[1])
        assert ops.device_error() == 0


def test_greedy_rows_beside_others(env):
    rng = np.random.default_rng(7)
    x = np.round(logits(rng, 6, 25000))     # several words share the maximum
    u = rng.random(6).astype(np.float32)
    ids = check(env, x, u, t=np.array([0, 1, 0, 0.5, -2, 1]))
    assert all(ids[r] == np.argmax(x[r]) for r in (0, 2, 4))


def test_strides_streams_and_repeats(env):
    torch, dev = env
    gen = torch.Generator(device=dev).manual_seed(8)
    rows, vocab = 5, 12345
    wide = 3 * torch.randn(rows, vocab + 7, generator=gen, device=dev)
    u = torch.rand(rows, generator=gen, device=dev)
    p = torch.full((rows,), 0.9, device=dev)
    for shift in range(4):
        x = wide[:, shift : shift + vocab]
        want = ops.sample(x.contiguous(), u, top_p=p)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(ops.sample(x, u, top_p=p), want))
    one = wide[:1, 1 : 1 + vocab]
    assert torch.equal(ops.sample(one, u[:1])[0], ops.sample(one.contiguous(), u[:1])[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample(wide[:, 3 : 3 + vocab] * 1.0, u, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_with_their_own_workspaces(env):
    torch, dev = env
    gen = torch.Generator(device=dev).manual_seed(9)
    rows, vocab = 4, 40000
    x, u = torch.empty(rows, vocab, device=dev), torch.empty(rows, device=dev)
    k = torch.tensor([0, 3, 50, 20000], dtype=torch.int32, device=dev)
    p = torch.tensor([0.9, 1.0, 0.5, 0.99], device=dev)
    x.normal_(generator=gen), u.uniform_(generator=gen)
    ops.sample(x, u, top_k=k, top_p=p)
    graphs, outs = [], []
    for how in (dict(top_k=k, top_p=p), dict(min_p=0.1 * p)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.sample(x, u, **how))
        graphs.append((g, how))
    for i in range(4):
        x.normal_(generator=gen).mul_(3), u.uniform_(generator=gen)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, how), got in zip(graphs, outs):
            assert all(torch.equal(a, b) for a, b in zip(ops.sample(x, u, **how), got)), i
    assert ops.device_error() == 0


def test_many_rows_and_long_vocabularies(env):
    rng = np.random.default_rng(10)
    x, u = logits(rng, 600, 777), rng.random(600).astype(np.float32)
    check(env, x, u, t=rng.uniform(0.3, 2, 600), k=rng.integers(0, 60, 600), p=rng.uniform(0.3, 1.2, 600), least=rng.uniform(-0.1, 0.1, 600))
    x, u = logits(rng, 2, 1 << 21, sigma=1.0, sure=3.0), rng.random(2).astype(np.float32)
    for how in ({}, dict(p=[0.95, 0.5]), dict(k=[700000, 100]), dict(least=[1e-3, 0.02])):
        check(env, x, u, **how, most_close=1)


def test_arguments_are_checked(env):
    torch, dev = env
    x, u = torch.zeros(3, 100, device=dev), torch.zeros(3, device=dev)
    with pytest.raises(TypeError):
        ops.sample(x.half(), u)
    with pytest.raises(TypeError):
        ops.sample(x, u.double())
    with pytest.raises(TypeError):
        ops.sample(x, u.cpu())
    with pytest.raises(TypeError):
        ops.sample(x, None)
    with pytest.raises(TypeError):
        ops.sample(x, u, top_k=torch.ones(3, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError):
        ops.sample(x, u[:2])
    with pytest.raises(ValueError):
        ops.sample(x[:, ::2], u)
    with pytest.raises(ValueError):
        ops.sample(x[0], u)
    with pytest.raises(ValueError):
        ops.sample(x, u, temperature=torch.ones(6, device=dev)[::2])
    with pytest.raises(_lib.RtaError):
        ops.sample(x, u, workspace=torch.empty(64, dtype=torch.uint8, device=dev))


@pytest.mark.parametrize("vocab", [5, 900, 70001])
def test_an_infinite_temperature_with_every_min_p_and_logits_near_zero(env, vocab):
    """Every finite logit weighs 1, whatever its size or sign, and 1 is not below a min-p of 1."""
    rng = np.random.default_rng(vocab)
    tiny = (rng.standard_normal(vocab) * np.exp2(rng.uniform(-149, -60, vocab))).astype(np.float32)
    rows = [logits(rng, 1, vocab)[0], -np.abs(tiny), np.abs(tiny), tiny, -np.abs(tiny), -np.abs(tiny), tiny, tiny]
    x = np.stack(rows).astype(np.float32)
    x[4, vocab // 2] = 3.0
    x[5, rng.random(vocab) < 0.3] = 0.0
    x[5, ::2] *= np.float32(-1.0)                                   # zeros of both signs
    x[6, rng.random(vocab) < 0.5] = -np.inf
    x[6, 1] = -np.finfo(np.float32).max
    x[7, rng.random(vocab) < 0.4] *= np.float32(1e38)
    x[7, 2], x[7, 3] = np.finfo(np.float32).max, np.finfo(np.float32).min
    n_rows = len(x)
    full = lambda v: np.full(n_rows, v)   # noqa: E731
    for how in (dict(), dict(least=full(1.0)), dict(least=full(0.5)), dict(least=full(2.0)), dict(k=rng.integers(1, vocab + 1, n_rows)),
                dict(p=full(0.5)), dict(k=rng.integers(1, vocab + 1, n_rows), least=full(1.0)), dict(p=full(0.25), least=full(1.0)),
                dict(k=rng.integers(1, vocab + 1, n_rows), p=full(0.5), least=full(1.0))):
        for u in (rng.random(n_rows).astype(np.float32), np.zeros(n_rows, np.float32), np.ones(n_rows, np.float32)):
            ids, probs = (v.cpu().numpy() for v in run(env, x, u, t=full(np.inf), **how))
            for r in range(n_rows):
                order = np.lexsort((np.arange(vocab), -x[r].astype(np.float64)))
                n = int((x[r] > -np.inf).sum())
                n = min(n, int(how["k"][r])) if "k" in how else n
                n = int(np.ceil(n * how["p"][r])) if "p" in how else n
                n = 1 if "least" in how and how["least"][r] > 1 else n
                want = np.sort(order[:n])[min(int(np.floor(float(u[r]) * n)), n - 1)]   # (whole sums: exact)
                assert ids[r] == want, (how, r, ids[r], want)
                assert abs(probs[r] * n - 1) <= 2.0**-24 + 2.0**-40, (how, r)
    assert ops.device_error() == 0


def pairs(seed, rows=16384, halves=False):
    """Rows (small word, large word) of logits up to 10^6 and temperatures down to 10^-4, a tenth of a temperature to three of
    them apart (halves: about one half, three halves, .. of an octave of weight), and the smaller one's weight in 64 bits of
    fraction."""
    rng = np.random.default_rng(seed)
    big = (rng.choice([-1.0, 1.0], rows) * np.exp(rng.uniform(np.log(0.1), np.log(1e6), rows))).astype(np.float32)
    t = np.maximum(np.exp(rng.uniform(np.log(1e-4), np.log(3.0), rows)), np.abs(big) * 2.0**-22).astype(np.float32)
    far = np.log(2) * (rng.integers(0, 4, rows) + rng.uniform(0.47, 0.53, rows)) if halves else rng.uniform(0.1, 3.0, rows)
    small = (big.astype(np.float64) - t.astype(np.float64) * far).astype(np.float32)
    apart = big.astype(np.longdouble) - small.astype(np.longdouble)
    use = (apart > 0) & (apart < 4 * t)
    w = np.exp(-apart / t.astype(np.longdouble))
    return big[use], small[use], t[use], w[use]


def check_pairs(env, seed, off, **how):
    """Draws and min-p at borders that lie between two floats: right wherever u, or min-p, is further from it than `off` of it."""
    big, small, t, w = pairs(seed, **how)
    x = np.stack((small, big), 1)
    share = w / (1 + w)
    u = share.astype(np.float32)
    far = np.abs(u.astype(np.longdouble) - share) > off * share
    assert far.mean() > 0.98
    for how in ({}, dict(k=np.full(len(u), 2))):
        ids, probs = (v.cpu().numpy() for v in run(env, x, u, t=t, **how))
        want = np.where(u < share, 0, 1)
        wrong = far & (ids != want)
        assert not wrong.any(), (int(wrong.sum()), np.nonzero(wrong)[0][:5])
        p = np.where(want, 1 - share, share)
        assert (np.abs(probs - p) <= p * (2.0**-24 + 2 * off))[far].all()
    least = w.astype(np.float32)
    far = np.abs(least.astype(np.longdouble) - w) > 2.0**-45 * w   # (no weight is computed: roundings of logarithms)
    assert far.mean() > 0.98
    ids = run(env, x[:, ::-1].copy(), np.ones(len(u)), t=t, least=least)[0].cpu().numpy()   # u = 1: the last word that stays
    wrong = far & (ids != np.where(w >= least, 1, 0))
    assert not wrong.any(), (int(wrong.sum()), np.nonzero(wrong)[0][:5])
    assert ops.device_error() == 0


@pytest.mark.parametrize("seed", [31, 32, 33, 34])
def test_weights_of_large_logits_and_low_temperatures(env, seed):
    """A series to the 9th power as it stands is 9.5e-12 (2^-36.6) off at most, wherever on the scale the logits lie: 2^-36 with
    the roundings (the difference's and two of its scale's, 2^-51 of up to 6 octaves; 2^-51 of a weight of 0.05 as a whole
    number: 2^-46)."""
    check_pairs(env, seed, 2.0**-36)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("seed", [41, 42, 43])
def test_weights_hold_what_the_shares_are_held_to(env, seed, halves):
    """check() allows a share 2^-40 besides its rounding, so a weight and its sum 2^-41 each.  The series is 2^-44.2 off at most (its
    ends: half an octave from a power of two), the roundings together 2^-46 as above: 2^-43."""
    check_pairs(env, seed, 2.0**-43, halves=halves)


@pytest.mark.parametrize("vocab", [3, 9000, 40000])
def test_the_least_weight_that_counts(env, vocab):
    """Words of 2^-47.74 of the largest are drawn where nothing lies in front of them (u = 0), words of 2^-47.88 never, wherever
    in its eighth of an octave the largest lies; in the largest's chunk and in one of their own."""
    rng = np.random.default_rng(vocab)
    rows = 64
    t = rng.uniform(0.1, 3.0, rows).astype(np.float32)
    top = rng.uniform(-40, 40, rows).astype(np.float32)
    for octaves, counts in ((47.74, True), (47.88, False)):
        x = np.full((rows, vocab), -np.inf, np.float32)
        x[:, vocab - 1] = top
        x[:, 0] = top.astype(np.float64) - octaves * np.log(2) * t.astype(np.float64)   # (fp32: 6e-5 of an octave off at most)
        for how in ({}, dict(k=np.full(rows, 2)), dict(least=np.full(rows, 1e-30))):
            ids = run(env, x, np.zeros(rows), t=t, **how)[0].cpu().numpy()
            assert (ids == (0 if counts else vocab - 1)).all(), (octaves, how)
    assert ops.device_error() == 0


def test_the_lowest_temperatures(env):
    """Exponents far past 32 bits: the largest word alone, by every rule, masked words beside it."""
    rng = np.random.default_rng(51)
    rows, vocab = 6, 20011
    x, u = logits(rng, rows, vocab), rng.random(rows).astype(np.float32)
    x[1, ::3] = -np.inf
    x[2] *= np.float32(1e37)
    x[3] *= np.float32(1e-37)
    x[4, 5:9000] = np.finfo(np.float32).min
    for t in (2.0**-149, 2.0**-126, 1e-30, 1e-20):   # (the fourth row's largest are 2e-38 apart)
        for how in ({}, dict(k=np.full(rows, 40)), dict(p=np.full(rows, 0.9)), dict(least=np.full(rows, 1e-9)),
                    dict(k=np.full(rows, 9000), p=np.full(rows, 0.99), least=np.full(rows, 0.1))):
            keep = np.array([0, 1, 2, 4, 5]) if t > 2.0**-149 else np.arange(rows)
            ids, probs = (v.cpu().numpy() for v in run(env, x, u, t=np.full(rows, t), **how))
            assert np.array_equal(ids[keep], np.argmax(x, 1)[keep]) and (probs[keep] == 1).all(), (t, how)
    assert ops.device_error() == 0


@pytest.mark.parametrize("words", [9000, 131072, 600000])
@pytest.mark.parametrize("far", [3.0, 17.0, 22.0, 25.0])
def test_top_p_among_many_equal_words_of_little_weight(env, words, far):
    """One word of all but a little of the weight and many equal ones of little: top-p's border among these lies where it ought to
    but for the whole numbers of 2^-50 (2^-51 a word), the weights' 2^-43 of what they are, and one word.  u = 1 is the last
    word that stays."""
    rows = 24
    w = np.exp(-np.longdouble(np.float32(far)))
    rest = words * w
    # p from 1 down to the first word's share, as floats
    first = float(1 / (1 + rest))
    p = np.unique(np.linspace(first, 1.0, rows + 2).astype(np.float32)[1:-1])
    p = p[(p < 1) & (p > np.float32(first))]
    assert len(p)
    x = np.full((len(p), words + 1), -far, np.float32)
    x[:, 5] = 0.0
    goal = p.astype(np.longdouble) * (1 + rest)
    want = np.ceil((goal - 1) / w)                  # of the equal words
    off = (words * 2.0**-51 + rest * 2.0**-43 + goal * 2.0**-52) / w + 1
    for how in ({}, dict(least=np.full(len(p), 1e-14)), dict(k=np.full(len(p), words + 1))):
        ids = run(env, x, np.ones(len(p)), p=p, **how)[0].cpu().numpy()
        stay = ids.astype(np.int64) + 1 - (ids > 5)     # the words up to the last one, without the large one
        assert (np.abs(stay - want) <= off).all(), (how, stay - want, off)
    assert ops.device_error() == 0
