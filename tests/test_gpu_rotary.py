"""Rotary positions on the GPU against their 64-bit restatement, and the append that applies them bit by bit
against the rotation and the append one after the other."""
import numpy as np
import pytest

import rotary_reference as ref
from rta import _lib, ops, rotary
from test_gpu_pages import env, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu
FORMATS = [_lib.F16, _lib.BF16, _lib.Q8_ROW, _lib.Q4_GROUP]
HOW = {"plain": {}, "linear": dict(factor=4.0), "base": dict(factor=8.0), "ramp": dict(factor=16.0, original=4096),
       "bands": dict(factor=8.0, original=8192, low=1.0, high=4.0)}


def rows_of(torch, dev, rows, heads, hd, seed, pad=0):
    x = torch.randn(rows, heads * hd + pad, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)
    return x[:, : heads * hd].unflatten(1, (heads, hd))


def check(y, x, positions, table, layout, amplitude):
    want, bound = ref.rotate(x.cpu().numpy(), positions.cpu().numpy(), table.cpu().numpy(), layout, amplitude)
    err = np.abs(y.cpu().double().numpy() - want)
    assert np.all(err <= bound), float((err - bound).max())


@pytest.mark.parametrize("layout", ["neighbours", "halves"])
@pytest.mark.parametrize("rows,heads,hd,dims", [(1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 64, 32), (17, 33, 128, 20),
                                                (5, 3, 256, 256), (2, 7, 96, 90), (9, 2, 512, 510), (4, 2, 512, 2),
                                                (6, 3, 77, 76), (2100, 3, 64, 64), (300, 40, 128, 64), (3, 400, 33, 8)])
def test_rows(env, layout, rows, heads, hd, dims):
    torch, _, dev = env
    r = rotary.Rotary(hd, dims, layout, theta=1e4)
    x = rows_of(torch, dev, rows, heads, hd, 1, pad=3)
    p = torch.randint(-5, 1 << 20, (rows,), generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    p[0] = 0
    if rows > 2:
        p[1], p[2] = (1 << 31) + 12345, -(1 << 33)
    y = r.rotate(x, p)
    check(y, x, p, r.turns, layout, 1.0)
    assert torch.equal(y[0], x[0])   # position 0
    assert torch.equal(y[..., dims:], x[..., dims:])
    assert torch.equal(r.rotate(x, p), y)
    # in place, and into rows of another stride with room behind them
    room = torch.full((rows, heads * hd + 5), 7.0, device=dev)
    out = room[:, : heads * hd].unflatten(1, (heads, hd))
    assert torch.equal(r.rotate(x, p, out=out), y) and (room[:, heads * hd :] == 7).all()
    z = rows_of(torch, dev, rows, heads, hd, 1, pad=3)
    base = z._base if z._base is not None else z
    behind = base.clone().view(-1)[heads * hd :: heads * hd + 3]
    assert r.rotate(z, p, out=z) is z and torch.equal(z, y)
    assert torch.equal(base.view(-1)[heads * hd :: heads * hd + 3], behind)


@pytest.mark.parametrize("scaling", sorted(HOW))
@pytest.mark.parametrize("layout", ["neighbours", "halves"])
def test_scalings(env, scaling, layout):
    torch, _, dev = env
    for theta in (1e4, 1e6):
        r = rotary.Rotary(128, 96, layout, theta=theta, scaling=scaling, **HOW[scaling])
        x = rows_of(torch, dev, 50, 4, 128, 3)
        p = torch.randint(0, 1 << 18, (50,), generator=torch.Generator(device=dev).manual_seed(4), device=dev)
        want = torch.from_numpy(ref.turns(96, theta, scaling, **HOW[scaling]))
        check(r.rotate(x, p), x, p, r.turns, layout, r.amplitude)
        assert torch.all((r.turns.cpu() - want).abs() <= 2.0**-46 * want)


def test_neighbours_are_rope(env):
    """The whole head without scaling is rta_rope's rotation (the angle's roundings apart)."""
    torch, _, dev = env
    x = rows_of(torch, dev, 40, 8, 128, 5).contiguous()
    p = torch.arange(40, device=dev) * 2500
    y = rotary.Rotary(128, 64, theta=1e6).rotate(x, p)
    z = ops.rope(x.clone(), p, rotary=64, theta=1e6)
    _, bound = ref.rotate(x.cpu().numpy(), p.cpu().numpy(), ref.turns(64), "neighbours")
    assert np.all((y - z).abs().cpu().numpy() <= 2 * bound)


@pytest.mark.parametrize("layout", ["neighbours", "halves"])
def test_gradient(env, layout):
    """Gradients are the rotation at negated positions: against autograd of the formula in 64 bits and
    against differences of the formula."""
    torch, _, dev = env
    r = rotary.Rotary(64, 48, layout, theta=1e4, scaling="ramp", factor=4.0, original=512)
    x, g = rows_of(torch, dev, 7, 3, 64, 6), rows_of(torch, dev, 7, 3, 64, 7)
    p = torch.randint(0, 4000, (7,), generator=torch.Generator(device=dev).manual_seed(8), device=dev)
    got = r.rotate(g, -p).cpu().double()

    def formula(x):
        t = p.cpu().double()[:, None] * r.turns.cpu()
        angle = 2 * np.pi * (t - t.round())[:, None]
        c, s = r.amplitude * angle.cos(), r.amplitude * angle.sin()
        a, b = (x[..., 0:48:2], x[..., 1:48:2]) if layout == "neighbours" else (x[..., :24], x[..., 24:48])
        u, w = a * c - b * s, a * s + b * c
        part = torch.stack((u, w), -1).flatten(-2) if layout == "neighbours" else torch.cat((u, w), -1)
        return torch.cat((part, x[..., 48:]), -1)

    leaf = x.cpu().double().requires_grad_()
    (formula(leaf) * g.cpu().double()).sum().backward()
    _, bound = ref.rotate(g.cpu().numpy(), -p.cpu().numpy(), r.turns.cpu().numpy(), layout, r.amplitude)
    assert np.all((got - leaf.grad).abs().numpy() <= bound)
    rng = np.random.default_rng(9)
    for _ in range(20):
        at = tuple(int(rng.integers(0, n)) for n in x.shape)
        step = torch.zeros(x.shape, dtype=torch.float64)
        step[at] = 0.5   # (linear: differences of any step are exact up to 2^-53 of the sums)
        x64, g64 = x.cpu().double(), g.cpu().double()
        slope = float(((formula(x64 + step) - formula(x64 - step)) * g64).sum())
        assert abs(slope - float(got[at])) <= bound[at] + 1e-12


def test_values_that_are_not_finite_stay_in_their_pairs(env):
    torch, _, dev = env
    for layout, partner in (("neighbours", 7), ("halves", 6 + 16)):
        x = rows_of(torch, dev, 2, 2, 64, 10).contiguous()
        x[1, 0, 6], x[1, 1, 50] = float("nan"), float("inf")
        y = rotary.Rotary(64, 32, layout).rotate(x, torch.tensor([3, 4], device=dev))
        bad = ~torch.isfinite(y)
        want = torch.zeros_like(bad)
        want[1, 0, [6, partner]] = want[1, 1, 50] = True
        assert torch.equal(bad, want)


def append_case(env, fmt, hkv, hd, page, lens, counts, lead=0):
    torch, _, dev = env
    c = filled(env, fmt, hkv, hd, page, lens, layers=2)
    cu = np.concatenate([[lead], lead + np.cumsum(counts)])
    rows = int(cu[-1]) + lead
    k, v = (rows_of(torch, dev, rows, hkv, hd, s, pad=4).flatten(1) for s in (11, 12))
    pos = torch.zeros(rows, dtype=torch.int64, device=dev)
    for s, n in enumerate(counts):
        pos[int(cu[s]) : int(cu[s + 1])] = torch.arange(lens[s] - n, lens[s], device=dev)
    return c, ints(torch, cu, dev), rows, k, v, pos


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", ["neighbours", "halves"])
@pytest.mark.parametrize("hq,hkv,hd,dims,page", [(8, 2, 128, 128, 16), (3, 1, 64, 20, 1), (12, 3, 256, 64, 33),
                                                 (1, 34, 64, 64, 7), (40, 8, 128, 2, 100), (5, 5, 128, 94, 24)])
def test_append_is_rotation_and_append(env, fmt, layout, hq, hkv, hd, dims, page):
    torch, _, dev = env
    lens, counts = [37, 5, 0, 64, 1], [37, 3, 0, 20, 1]
    c, cu, rows, k, v, pos = append_case(env, fmt, hkv, hd, page, lens, counts, lead=2)
    r = rotary.Rotary(hd, dims, layout, theta=1e4, scaling="ramp", factor=8.0, original=64)
    q = rows_of(torch, dev, rows, hq, hd, 13, pad=1)
    c.pool.zero_()
    kr = r.rotate(k.unflatten(1, (hkv, hd)), pos).flatten(1)
    c.append(kr, v, layer=1, cu_rows=cu)
    want, want_q = c.pool.clone(), r.rotate(q, pos)
    c.pool.zero_()
    q_out = torch.full((rows, hq, hd), 7.0, device=dev)
    assert c.append_rotary(r, k, v, q, q_out, layer=1, cu_rows=cu) is q_out
    assert torch.equal(c.pool, want)
    assert torch.equal(q_out[2:-2], want_q[2:-2]) and (q_out[:2] == 7).all() and (q_out[-2:] == 7).all()
    # without queries, and with queries in place
    c.pool.zero_()
    assert c.append_rotary(r, k, v, layer=1, cu_rows=cu) is None
    assert torch.equal(c.pool, want)
    x = q.clone() if q.is_contiguous() else rows_of(torch, dev, rows, hq, hd, 13, pad=1)
    c.append_rotary(r, k, v, x, x, layer=1, cu_rows=cu)
    assert torch.equal(x[2:-2], want_q[2:-2]) and torch.equal(x[:2], q[:2])
    assert ops.device_error() == 0


@pytest.mark.parametrize("fmt", [_lib.F16, _lib.Q4_GROUP])
def test_many_rows(env, fmt):
    """Rows enough that a workgroup takes all of one's heads."""
    torch, _, dev = env
    lens, counts = [2500, 700], [2400, 31]
    c, cu, rows, k, v, pos = append_case(env, fmt, 2, 128, 64, lens, counts)
    q = rows_of(torch, dev, rows, 24, 128, 14)
    for layout in ("neighbours", "halves"):
        r = rotary.Rotary(128, 128, layout)
        c.pool.zero_()
        c.append(r.rotate(k.unflatten(1, (2, 128)), pos).flatten(1), v, cu_rows=cu)
        want = c.pool.clone()
        c.pool.zero_()
        assert torch.equal(c.append_rotary(r, k, v, q, cu_rows=cu), r.rotate(q, pos))
        assert torch.equal(c.pool, want)
        y = q.clone()
        assert torch.equal(c.append_rotary(r, k, v, y, y, cu_rows=cu), r.rotate(q, pos))
    assert ops.device_error() == 0


def test_rows_past_two_to_the_31(env):
    torch, _, dev = env
    r, p = rotary.Rotary(64, 32, "halves"), torch.tensor([7, 123456], device=dev)
    x = rows_of(torch, dev, 2, 3, 64, 16).contiguous()
    far = torch.zeros((1 << 31) + 1000, device=dev)
    view = far.as_strided((2, 3, 64), (1 << 31, 64, 1), 3)
    view.copy_(x)
    assert torch.equal(r.rotate(view, p), r.rotate(x, p))
    r.rotate(x, p, out=view)
    assert torch.equal(view, r.rotate(x, p))


def test_bad_rows_are_left_undone(env):
    torch, _, dev = env
    c = filled(env, _lib.F16, 2, 64, 4, [10, 6], extra=4)
    r = rotary.Rotary(64)
    c.table[1, 1] = -1                      # positions 4, 5 of sequence 1 have no page
    before = c.pool.clone()
    k = torch.randn(6, 128, device=dev)
    q, out = torch.randn(6, 3, 64, device=dev), torch.full((6, 3, 64), 7.0, device=dev)
    # two rows without a page, a sequence that is not there, and more rows than positions
    c.append_rotary(r, k, k, q, out, seqs=ints(torch, [1, 9, 5], dev), cu_rows=ints(torch, [0, 2, 4, 6], dev))
    assert ops.device_error() == _lib.DEVERR_PAGES
    assert torch.equal(c.pool, before) and (out == 7).all()
    c.append_rotary(r, k[:2], k[:2], q[:2], out[:2], seqs=ints(torch, [0], dev), cu_rows=ints(torch, [0, 2], dev))
    assert ops.device_error() == 0 and (out[:2] != 7).all()
    # an entry whose rows do not lie in the call's is refused beside one that is taken
    c.append_rotary(r, k, k, q, out, seqs=ints(torch, [0, 1], dev), cu_rows=ints(torch, [0, 2, 99], dev))
    assert ops.device_error() == _lib.DEVERR_PAGES and (out[2:] == 7).all()


def test_arguments_are_checked(env):
    torch, pages, dev = env
    c = filled(env, _lib.F16, 2, 64, 4, [10, 6])
    r = rotary.Rotary(64)
    k, q = torch.zeros(2, 128, device=dev), torch.zeros(2, 4, 64, device=dev)
    p = torch.zeros(2, dtype=torch.int64, device=dev)
    with pytest.raises(TypeError):
        r.rotate(q, p.int())
    with pytest.raises(TypeError):
        r.rotate(q.half(), p)
    with pytest.raises(TypeError):
        r.rotate(q.cpu(), p)
    with pytest.raises(ValueError):
        r.rotate(q, p[:1])
    with pytest.raises(ValueError):
        r.rotate(q[:, :, :32], p)
    with pytest.raises(ValueError):
        r.rotate(q, p, out=q[:, :2])
    with pytest.raises(ValueError):
        r.rotate(q[:, ::2], p)
    with pytest.raises(ValueError):
        c.append_rotary(rotary.Rotary(128), k, k)
    with pytest.raises(ValueError):
        c.append_rotary(r, k, k, q_out=q)
    with pytest.raises(ValueError):
        c.append_rotary(r, k, k, q[:1])
    with pytest.raises(ValueError):
        c.append_rotary(r, k, k, q, q_out=q[:, :2])
    with pytest.raises(_lib.RtaError):
        c.append_rotary(r, k, k, layer=9)


def test_streams_and_graphs(env):
    torch, _, dev = env
    lens = [30, 9]
    c, cu, rows, k, v, pos = append_case(env, _lib.Q4_GROUP, 2, 128, 16, lens, [1, 1])
    r = rotary.Rotary(128, layout="halves")
    q = rows_of(torch, dev, rows, 4, 128, 15).contiguous()
    k, v = k.contiguous(), v.contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.append_rotary(r, k * 1.0, v, q * 1.0, cu_rows=cu)
        turned = r.rotate(q * 1.0, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, turned) and torch.equal(turned, r.rotate(q, pos))
    g, out = torch.cuda.CUDAGraph(), torch.zeros_like(q)
    with torch.cuda.graph(g):
        c.extend(n=2)
        c.append_rotary(r, k, v, q, out, cu_rows=cu)
        alone = r.rotate(q, pos)
    for i in range(4):
        for t in (k, v, q):
            t.normal_()
        pos.add_(1)
        g.replay()
        torch.cuda.synchronize()
        assert c.lengths[:2].tolist() == [31 + i, 10 + i]
        want = r.rotate(q, pos)
        assert torch.equal(out, want) and torch.equal(alone, want), i
        stored = c.read(rows, cu_rows=cu)
        c.append(r.rotate(k.unflatten(1, (2, 128)), pos).flatten(1), v, cu_rows=cu)
        assert all(torch.equal(a, b) for a, b in zip(stored, c.read(rows, cu_rows=cu))), i
    assert ops.device_error() == 0


@pytest.mark.parametrize("layout", ["neighbours", "halves"])
def test_far_positions_lose_nothing(env, layout):
    """Positions up to 2^53 against the exact product of position and turns: its fraction of a turn, however many were made, is held
    to 2^-53 and the result to one rounding (the rounded product would be off by up to an eighth of a turn)."""
    from fractions import Fraction
    torch, _, dev = env
    rows, heads, hd, dims = 64, 3, 64, 48
    r = rotary.Rotary(hd, dims, layout, theta=1e4, scaling="bands", factor=8.0, original=8192, low=1.0, high=4.0)
    rng = np.random.default_rng(17)
    p = np.round(np.exp2(rng.uniform(20, 53, rows))).astype(np.int64) * rng.choice([-1, 1], rows)
    p[:4] = [1 << 53, -(1 << 53), (1 << 53) - 1, 1 << 52]
    x = rows_of(torch, dev, rows, heads, hd, 18)
    y = r.rotate(x, torch.tensor(p, device=dev)).cpu().double().numpy()
    table = r.turns.cpu().numpy()
    part = np.empty((rows, dims // 2))
    for i in range(rows):
        for j in range(dims // 2):
            made = int(p[i]) * Fraction(float(table[j]))
            part[i, j] = float(made - round(made))
    angle = 2 * np.pi * part[:, None]
    c, s = np.cos(angle), np.sin(angle)
    lo, hi = (np.arange(0, dims, 2), np.arange(1, dims, 2)) if layout == "neighbours" else (np.arange(dims // 2), np.arange(dims // 2, dims))
    x = x.cpu().double().numpy()
    a, b = x[..., lo], x[..., hi]
    # one rounding; the fraction's, the series' and the products' in fp64, here and in numpy, below 2^-48 together
    bound = (np.abs(a) + np.abs(b)) * (2.0**-24 + 2.0**-48)
    assert np.all(np.abs(y[..., lo] - (a * c - b * s)) <= bound)
    assert np.all(np.abs(y[..., hi] - (a * s + b * c)) <= bound)
    assert np.array_equal(y[..., dims:], x[..., dims:])


@pytest.mark.parametrize("hd,dims", [(64, 20), (64, 62), (128, 94), (128, 12), (256, 250), (256, 130)])
@pytest.mark.parametrize("rows,hq", [(3, 40), (700, 24), (2100, 7)])
def test_queries_in_place_with_partners_one_by_one(env, hd, dims, rows, hq):
    """Halves that are no multiple of eight values: partners that other lanes of the wave store to, in rows of one workgroup and
    of several, heads of one wave and of many."""
    torch, _, dev = env
    c, cu, rows, k, v, pos = append_case(env, _lib.Q8_ROW, 2, hd, 32, [rows + 5], [rows])
    r = rotary.Rotary(hd, dims, "halves", theta=1e4)
    q = rows_of(torch, dev, rows, hq, hd, 19).contiguous()
    want = r.rotate(q, pos)
    for _ in range(3):
        y = q.clone()
        assert torch.equal(c.append_rotary(r, k, v, y, y, cu_rows=cu), want)
    assert torch.equal(c.append_rotary(r, k, v, q, cu_rows=cu), want)
    assert ops.device_error() == 0
