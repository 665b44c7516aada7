"""The attention weight that each cell of a 4-bit K cache gets (tsr_hip_attn_weights_kv4) against 64 bits."""
import math

import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P
import weights4_ref as W

pytestmark = pytest.mark.gpu


def run(dev, q, kc, D, nh, nkv, n_kv, runs=None, before=None, decay=1.0, ws=None, in_place=False, scale=None):
    T = q.shape[0]
    bb = None if before is None else dev.upload(np.concatenate([np.asarray(before, np.float32), np.full(7, 5.0, np.float32)]))
    out = bb if in_place else dev.upload(np.full(n_kv + 7, 5.0, np.float32))
    dev.attn_weights_kv4(dev.upload(q), T, nh * D, kc, D, nh, nkv, scale or 1 / math.sqrt(D), n_kv, out, before=bb, decay=decay,
                         runs=None if runs is None else dev.upload(np.asarray(runs, np.uint32)), ws=ws)
    got = out.read(np.float32, (n_kv + 7,))
    assert (got[n_kv:] == 5.0).all()
    return got[:n_kv]


def check(got, want, tol):
    R.check(got, want, tol)


SHAPES = [
    # n_head, n_head_kv, D, T, n_kv
    (32, 8, 128, 1, 3000), (14, 2, 64, 1, 900), (1, 1, 64, 1, 1), (8, 8, 128, 1, 33), (4, 4, 64, 5, 257), (14, 2, 64, 7, 700),
    (32, 8, 128, 9, 500), (16, 2, 128, 3, 400), (16, 2, 128, 40, 300), (8, 4, 256, 1, 600), (8, 4, 256, 20, 300), (4, 1, 512, 6, 200),
    (64, 1, 64, 3, 300), (40, 2, 64, 2, 128), (8, 1, 128, 70, 1000),
]


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", SHAPES)
def test_shapes(dev, typ, nh, nkv, D, T, n_kv):
    rng = np.random.default_rng(nh * D + T)
    kc, _ = P.fill(dev, P.cache_rows(nh + D, n_kv + 40, nkv * D), typ)
    ki = R.quantize(P.cache_rows(nh + D, n_kv + 40, nkv * D), typ)
    q = rng.standard_normal((T, nh * D)).astype(np.float32)
    check(run(dev, q, kc, D, nh, nkv, n_kv), *W.weights(q, ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv))
    runs = np.sort(rng.integers(0, n_kv + 30, (T, 2, 2)), -1).reshape(T, 4)
    before = rng.uniform(0, 3, n_kv).astype(np.float32)
    for decay, in_place in ((0.75, False), (1.0, True), (0.0, False)):
        want = W.weights(q, ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs, before, decay)
        check(run(dev, q, kc, D, nh, nkv, n_kv, runs, before, decay, in_place=in_place), *want)


def test_causal_rows_and_the_sum(dev):
    """A causal ubatch: every row's weights sum to one."""
    nh, nkv, D, T, hist = 8, 2, 64, 90, 400
    n_kv = hist + T
    rows = P.cache_rows(2, n_kv, nkv * D)
    kc, ki = P.fill(dev, rows, R.Q4_0)[0], R.quantize(rows, R.Q4_0)
    q = np.random.default_rng(1).standard_normal((T, nh * D)).astype(np.float32)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = hist + 1 + np.arange(T)
    got = run(dev, q, kc, D, nh, nkv, n_kv, runs)
    want, tol = W.weights(q, ki, R.Q4_0, D, nh, nkv, 0.125, n_kv, runs)
    check(got, want, tol)
    assert abs(got.astype(np.float64).sum() - T * nh) <= tol.sum()


def test_rows_that_see_nothing(dev):
    nh, nkv, D, n_kv = 4, 2, 64, 300
    rows = P.cache_rows(2, n_kv, nkv * D)
    kc, ki = P.fill(dev, rows, R.Q4_1)[0], R.quantize(rows, R.Q4_1)
    q = np.random.default_rng(1).standard_normal((4, nh * D)).astype(np.float32)
    none = np.array([[5, 5, 0, 0], [300, 400, 9, 2], [0, 0, 0, 0], [7, 3, 350, 360]], np.uint32)
    assert (run(dev, q, kc, D, nh, nkv, n_kv, none) == 0).all()
    before = np.arange(n_kv, dtype=np.float32)
    assert (run(dev, q, kc, D, nh, nkv, n_kv, none, before, 0.5) == 0.5 * before).all()
    some = none.copy()
    some[2] = (100, 101, 0, 0)                                      # one row, one cell
    got = run(dev, q, kc, D, nh, nkv, n_kv, some)
    assert got[100] == nh and (np.delete(got, 100) == 0).all()


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
def test_cells_that_are_not_seen_reach_nothing(dev, typ):
    """Infinities and NaNs in cells that a row does not see; a row that sees one gives its cells NaN, the others keep theirs."""
    nh, nkv, D, n_kv = 4, 2, 128, 200
    rows = P.cache_rows(3, n_kv, nkv * D)
    rows[50:60], rows[150, 3] = np.inf, -np.inf
    kc, ki = P.fill(dev, rows, typ)[0], R.quantize(rows, typ)
    q = np.random.default_rng(2).standard_normal((3, nh * D)).astype(np.float32)
    runs = np.array([[0, 50, 60, 150], [0, 40, 160, 200], [61, 149, 0, 0]], np.uint32)
    before = np.ones(n_kv, np.float32)
    want, tol = W.weights(q, ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs, before)
    assert np.isfinite(want).all()
    check(run(dev, q, kc, D, nh, nkv, n_kv, runs, before), want, tol)
    runs[1, 1] = 55
    got = run(dev, q, kc, D, nh, nkv, n_kv, runs, before)
    assert np.isnan(got[:55]).all() and np.isnan(got[160:]).all()
    w2, t2 = W.weights(q[[0, 2]], ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs[[0, 2]], before)
    check(got[55:160], w2[55:160], t2[55:160])


def test_large_scores_and_large_scales(dev):
    """Scores of thousands (one cell takes it all) and K of 1e30 under a small scale."""
    nh, nkv, D, n_kv = 2, 1, 64, 500
    rows = P.cache_rows(4, n_kv, D)
    kc, ki = P.fill(dev, rows, R.Q4_0)[0], R.quantize(rows, R.Q4_0)
    q = (300 * np.random.default_rng(3).standard_normal((2, nh * D))).astype(np.float32)
    check(run(dev, q, kc, D, nh, nkv, n_kv, scale=1.0), *W.weights(q, ki, R.Q4_0, D, nh, nkv, 1.0, n_kv))
    q = (q * np.float32(1e30)).astype(np.float32)
    check(run(dev, q, kc, D, nh, nkv, n_kv, scale=1e-33), *W.weights(q, ki, R.Q4_0, D, nh, nkv, float(np.float32(1e-33)), n_kv))


def test_the_same_bits_again_and_in_parts(dev):
    """The order of the sums is fixed; a long call that goes out in several launches is the sum of its parts."""
    nh, nkv, D, T, n_kv = 2, 1, 64, 900, 20000
    kc, _ = P.fill(dev, P.cache_rows(5, n_kv, D), R.Q4_0)
    q = np.random.default_rng(4).standard_normal((T, nh * D)).astype(np.float32)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = n_kv - T + 1 + np.arange(T)
    a = run(dev, q, kc, D, nh, nkv, n_kv, runs)
    assert (a == run(dev, q, kc, D, nh, nkv, n_kv, runs)).all()
    long = np.tile(q, (40, 1))                                      # 36000 tokens: more than a launch takes
    b = run(dev, long, kc, D, nh, nkv, n_kv, np.tile(runs, (40, 1)))
    # each sum's roundings: one a row (40 T nh of them), 2^-24 of the sum
    assert (np.abs(b - 40.0 * a.astype(np.float64)) <= 40.0 * a * (41 * T * nh) * 2.0 ** -24).all()
    assert abs(b.astype(np.float64).sum() - 40 * T * nh) <= 40 * T * nh * 1e-4


def test_in_a_graph(dev):
    """A captured call, its workspace with it, accumulates in place at every replay."""
    nh, nkv, D, n_kv = 8, 2, 128, 1500
    rows = P.cache_rows(6, n_kv, nkv * D)
    kc, ki = P.fill(dev, rows, R.Q4_0)[0], R.quantize(rows, R.Q4_0)
    need = dev.attn_weights_kv4_ws(1, D, nh, nkv, n_kv)
    ws, qb, rb = dev.alloc(need), dev.alloc(4 * nh * D), dev.alloc(16)
    acc = dev.upload(np.zeros(n_kv, np.float32))
    args = (qb, 1, nh * D, kc, D, nh, nkv, 0.09, n_kv, acc)
    dev.graph_begin()
    with pytest.raises(Exception):
        dev.attn_weights_kv4(*args, before=acc, runs=rb)
    dev.attn_weights_kv4(*args, before=acc, decay=0.5, runs=rb, ws=ws)
    g = dev.graph_end()
    want, tol = np.zeros(n_kv), np.zeros(n_kv)
    for k, end in enumerate((1500, 40, 1000, 1)):
        q = np.random.default_rng(k).standard_normal((1, nh * D)).astype(np.float32)
        qb.write(q)
        rb.write(np.array([0, end, 0, 0], np.uint32))
        ws.fill(0xFF)
        g.launch()
        w, t = W.weights(q, ki, R.Q4_0, D, nh, nkv, 0.09, n_kv, np.array([[0, end, 0, 0]]))
        want, tol = 0.5 * want + w, 0.5 * tol + t + 2.0 ** -24 * (0.5 * want + w)
        check(acc.read(np.float32, (n_kv,)), want, tol)
    g.free()


MANY = [
    # n_head, n_head_kv, D, T, n_kv
    (8, 2, 64, 40, 700), (32, 8, 128, 33, 500), (4, 1, 256, 70, 400), (3, 3, 64, 200, 130), (8, 1, 128, 16, 31), (16, 1, 64, 9, 2100),
]


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", MANY)
def test_many_rows(dev, typ, nh, nkv, D, T, n_kv):
    """Rows for several waves: all cells, causal, sequences side by side in one cache, ragged runs, some empty."""
    rng = np.random.default_rng(D + T)
    rows = P.cache_rows(nh + D, n_kv + 40, nkv * D)
    rows[n_kv:] = 6e4                                               # (behind the cells in use)
    kc, ki = P.fill(dev, rows, typ)[0], R.quantize(rows, typ)
    q = rng.standard_normal((T, nh * D)).astype(np.float32) * 10.0 ** rng.integers(-2, 1, (T, 1)).astype(np.float32)
    causal, apart = np.zeros((T, 4), np.uint32), np.zeros((T, 4), np.uint32)
    causal[:, 1] = np.clip(n_kv - T + 1 + np.arange(T), 0, n_kv)
    cut = np.sort(rng.integers(0, n_kv + 1, 4))
    for t in range(T):
        s = 5 * t // T
        apart[t] = (0 if s == 0 else cut[s - 1], n_kv if s == 4 else cut[s], 0, 0)
    ragged = np.sort(rng.integers(0, n_kv + 30, (T, 2, 2)), -1).reshape(T, 4)
    ragged[::7] = (3, 3, 9, 2)
    for runs in (None, causal, apart, ragged):
        check(run(dev, q, kc, D, nh, nkv, n_kv, runs), *W.weights(q, ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs))


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("size", [1e-6, 2e-3, 300.0, 6e4])
def test_many_rows_of_any_size(dev, typ, size):
    """K from what leaves subnormal scales to what fills f16's range; next to cells that are not seen and hold what is not finite."""
    nh, nkv, D, T, n_kv = 8, 2, 128, 40, 300
    rows = np.clip(P.cache_rows(9, n_kv, nkv * D) * size, -6e4, 6e4).astype(np.float32)
    rows[100:110], rows[290], rows[291] = np.inf, np.nan, 6e4
    kc, ki = P.fill(dev, rows, typ)[0], R.quantize(rows, typ)
    q = np.random.default_rng(2).standard_normal((T, nh * D)).astype(np.float32)
    runs = np.tile(np.array([[0, 100, 110, 290]], np.uint32), (T, 1))
    runs[5:20, 1] = 64 + np.arange(15)
    scale = 0.1 / max(size, 1e-6) / math.sqrt(D)
    check(run(dev, q, kc, D, nh, nkv, n_kv, runs, scale=scale), *W.weights(q, ki, typ, D, nh, nkv, float(np.float32(scale)), n_kv, runs))


def test_many_rows_again(dev):
    """The same bits again, with a workspace, in a graph between eager calls; a row of NaNs."""
    nh, nkv, D, T, n_kv = 16, 4, 128, 48, 900
    rows = P.cache_rows(9, n_kv, nkv * D)
    kc = P.fill(dev, rows, R.Q4_1)[0]
    q = np.random.default_rng(2).standard_normal((T, nh * D)).astype(np.float32)
    one = run(dev, q, kc, D, nh, nkv, n_kv)
    assert (one == run(dev, q, kc, D, nh, nkv, n_kv)).all()
    ws = dev.alloc(dev.attn_weights_kv4_ws(T, D, nh, nkv, n_kv))
    assert (one == run(dev, q, kc, D, nh, nkv, n_kv, ws=ws)).all()
    out, qb = dev.alloc(4 * n_kv), dev.upload(q)
    dev.graph_begin()
    dev.attn_weights_kv4(qb, T, nh * D, kc, D, nh, nkv, 1 / math.sqrt(D), n_kv, out, ws=ws)
    g = dev.graph_end()
    for i in range(3):
        g.launch()
        assert (out.read(np.float32, (n_kv,)) == one).all()
        assert (run(dev, q[:9], kc, D, nh, nkv, n_kv) >= 0).all()
    bad = rows.copy()
    bad[500] = np.nan                                               # (stored as a row of zeros)
    kc, ki = P.fill(dev, bad, R.Q4_1)[0], R.quantize(bad, R.Q4_1)
    runs = np.tile(np.array([[0, 500, 501, 900]], np.uint32), (T, 1))
    runs[7, 1] = 501
    check(run(dev, q, kc, D, nh, nkv, n_kv, runs), *W.weights(q, ki, R.Q4_1, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs))


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
def test_many_rows_and_an_infinity(dev, typ):
    """A row that sees a cell of infinities gives its cells NaN, the others keep theirs."""
    nh, nkv, D, T, n_kv = 16, 4, 128, 48, 900
    rows = P.cache_rows(9, n_kv, nkv * D)
    rows[500] = np.inf
    kc, ki = P.fill(dev, rows, typ)[0], R.quantize(rows, typ)
    q = np.random.default_rng(2).standard_normal((T, nh * D)).astype(np.float32)
    runs = np.tile(np.array([[0, 500, 501, 900]], np.uint32), (T, 1))
    check(run(dev, q, kc, D, nh, nkv, n_kv, runs), *W.weights(q, ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs))
    runs[7] = (490, 520, 0, 0)
    got = run(dev, q, kc, D, nh, nkv, n_kv, runs)
    others = np.delete(np.arange(T), 7)
    want, tol = W.weights(q[others], ki, typ, D, nh, nkv, 1 / math.sqrt(D), n_kv, runs[others])
    assert np.isnan(got[490:520]).all()
    outside = np.delete(np.arange(n_kv), np.arange(490, 520))
    check(got[outside], want[outside], tol[outside])
