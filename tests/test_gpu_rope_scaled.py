"""Rotary positions scaled for long contexts (tsr_hip_rope_scaled, tsr_hip_rope_scaled_table) against 64 bits."""
import numpy as np
import pytest

import rope_scaled_ref as R
import tsr_hip as H

pytestmark = pytest.mark.gpu


def run(dev, x, pos, heads, hd, n, mode, sc, ff=None, stride=None, y=None, off=0):
    """x [T, stride] (device rows of heads hd values, the rest behind them); off: floats in front of the first row."""
    T = len(pos)
    stride = x.shape[1] if stride is None else stride
    whole = np.concatenate([np.full(off, 7.0, np.float32), np.ascontiguousarray(x, np.float32).ravel()])
    xb, pb = dev.upload(whole), dev.upload(np.asarray(pos, np.int32))
    fb = None if ff is None else dev.upload(np.asarray(ff, np.float32))
    if y is None:                                                  # in place
        dev.rope_scaled(xb.ptr + 4 * off, T, stride, hd, heads, n, mode, pb, sc, xb.ptr + 4 * off, stride, freq_factors=fb)
        return xb.read(np.float32, (whole.size,))[off:].reshape(x.shape)
    yb = dev.upload(np.full((T, y), 5.0, np.float32))
    dev.rope_scaled(xb.ptr + 4 * off, T, stride, hd, heads, n, mode, pb, sc, yb, y, freq_factors=fb)
    return yb.read(np.float32, (T, y))


CASES = [
    # T, heads, hd, n_dims, mode, base, factor, ext, orig, factors, first position
    (1, 40, 128, 128, 0, 500000.0, 16.0, 1.0, 8192, False, 131070),
    (1, 1, 2, 2, 2, 10000.0, 4.0, 0.0, 0, False, 0),
    (3, 40, 128, 128, 2, 10000.0, 8.0, 1.0, 4096, True, 1000000),
    (65, 7, 128, 96, 2, 10000.0, 4.0, 0.5, 4096, True, 20000),
    (33, 9, 80, 50, 0, 10000.0, 32.0, 1.0, 2048, False, 60000),
    (33, 9, 80, 50, 2, 10000.0, 32.0, 1.0, 2048, False, 60000),
    (17, 5, 99, 64, 0, 500000.0, 1.0, 0.0, 0, False, 5),
    (17, 5, 99, 64, 2, 500000.0, 1.0, 1.0, 8192, False, 5),
    (5, 3, 64, 4, 2, 10000.0, 2.0, 1.0, 2048, False, -40000),
    (2, 16, 1024, 1024, 0, 10000.0, 4.0, 1.0, 4096, True, 70000),
    (2, 16, 1024, 1024, 2, 10000.0, 4.0, 1.0, 4096, True, 70000),
    (4, 300, 64, 64, 40, 10000.0, 4.0, 1.0, 4096, False, 2147483000),
]


@pytest.mark.parametrize("T,heads,hd,n,mode,base,factor,ext,orig,with_ff,pos0", CASES)
def test_against_64_bits(dev, T, heads, hd, n, mode, base, factor, ext, orig, with_ff, pos0):
    rng = np.random.default_rng(T * hd + n + mode)
    stride = heads * hd + 16
    x = rng.standard_normal((T, stride)).astype(np.float32)
    ff = rng.uniform(1.0, 4.0, n // 2).astype(np.float32) if with_ff else None
    pos = pos0 + np.arange(T)
    sc = H.RopeScaling(freq_base=base, freq_scale=1.0 / factor, ext_factor=ext, n_ctx_orig=orig, attn_factor=1.25)
    f, m = R.frequencies(n, base, 1.0 / factor, ext, orig, ff, attn=1.25)
    want, tol = R.rope(x[:, :heads * hd].reshape(T, heads, hd), pos, n, mode != 0, f, m)
    for y, off in ((heads * hd, 0), (heads * hd + 12, 0), (None, 0), (None, 1)):
        got = run(dev, x, pos, heads, hd, n, mode, sc, ff, y=y, off=off)
        rows = got[:, :heads * hd].reshape(T, heads, hd)
        assert (np.abs(rows - want) <= tol).all(), (y, off, np.abs(rows - want).max(), tol.min())
        assert (rows[..., n:] == x[:, :heads * hd].reshape(T, heads, hd)[..., n:]).all()       # copied bit for bit
        rest = x[:, heads * hd:] if y is None else np.full((T, y - heads * hd), 5.0, np.float32)
        assert (got[:, heads * hd:] == rest).all()                                             # what is behind a row


def test_turned_back(dev):
    """Position -p is the transposed turn of p: a key turned and turned back by a context shift is the key."""
    rng = np.random.default_rng(3)
    T, heads, hd = 50, 8, 128
    x = rng.standard_normal((T, heads * hd)).astype(np.float32)
    pos = rng.integers(0, 131072, T)
    sc = H.RopeScaling(freq_base=500000.0, freq_scale=0.125)
    there = run(dev, x, pos, heads, hd, hd, 0, sc)
    back = run(dev, there, -pos, heads, hd, hd, 0, sc)
    # two turns, each off by 3 2^-24 of |p c| + |q s| <= sqrt 2 |(p, q)| (the first's error is turned with it)
    size = np.repeat(np.hypot(x[:, 0::2], x[:, 1::2]), 2, axis=1)
    assert (np.abs(back - x) <= 2 * np.sqrt(2) * 3.1 * 2.0 ** -24 * np.sqrt(2) * size).all()


@pytest.mark.parametrize("n", [2, 64, 128])
def test_table(dev, n):
    ff = np.random.default_rng(n).uniform(1.0, 3.0, n // 2).astype(np.float32)
    tab, fb = dev.alloc(4 * n), dev.upload(ff)
    for pos in (0, 1, 131071, -131071, 10 ** 6):
        sc = H.RopeScaling(freq_base=500000.0, freq_scale=1 / 32, ext_factor=1.0, n_ctx_orig=8192)
        f, m = R.frequencies(n, 500000.0, 1 / 32, 1.0, 8192, ff)
        dev.rope_scaled_table(dev.upload(np.array([pos], np.int32)), n, sc, tab, freq_factors=fb)
        got = tab.read(np.float32, (n // 2, 2))
        want = m * np.stack([np.cos(pos * f), np.sin(pos * f)], 1)
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + m * (np.abs(pos * f)[:, None] * 2.0 ** -50 + 1.5e-10)).all()


def test_values_that_are_not_finite_stay_in_their_pairs(dev):
    x = np.ones((1, 256), np.float32)
    x[0, 6], x[0, 9], x[0, 200] = np.nan, np.inf, np.inf
    sc = H.RopeScaling(freq_base=10000.0, freq_scale=0.5)
    got = run(dev, x, [9], 2, 128, 64, 0, sc)
    bad = np.flatnonzero(~np.isfinite(got[0]))
    assert bad.tolist() == [6, 7, 8, 9, 200]


@pytest.mark.parametrize("hd,n,mode", [(64, 64, 0), (64, 48, 2), (24, 20, 2), (10, 6, 0)])
def test_rope_s_operations(dev, hd, n, mode):
    """The angles are those of the table; products and sums flush subnormals and give one NaN, bit for bit."""
    rng = np.random.default_rng(hd + n)
    x = (rng.standard_normal((5, 3 * hd)) * 10.0 ** rng.choice([0, 0, -37.5, -38.5, 38], (5, 3 * hd))).astype(np.float32)
    x[1] = rng.standard_normal(3 * hd)
    x[2, ::7], x[3, ::5], x[3, 1::6] = np.nan, np.inf, -0.0
    x.view(np.uint32)[4, ::9] = 0xFFC01234
    sc = H.RopeScaling(freq_base=10000.0, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=256)
    pos, tab, cs = np.array([0, 1, 77, 1000, 131071], np.int32), dev.alloc(4 * n), []
    for p in pos:
        dev.rope_scaled_table(dev.upload(np.array([p], np.int32)), n, sc, tab)
        cs.append(tab.read(np.float32, (n // 2, 2)))
    c, s = np.stack(cs)[:, None].transpose(3, 0, 1, 2)

    def daz(v):
        return np.where(np.abs(v) < np.float32(2.0 ** -126), np.copysign(np.float32(0), v), v)

    def fin(v):
        return np.where(np.isnan(v), np.uint32(0x7FC00000).view(np.float32), daz(v))

    h = x.reshape(5, 3, hd)
    i, j = (np.arange(0, n, 2), np.arange(1, n, 2)) if mode == 0 else (np.arange(n // 2), n // 2 + np.arange(n // 2))
    want, a, b = h.copy(), daz(h[:, :, i]), daz(h[:, :, j])
    with np.errstate(all="ignore"):
        want[:, :, i] = fin(fin(a * c) - fin(b * s))
        want[:, :, j] = fin(fin(a * s) + fin(b * c))
    got = run(dev, x, pos, 3, hd, n, mode, sc)
    assert (got.view(np.uint32) == want.reshape(got.shape).view(np.uint32)).all()


def test_in_a_graph(dev):
    """A captured call reads the positions that are there when it is replayed."""
    rng = np.random.default_rng(8)
    T, heads, hd = 3, 4, 64
    x = rng.standard_normal((T, heads * hd)).astype(np.float32)
    sc = H.RopeScaling(freq_base=10000.0, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)
    f, m = R.frequencies(hd, 10000.0, 0.25, 1.0, 4096)
    xb, pb, yb = dev.upload(x), dev.upload(np.zeros(T, np.int32)), dev.alloc(x.nbytes)
    dev.graph_begin()
    dev.rope_scaled(xb, T, heads * hd, hd, heads, hd, 2, pb, sc, yb, heads * hd)
    g = dev.graph_end()
    for pos0 in (0, 7, 16000, 7):
        pos = pos0 + np.arange(T, dtype=np.int32)
        pb.write(pos)
        g.launch()
        want, tol = R.rope(x.reshape(T, heads, hd), pos, hd, True, f, m)
        assert (np.abs(yb.read(np.float32, want.shape) - want) <= tol).all()
    g.free()
