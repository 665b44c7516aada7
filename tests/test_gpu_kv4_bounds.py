"""The bounds of a 4-bit K cache's blocks (tsr_hip_kv4_bounds), bit for bit."""
import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P

pytestmark = pytest.mark.gpu


def read(buf, E, D, nb):
    return P.words(buf.read(np.uint32, (E // D, nb, D)))


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("D,heads,n,block", [(64, 1, 1, 32), (64, 2, 333, 32), (128, 3, 200, 64), (256, 1, 129, 96), (512, 1, 70, 1024),
                                             (128, 8, 1000, 128), (64, 5, 64, 32), (128, 1, 31, 32)])
def test_all_blocks(dev, typ, D, heads, n, block):
    E, size = heads * D, n + 45                                    # (cells behind the last: not in use, of other values)
    kv, values = P.fill(dev, P.cache_rows(n + D, size, E) * np.linspace(1, 9, size, dtype=np.float32)[:, None], typ)
    nb = -(-size // block)
    out = dev.upload(np.full(E * nb, 0x12345678, np.uint32))
    dev.kv4_bounds(kv, D, block, n, out)
    lo, hi = P.bounds(values, D, block, n)
    got_lo, got_hi = read(out, E, D, nb)
    used = lo.shape[1]
    assert (got_lo[:, :used] == lo).all() and (got_hi[:, :used] == hi).all()
    assert (out.read(np.uint32, (heads, nb, D))[:, used:] == 0x12345678).all()                 # blocks without a cell


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
def test_new_cells(dev, typ):
    """Only the blocks of the cells [lo, hi) are made, of their cells below hi; a captured call reads lo and hi when it runs."""
    D, E, size, block = 64, 128, 700, 32
    kv, values = P.fill(dev, P.cache_rows(5, size, E), typ)
    nb = -(-size // block)
    out, cells = dev.alloc(4 * E * nb), dev.upload(np.zeros(2, np.uint32))
    n_new, n_kv = 70, 690
    dev.graph_begin()
    dev.kv4_bounds(kv, D, block, n_kv, out, cells=cells, n_new=n_new)
    g = dev.graph_end()
    for lo, hi in ((0, 1), (31, 32), (31, 33), (5, 75), (100, 170), (640, 710), (689, 1000), (690, 691), (10, 10), (20, 3),
                   (4000000000, 4000000001), (64, 96)):
        out.write(np.full(E * nb, 0x7F807F80, np.uint32))
        cells.write(np.array([lo, hi], np.uint32))
        g.launch()
        got = out.read(np.uint32, (E // D, nb, D))
        end = min(hi, n_kv)
        touched = set() if lo >= end else set(range(lo // block, -(-end // block)))
        for b in range(nb):
            if b in touched:
                want = P.bounds(values[b * block:min(end, (b + 1) * block)], D, block)
                for x, y in zip(P.words(got[:, b:b + 1]), want):
                    assert (x == y).all(), (lo, hi, b)
            else:
                assert (got[:, b] == 0x7F807F80).all(), (lo, hi, b)
    g.free()


def test_scales_that_are_not_finite_count_as_the_largest(dev):
    D = 64
    x = P.cache_rows(9, 64, D)
    for typ in (R.Q4_0, R.Q4_1):
        img = R.quantize(x, typ).reshape(64, 2, -1)
        for cell, d in ((3, np.inf), (40, -np.inf)):
            img[cell, 0, :2] = np.array([d], np.float16).view(np.uint8)
        kv = dev.kv(D, 64, typ)
        kv.set_bytes(0, img)
        n, d, m = R.split(img.reshape(64, -1), typ)
        d = np.clip(d, -65504, 65504)
        m = -8.0 * d if typ == R.Q4_0 else m
        values = (d[..., None] * n + m[..., None]).reshape(64, D).astype(np.float32)
        out = dev.alloc(4 * D * 2)
        dev.kv4_bounds(kv, D, 32, 64, out)
        for got, want in zip(read(out, D, D, 2), P.bounds(values, D, 32)):
            assert np.isfinite(got).all() and (got == want).all()


def test_every_cell_scores_at_most_its_block(dev):
    """max(q lo, q hi) summed is at least q k of every cell, in exact sums."""
    D, n, block = 128, 500, 64
    kv, values = P.fill(dev, P.cache_rows(2, n, D), R.Q4_0)
    out = dev.alloc(4 * D * 8)
    dev.kv4_bounds(kv, D, block, n, out)
    lo, hi = read(out, D, D, 8)
    q = np.random.default_rng(1).standard_normal((20, D))
    most = np.maximum(q[:, None] * lo[0], q[:, None] * hi[0]).sum(-1)
    s = q @ values.astype(np.float64).T
    for b in range(8):
        assert (s[:, b * block:(b + 1) * block] <= most[:, b:b + 1] + 1e-9).all()
