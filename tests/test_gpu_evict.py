"""The cells that are kept (tsr_hip_kv_pick) and their move (tsr_hip_kv_gather), bit for bit."""
import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P
import tsr_hip as H

pytestmark = pytest.mark.gpu


def pick_ref(w, keep, first, last):
    n = w.size
    mid = np.arange(first, n - last)
    key = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    nan = np.isnan(w[mid])
    order = np.lexsort((mid, nan, -key))                            # the largest first, numbers ahead of NaNs, low cells first
    return np.sort(np.concatenate([np.arange(first), mid[order[:keep - first - last]], np.arange(n - last, n)]))


def pick(dev, w, keep, first, last, kept=True):
    wb = dev.upload(w)
    idx, kb = dev.upload(np.full(keep + 2, -9, np.int64)), dev.upload(np.full(keep + 2, -9, np.float32))
    dev.kv_pick(wb, w.size, keep, first, last, idx, kept=kb if kept else None)
    i, k = idx.read(np.int64, (keep + 2,)), kb.read(np.float32, (keep + 2,))
    assert (i[keep:] == -9).all() and (k[keep:] == -9).all()
    if not kept:
        assert (k == -9).all()
    return i[:keep], k[:keep]


@pytest.mark.parametrize("n,keep,first,last", [
    (1, 1, 0, 0), (2, 1, 0, 0), (5, 5, 1, 1), (64, 10, 2, 3), (65, 64, 0, 0), (1000, 1, 0, 0), (1000, 999, 0, 0), (777, 300, 300, 0),
    (777, 300, 100, 200), (4096, 2000, 4, 64), (4097, 2000, 4, 64), (16384, 100, 0, 1), (20000, 15000, 4, 500), (65536, 16384, 4, 256),
    (65537, 30000, 4, 256), (131071, 65000, 0, 0)])
def test_pick(dev, n, keep, first, last):
    rng = np.random.default_rng(n + keep)
    w = np.exp(3 * rng.standard_normal(n)).astype(np.float32)
    w[rng.random(n) < 0.1] = 0.0
    want = pick_ref(w, keep, first, last)
    for kept in (True, False):
        idx, k = pick(dev, w, keep, first, last, kept)
        assert (idx == want).all()
        if kept:
            assert (k == w[want]).all()


def test_pick_ties_and_odd_values(dev):
    """Equal weights go to the lowest cells (zeros of either sign are equal), NaNs are below everything, -inf included."""
    n = 3000
    rng = np.random.default_rng(1)
    for w in (np.zeros(n), np.where(rng.random(n) < 0.5, 0.0, -0.0), rng.integers(0, 3, n).astype(float), np.full(n, np.nan),
              np.where(rng.random(n) < 0.3, np.nan, rng.standard_normal(n)), np.where(rng.random(n) < 0.5, -np.inf, np.nan),
              rng.choice([np.inf, -np.inf, 1e-42, -1e-42, 3e38, 0.0], n), 1.0 + rng.integers(0, 40, n) * 2.0 ** -23):
        w = w.astype(np.float32)
        for keep, first, last in ((1000, 0, 0), (1500, 7, 9), (2999, 0, 0), (3000, 0, 0)):
            assert (pick(dev, w, keep, first, last)[0] == pick_ref(w, keep, first, last)).all()


def cache(dev, typ, E, n, which, seed):
    rng = np.random.default_rng(seed)
    img = rng.integers(0, 256, (n, E // 32 * H.KV_BLOCK_BYTES[typ]), dtype=np.uint8)
    kv = dev.kv(E, n, typ)
    kv.set_bytes(which, img)
    return kv, img


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("typ", [H.KV_Q8_0, H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("E,size,n", [(64, 1, 1), (64, 100, 33), (128, 333, 200), (1024, 97, 97), (192, 500, 16), (320, 70, 65)])
def test_gather(dev, typ, which, E, size, n):
    """Into another cache (of another length) and into itself: any order, cells twice, ascending; cells behind stay."""
    rng = np.random.default_rng(E + size + n)
    for idx in (np.sort(rng.permutation(size)[:n]), rng.integers(0, size, n), np.arange(n)[::-1] + (size - n)):
        ib = dev.upload(np.ascontiguousarray(idx, np.int64))
        src, img = cache(dev, typ, E, size, which, 5)
        dst, was = cache(dev, typ, E, n + 40, which, 6)
        dev.kv_gather(dst, src, which, ib, n)
        got = dst.get_bytes(which).reshape(n + 40, -1)
        assert (got[:n] == img[idx]).all() and (got[n:] == was[n:]).all()
        assert (src.get_bytes(which).reshape(size, -1) == img).all()
        dev.kv_gather(src, src, which, ib, n)
        got = src.get_bytes(which).reshape(size, -1)
        assert (got[:n] == img[idx]).all() and (got[n:] == img[n:]).all()


@pytest.mark.parametrize("typ", [H.KV_Q8_0, H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("which", [0, 1])
def test_gather_indices_outside(dev, typ, which):
    """They leave their cells as they were and raise the flag, in another cache and within one."""
    E, size, n = 128, 90, 70
    idx = np.arange(n, dtype=np.int64) + 15
    idx[[3, 40, 41, 69]] = (-1, 90, 2 ** 40, -2 ** 62)
    fine = np.ones(n, bool)
    fine[[3, 40, 41, 69]] = False
    ib, bad = dev.upload(idx), dev.upload(np.zeros(1, np.int32))
    src, img = cache(dev, typ, E, size, which, 1)
    dst, was = cache(dev, typ, E, n, which, 2)
    dev.kv_gather(dst, src, which, ib, n, bad=bad)
    assert bad.read(np.int32, (1,))[0] == 1
    assert (dst.get_bytes(which).reshape(n, -1) == np.where(fine[:, None], img[np.where(fine, idx, 0)], was)).all()
    dev.get_flags()
    dev.kv_gather(src, src, which, ib, n)
    assert dev.get_flags() == 1 and dev.get_flags() == 0
    got = src.get_bytes(which).reshape(size, -1)
    assert (got[:n] == np.where(fine[:, None], img[np.where(fine, idx, 0)], img[:n])).all() and (got[n:] == img[n:]).all()


def test_gather_in_a_graph(dev):
    """Captured within a cache with its workspace, replayed with other lists; without a workspace it is refused."""
    E, size, n = 128, 200, 100
    kv, img = cache(dev, H.KV_Q4_1, E, size, 1, 3)
    ib, ws = dev.upload(np.zeros(n, np.int64)), dev.alloc(dev.kv_gather_ws(kv, n))
    dev.graph_begin()
    with pytest.raises(H.TsrHipError):
        dev.kv_gather(kv, kv, 1, ib, n)
    dev.kv_gather(kv, kv, 1, ib, n, ws=ws)
    g = dev.graph_end()
    rng = np.random.default_rng(0)
    for _ in range(4):
        idx = rng.permutation(size)[:n]
        ib.write(idx.astype(np.int64))
        g.launch()
        img = np.concatenate([img[idx], img[n:]])
        assert (kv.get_bytes(1).reshape(size, -1) == img).all()
    g.free()


def test_evicted_as_it_is_used(dev):
    """Weights of a few tokens, the cells that are kept, K and V moved to the front: attention over them is attention over the
    kept cells, and their weights go on."""
    import weights4_ref as W
    nh, nkv, D, n, keep = 8, 2, 64, 700, 300
    E = nkv * D
    k, v = P.cache_rows(1, n, E), P.cache_rows(2, n, E)
    ki, vi = R.quantize(k, R.Q4_0), R.quantize(v, R.Q4_0)
    kc, vc = dev.kv(E, n, R.Q4_0), dev.kv(E, n, R.Q4_0)
    kc.set_bytes(0, ki)
    vc.set_bytes(1, vi)
    rng = np.random.default_rng(0)
    acc, kept, idx = dev.upload(np.zeros(n, np.float32)), dev.alloc(4 * n), dev.alloc(8 * keep)
    for t in range(5):
        q = rng.standard_normal((1, nh * D)).astype(np.float32)
        dev.attn_weights_kv4(dev.upload(q), 1, nh * D, kc, D, nh, nkv, 0.125, n, acc, before=acc)
    w = acc.read(np.float32, (n,))
    dev.kv_pick(acc, n, keep, 4, 100, idx, kept=kept)
    dev.kv_gather(kc, kc, 0, idx, keep)
    dev.kv_gather(vc, vc, 1, idx, keep)
    cells = idx.read(np.int64, (keep,))
    assert (cells == pick_ref(w, keep, 4, 100)).all()
    q = rng.standard_normal((1, nh * D)).astype(np.float32)
    out = dev.alloc(4 * nh * D)
    dev.flash_attn_kv4(dev.upload(q), 1, nh * D, kc, vc, D, nh, nkv, 0.125, keep, out, nh * D)
    R.check(out.read(np.float32, (1, nh, D)), *R.attention(q, ki[cells], vi[cells], R.Q4_0, D, nh, nkv, 0.125))
    dev.attn_weights_kv4(dev.upload(q), 1, nh * D, kc, D, nh, nkv, 0.125, keep, kept, before=kept)
    R.check(kept.read(np.float32, (keep,)), *W.weights(q, ki[cells], R.Q4_0, D, nh, nkv, 0.125, keep, before=w[cells]))
