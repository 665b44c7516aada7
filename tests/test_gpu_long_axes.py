"""More cells than the threads along one axis of a launch, of which there are fewer than 2^32 (tsr_hip_kv_gather,
tsr_hip_attn_weights_kv4)."""
import numpy as np
import pytest

import tsr_hip as H
from test_gpu_evict import cache

pytestmark = pytest.mark.gpu


def test_gather(dev):
    """2^28 cells of q8_0 and some, of a small cache's: the first, those at the axis' end, the last, and what lies behind."""
    E, size, n, spare = 64, 100, (1 << 28) + 1000, 16
    src, img = cache(dev, H.KV_Q8_0, E, size, 0, 1)
    dst = dev.kv(E, n + spare, H.KV_Q8_0)
    idx = dev.upload(np.resize(np.random.default_rng(2).permutation(size).astype(np.int64), n))
    order = idx.read(np.int64, (size,))
    dev.kv_gather(dst, src, 0, idx, n)
    row = dst.row_bytes
    for c0, cells in ((0, 300), ((1 << 27) - 50, 100), ((1 << 28) - 500, 1000), (n - 100, 100)):
        got = dst.get_bytes(0, c0 * row, cells * row).reshape(cells, row)
        assert (got == img[order[(c0 + np.arange(cells)) % size]]).all(), c0
    assert (dst.get_bytes(0, n * row, spare * row) == 0).all()
    for x in (idx, dst, src):
        x.free()


def test_weights(dev):
    """2^30 cells and some, all alike: each gets the same weight."""
    n, D, nh = (1 << 30) + 1000, 64, 2
    kc, out = dev.kv(D, n, H.KV_Q4_0), dev.alloc(4 * n)
    for c0 in (0, n - 2000):
        H.BufferPart(out, 4 * c0, 8000).fill(0x55)
    q = np.random.default_rng(1).standard_normal((1, nh * D)).astype(np.float32)
    dev.attn_weights_kv4(dev.upload(q), 1, nh * D, kc, D, nh, 1, 0.125, n, out)
    for c0 in (0, 1 << 29, n - 2000):
        got = H.BufferPart(out, 4 * c0, 8000).read(np.float32, (2000,)).astype(np.float64)
        # sums of whole numbers; a row's inverse and its weight are rounded once each, and their sum
        assert (np.abs(got * n - nh) <= nh * 3 * 2.0 ** -24 + nh * 2.0 ** -22).all(), c0
    kc.free()
    out.free()
