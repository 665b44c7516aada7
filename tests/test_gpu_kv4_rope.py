"""ROPE + SET_ROWS_KV into K and V caches of different lengths: a cell outside either of them is stored in neither."""
import numpy as np
import pytest

import tsr_hip as H
import tsr_synth as S
from helpers import assert_bits_equal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tk,tv", [(0, 0), (1, 1), (2, 1), (0, 2), (1, 0)])
@pytest.mark.parametrize("nk,nv", [(100, 50), (50, 100)])
def test_a_cell_outside_either_cache(dev, tk, tv, nk, nv):
    D, nh, nkv = 64, 4, 2
    E, w = nkv * D, (nh + 2 * nkv) * D
    cells = np.array([7, 70, 49, 50, -1, 99, 100, 1 << 33, 0], np.int64)
    T, inside = len(cells), (cells >= 0) & (cells < min(nk, nv))
    x = S.normal(19, T * w).reshape(T, w)
    pos = dev.upload(np.arange(T, dtype=np.int32))
    a, b = dev.upload(x), dev.upload(x)
    kc, vc, k2, v2 = dev.kv(E, nk, tk), dev.kv(E, nv, tv), dev.kv(E, nk, tk), dev.kv(E, nv, tv)
    bad = dev.upload(np.zeros(1, np.int32))
    dev.rope_kv(a, T, w, D, nh, nkv, D, H.ROPE_NORMAL, pos, 10000.0, kc, vc, dev.upload(cells), bad)
    # its three ops, the rows inside both caches alone
    dev.rope(b, T, w, D, nh + nkv, D, H.ROPE_NORMAL, pos, 10000.0, b, w)
    dev.sync()
    rows = b.read(np.float32, (T, w))
    assert_bits_equal(a.read(np.float32, (T, w)), rows, "rotated rows")
    part, idx = dev.upload(rows[inside]), dev.upload(cells[inside])
    for kv, which, at in ((k2, 0, nh * D), (v2, 1, (nh + nkv) * D)):
        dev.kv_set_rows(kv, which, part.ptr + 4 * at, int(inside.sum()), w, idx)
    dev.sync()
    assert bad.read(np.int32, (1,))[0] == 1
    for got, want, which in ((kc, k2, 0), (vc, v2, 1)):
        assert (got.get_bytes(which) == want.get_bytes(which)).all(), which
    # all inside both: no flag
    bad.fill(0)
    dev.rope_kv(a, 1, w, D, nh, nkv, D, H.ROPE_NORMAL, pos, 10000.0, kc, vc, dev.upload(np.array([49], np.int64)), bad)
    dev.sync()
    assert bad.read(np.int32, (1,))[0] == 0
