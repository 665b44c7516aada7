"""GPU attention over 4-bit KV caches: what the scales of cells that a row does not see, and of cells at other times, do to
its results, against a plain computation in 64 bits. Bounds are on the length of a row's error, which a value rounded to 11
bits anywhere passes by far."""
import numpy as np
import pytest

import kv4_ref as R
import tsr_hip as H
import tsr_synth as S
from test_gpu_attn4 import caches

pytestmark = pytest.mark.gpu
TYPES = [H.KV_Q4_0, H.KV_Q4_1]
# A row's error by its length. On normal values with scores of spread 1 it is 2^-21 on average and 2^-19 leaves four times
# that: test_gpu_attn4.test_precision has the terms.
BOUND = 2.0 ** -19


def attention64(q, kimg, vimg, typ, nh, nkv, scale, runs=None, mask=None):
    """softmax(scale q K^T + mask) V in 64 bits, [T, nh, D]; rows that see nothing are 0."""
    T, n_kv, G = q.shape[0], kimg.shape[0], nh // nkv
    K, V = (R.values(i, typ).reshape(n_kv, nkv, -1) for i in (kimg, vimg))
    see, add = R.visible(T, n_kv, runs, mask)
    q = np.asarray(q, np.float64).reshape(T, nh, -1)
    out = np.zeros(q.shape)
    for h in range(nh):
        s = np.where(see, q[:, h] @ K[:, h // G].T * scale + add, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isinf(top), 0.0, top))
        out[:, h] = p @ V[:, h // G] / np.maximum(p.sum(1, keepdims=True), 1e-300)
    return out


def row_errors(got, want):
    """The length of each row's error by the row's own length, [T, nh]."""
    d = np.linalg.norm(np.asarray(got, np.float64).reshape(want.shape) - want, axis=-1)
    return d / np.maximum(np.linalg.norm(want, axis=-1), 1e-300)


def check(got, want, bound=BOUND, what=""):
    e = row_errors(got, want)
    assert (e <= bound).all(), (what, e.max(), np.unravel_index(e.argmax(), e.shape))


@pytest.mark.parametrize("typ", TYPES)
def test_stores_into_other_cells_meanwhile(dev, typ):
    """Rows of a sequence attended to on one stream while larger rows of another one, whose cells they do not see, are
    stored into the same planes on a second stream. (Values of 100 against 0.5: 2^8 times the scale, and 2^-33 of the largest
    scale is still 2^-24 of the values'.)"""
    other = H.Device(0)
    nh, nkv, D, n_kv, room = 32, 8, 128, 6000, 512
    E = nkv * D
    q = S.normal(203, nh * D).reshape(1, nh * D)
    bq, out = dev.upload(q), [dev.alloc(4 * nh * D) for _ in range(8)]
    x = S.normal(205, room * E).reshape(room, E) * np.float32(100.0)
    bx, bi = dev.upload(x), dev.upload(n_kv + np.arange(room, dtype=np.int64))
    ws = dev.alloc(dev.flash_attn_kv4_ws(1, D, nh, nkv, n_kv))
    want = None
    for i in range(6):
        ki, kc, vi, vc = caches(dev, typ, n_kv, E, 207, kv_size=n_kv, v_scale=0.5)
        big = [dev.kv(E, n_kv + room, typ) for _ in range(2)]
        for c, img, which in zip(big, (ki, vi), (0, 1)):
            c.set_bytes(which, img)
        if want is None:
            want = attention64(q, ki, vi, typ, nh, nkv, 0.1)
        dev.sync()
        for j, o in enumerate(out):
            dev.flash_attn_kv4(bq, 1, nh * D, big[0], big[1], D, nh, nkv, 0.1, n_kv, o, nh * D, ws=ws)
            if j == i:
                for which in (0, 1):
                    dev.kv_set_rows(big[which], which, bx, room, E, bi, stream=other.stream)
        dev.sync(other.stream)
        dev.sync()
        for j, o in enumerate(out):
            check(o.read(np.float32, (1, nh, D)), want, what=f"round {i}, call {j}")
        for c in (kc, vc, *big):
            c.free()
    other.close()
