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
    stored into the same planes on a second stream: the same bits in every call."""
    other = H.Device(0)
    nh, nkv, D, n_kv, room = 32, 8, 128, 6000, 512
    E = nkv * D
    q = S.normal(203, nh * D).reshape(1, nh * D)
    bq, out = dev.upload(q), [dev.alloc(4 * nh * D) for _ in range(8)]
    x = S.normal(205, room * E).reshape(room, E) * np.float32(100.0)
    bx, bi = dev.upload(x), dev.upload(n_kv + np.arange(room, dtype=np.int64))
    ws = dev.alloc(dev.flash_attn_kv4_ws(1, D, nh, nkv, n_kv))
    want = bits = None
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
            got = o.read(np.float32, (1, nh, D))
            check(got, want, what=f"round {i}, call {j}")
            bits = got.view(np.uint32) if bits is None else bits
            assert (got.view(np.uint32) == bits).all(), (i, j)
        for c in (kc, vc, *big):
            c.free()
    other.close()


SHAPES = [  # n_head, n_head_kv, D, T, n_kv: one and several tokens, cells in splits and not, several columns a row and one,
            # an odd number of rows in an odd number of splits
    (32, 8, 128, 1, 8192), (14, 2, 64, 5, 3000), (32, 8, 128, 80, 1000), (8, 4, 256, 90, 500), (16, 1, 512, 3, 700),
    (32, 8, 64, 600, 333), (7, 1, 64, 1, 1056),
]


def attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, runs=None, mask=None):
    T = q.shape[0]
    out = dev.alloc(4 * T * nh * D).fill(0xFF)
    bq = dev.upload(q)
    br = None if runs is None else dev.upload(np.ascontiguousarray(runs, np.uint32))
    bm = None if mask is None else dev.upload(mask)
    dev.flash_attn_kv4(bq, T, nh * D, kc, vc, D, nh, nkv, scale, n_kv, out, nh * D, runs=br, mask=bm,
                       mask_stride=0 if mask is None else mask.shape[1])
    dev.sync()
    return out.read(np.float32, (T, nh, D))


def planes(dev, typ, k, v):
    """Caches that hold the rows k and v, and their images."""
    out = []
    for which, x in ((0, k), (1, v)):
        img = R.quantize(x, typ)
        c = dev.kv(x.shape[1], x.shape[0], typ)
        c.set_bytes(which, img)
        out += [img, c]
    return out


def rows(seed, n_kv, E, v_scale):
    return (S.normal(seed, n_kv * E).reshape(n_kv, E),
            S.normal(seed + 1, n_kv * E).reshape(n_kv, E) * np.asarray(v_scale, np.float32))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", SHAPES)
@pytest.mark.parametrize("v_scale", [0.5, 0.05, 3e-4])
def test_what_a_plane_held_before(dev, typ, nh, nkv, D, T, n_kv, v_scale):
    """A cell that held infinities or 5e5 and was written over leaves no trace: the bits of a plane that never held them,
    within the bound for values of any size."""
    E, scale = nkv * D, 1.0 / np.sqrt(D)
    k, v = rows(211, n_kv, E, v_scale)
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(213, T * nh * D).reshape(T, nh * D)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = n_kv - np.arange(T) % 70
    want = attention64(q, ki, vi, typ, nh, nkv, scale, runs)
    fresh = attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, runs)
    check(fresh, want, what="fresh")
    at = dev.upload(np.array([3, n_kv // 2], np.int64))
    for held, by_bytes in ((np.inf, True), (5e5, False)):
        x = np.full((2, E), held, np.float32)
        dev.kv_set_rows(vc, 1, dev.upload(x), 2, E, at)
        if by_bytes:
            vc.set_bytes(1, vi)
        else:
            dev.kv_set_rows(vc, 1, dev.upload(v[[3, n_kv // 2]]), 2, E, at)
        got = attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, runs)
        assert (got.view(np.uint32) == fresh.view(np.uint32)).all(), (held, row_errors(got, want).max())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", [s for s in SHAPES if s[3] > 2])
@pytest.mark.parametrize("by_mask", [False, True])
def test_scales_of_cells_that_others_see(dev, typ, nh, nkv, D, T, n_kv, by_mask):
    """Sequences side by side in one cache, their rows in one workgroup: the third one's values are 5e5, infinite in places,
    the others' from 3e-4 to 0.5."""
    E, scale, n_seq = nkv * D, 1.0 / np.sqrt(D), 5
    size = n_kv // n_seq
    seq = np.minimum(np.arange(n_kv) // size, n_seq - 1)
    k, v = rows(221, n_kv, E, np.array([0.5, 3e-4, 5e5, 0.05, 1e-3])[seq][:, None])
    v[2 * size + 7, 5::40] = np.inf
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(223, T * nh * D).reshape(T, nh * D)
    of = np.arange(T) % n_seq                         # the token's sequence
    runs = mask = None
    if by_mask:
        mask = np.where(seq[None] == of[:, None], 0.25, -np.inf).astype(np.float16)
    else:
        runs = np.zeros((T, 4), np.uint32)
        runs[:, 0], runs[:, 1] = of * size, np.where(of == n_seq - 1, n_kv, (of + 1) * size)
    with np.errstate(all="ignore"):
        fine = of != 2
        want = attention64(q[fine], ki, np.where((seq == 2)[:, None], np.uint8(0), vi), typ, nh, nkv, scale,
                           None if by_mask else runs[fine], mask[fine] if by_mask else None)
    got = attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, runs, mask)
    check(got[fine], want)
    assert not np.isfinite(got[~fine]).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", [s for s in SHAPES if s[1] > 1])
def test_scales_of_other_heads(dev, typ, nh, nkv, D, T, n_kv):
    """One KV head with values around 500 beside heads of 0.05 and 3e-4."""
    E, scale = nkv * D, 1.0 / np.sqrt(D)
    k, v = rows(231, n_kv, E, np.repeat(np.resize([500.0, 0.05, 3e-4], nkv), D)[None])
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(233, T * nh * D).reshape(T, nh * D)
    check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv), attention64(q, ki, vi, typ, nh, nkv, scale))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", SHAPES)
@pytest.mark.parametrize("order", [1, -1])
def test_scales_along_the_cells(dev, typ, nh, nkv, D, T, n_kv, order):
    """Values that grow from 1e-3 to 100 along the cells, or shrink: every wave and split meets scales of its own, and follows
    them from tile to tile."""
    E, scale = nkv * D, 1.0 / np.sqrt(D)
    k, v = rows(241, n_kv, E, (10.0 ** np.linspace(-3, 2, n_kv))[::order, None])
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(243, T * nh * D).reshape(T, nh * D)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = n_kv - np.arange(T) % 100
    for n in (None, runs):
        check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, n), attention64(q, ki, vi, typ, nh, nkv, scale, n))
    # a mask that takes turns: every tile is partly hidden
    mask = np.zeros((T, n_kv + 1), np.float16)
    mask[np.random.default_rng(9).random((T, n_kv + 1)) < 0.4] = -np.inf
    check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, None, mask), attention64(q, ki, vi, typ, nh, nkv, scale, None, mask))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", SHAPES)
@pytest.mark.parametrize("v_scale", [1e-5, 3e-4, 0.03, 1e4])
def test_values_of_any_size(dev, typ, nh, nkv, D, T, n_kv, v_scale):
    """Small values (their scales are f16 subnormals) and values near the end of f16's range keep the bound."""
    E, scale = nkv * D, 1.0 / np.sqrt(D)
    k, v = rows(251, n_kv, E, v_scale)
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(253, T * nh * D).reshape(T, nh * D)
    check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv), attention64(q, ki, vi, typ, nh, nkv, scale))
