"""GPU attention over 4-bit KV caches (tsr_hip_flash_attn_kv4) against a plain computation in 64 bits, within the bound
that kv4_ref derives from the kernels' arithmetic."""
import math

import numpy as np
import pytest

import kv4_ref as R
import tsr_hip as H
import tsr_synth as S

pytestmark = pytest.mark.gpu
TYPES = [H.KV_Q4_0, H.KV_Q4_1]
LOWEST = np.float16(-65504.0)


def caches(dev, typ, n_kv, E, seed, kv_size=None, v_scale=1.0):
    """K and V images of n_kv cells and the caches that hold them (behind them: blocks whose scales are NaN and inf)."""
    kv_size = kv_size or n_kv
    out = []
    for which in (0, 1):
        x = S.normal(seed + which, n_kv * E).reshape(n_kv, E) * np.float32(v_scale if which else 1.0)
        img = np.empty((kv_size, E // 32 * R.BLOCK[typ]), np.uint8)
        img[:n_kv] = R.quantize(x, typ)
        img[n_kv:] = 0x7C if which else 0x7E
        c = dev.kv(E, kv_size, typ)
        c.set_bytes(which, img)
        out += [img[:n_kv], c]
    return out


def attend(dev, q, kc, vc, D, nh, nkv, scale, n_kv, runs=None, mask=None, mask_stride=0, q_pad=0, out_pad=0, ws=None):
    T, K = q.shape[0], nh * D
    qq = np.full((T, K + q_pad), np.nan, np.float32)
    qq[:, :K] = q
    out = dev.alloc(4 * T * (K + out_pad)).fill(0xFF)
    bq = dev.upload(qq)
    br = None if runs is None else dev.upload(np.ascontiguousarray(runs, np.uint32))
    bm = None if mask is None else dev.upload(mask)
    dev.flash_attn_kv4(bq, T, K + q_pad, kc, vc, D, nh, nkv, scale, n_kv, out, K + out_pad, runs=br, mask=bm,
                       mask_stride=mask_stride or (0 if mask is None else mask.shape[1]), ws=ws)
    dev.sync()
    got = out.read(np.float32, (T, K + out_pad))
    assert (got[:, K:].view(np.uint32) == 0xFFFFFFFF).all()
    return got[:, :K].reshape(T, nh, D)


def causal(T, hist):
    r = np.zeros((T, 4), np.uint32)
    r[:, 1] = hist + 1 + np.arange(T)
    return r


SHAPES = [  # n_head, n_head_kv, D, T, hist
    (1, 1, 64, 1, 0), (14, 2, 64, 1, 200), (32, 8, 128, 1, 31), (32, 8, 128, 1, 1000), (8, 1, 128, 1, 5000),
    (8, 4, 256, 1, 333), (2, 1, 512, 1, 100), (64, 1, 64, 1, 95), (6, 2, 128, 3, 65), (5, 1, 64, 17, 40),
    (32, 8, 128, 40, 0), (14, 2, 64, 100, 37), (8, 4, 256, 19, 70), (4, 2, 512, 9, 33), (8, 8, 64, 70, 130),
    (16, 2, 128, 130, 300),
]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,hist", SHAPES)
def test_causal(dev, typ, nh, nkv, D, T, hist):
    n_kv = hist + T
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 11, kv_size=n_kv + 45)
    q = S.normal(13, T * nh * D).reshape(T, nh * D)
    scale = 1.0 / math.sqrt(D)
    runs = causal(T, hist)
    want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, scale, runs)
    R.check(attend(dev, q, kc, vc, D, nh, nkv, scale, n_kv, runs, q_pad=4, out_pad=8), want, tol, "causal")
    # n_kv beyond the rows' cells (a captured graph's bound): the cells behind hold NaN and infinities
    R.check(attend(dev, q, kc, vc, D, nh, nkv, scale, n_kv + 45, runs), want, tol, "a wider bound")


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,n_kv", [(8, 2, 64, 333), (4, 2, 128, 700), (2, 1, 256, 97)])
def test_runs(dev, typ, nh, nkv, D, n_kv):
    """Rows of two runs, empty rows, runs past the end, runs in reverse order, and overlapping ones."""
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 21)
    runs = np.array([[0, n_kv, 0, 0], [0, 0, 0, 0], [5, 6, 0, 0], [0, 4, n_kv - 33, n_kv], [40, 20, 70, 60],
                     [n_kv - 1, n_kv + 1000, 0, 0], [32, 64, 0, 0], [31, 33, 63, 65], [n_kv, n_kv + 5, 0, 0],
                     [64, 96, 0, 32], [0, 0, 1, 2], [10, 80, 50, 90]] * 3, np.uint32)
    T = len(runs)
    q = S.normal(23, T * nh * D).reshape(T, nh * D)
    want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, 0.1, np.minimum(runs, n_kv))
    got = attend(dev, q, kc, vc, D, nh, nkv, 0.1, n_kv, runs)
    R.check(got, want, tol, "runs")
    assert (got[[1, 4, 8]] == 0).all()
    for t in (0, 1, 5):                                # a row alone
        R.check(attend(dev, q[t:t + 1], kc, vc, D, nh, nkv, 0.1, n_kv, runs[t:t + 1]), want[t:t + 1], tol[t:t + 1], t)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T", [1, 6, 90])
def test_f16_mask(dev, typ, T):
    nh, nkv, D, n_kv = 8, 2, 128, 211
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 31)
    rng = np.random.default_rng(T)
    mask = np.full((T, n_kv + 7), np.nan, np.float16)
    mask[:, :n_kv] = rng.standard_normal((T, n_kv))
    mask[:, :n_kv][rng.random((T, n_kv)) < 0.4] = -np.inf
    mask[0, :n_kv] = LOWEST                            # the type's lowest value everywhere: an even mean
    if T > 1:
        mask[1, :n_kv] = -np.inf                       # nothing left
        mask[2, :n_kv] = LOWEST
        mask[2, 9] = -3.0
        mask[3, :n_kv] = -np.inf
        mask[3, n_kv - 1] = 0.5
    q = S.normal(33, T * nh * D).reshape(T, nh * D)
    want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, 0.2, None, mask)
    got = attend(dev, q, kc, vc, D, nh, nkv, 0.2, n_kv, mask=mask)
    R.check(got, want, tol, "mask")
    if T > 1:
        assert (got[1] == 0).all()
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 0], runs[:, 1] = 3, 150 + np.arange(T) % 40
    want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, 0.2, runs, mask)
    R.check(attend(dev, q, kc, vc, D, nh, nkv, 0.2, n_kv, runs, mask), want, tol, "mask and runs")


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T", [2, 40])
def test_masked_infinities_and_nan(dev, typ, T):
    """Cells with infinite and NaN scales reach the rows that see them and no other."""
    nh, nkv, D, n_kv = 4, 2, 64, 150
    E = nkv * D
    ki, kc, vi, vc = caches(dev, typ, n_kv, E, 41)
    for img, c, which, cell, word in ((ki, kc, 0, 70, 0x7C00), (vi, vc, 1, 71, 0x7C00), (vi, vc, 1, 72, 0x7E01),
                                      (ki, kc, 0, 73, 0x7E01)):
        b = img[cell].reshape(-1, R.BLOCK[typ])
        b[:, 0], b[:, 1] = word & 255, word >> 8
        c.set_bytes(which, img[cell], cell * c.row_bytes)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1], runs[:, 2], runs[:, 3] = 70, 74, n_kv
    runs[0] = [0, n_kv, 0, 0]                          # this one sees them
    q = S.normal(43, T * nh * D).reshape(T, nh * D)
    got = attend(dev, q, kc, vc, D, nh, nkv, 0.125, n_kv, runs)
    want, tol = R.attention(q[1:], ki, vi, typ, D, nh, nkv, 0.125, runs[1:])
    R.check(got[1:], want, tol, "rows that do not see them")
    assert not np.isfinite(got[0]).any()
    mask = np.zeros((T, n_kv), np.float16)
    mask[1:, 70:74] = -np.inf
    got = attend(dev, q, kc, vc, D, nh, nkv, 0.125, n_kv, mask=mask)
    want, tol = R.attention(q[1:], ki, vi, typ, D, nh, nkv, 0.125, None, mask[1:])
    R.check(got[1:], want, tol, "rows whose mask hides them")
    # a query row that is not finite stays alone
    q[T - 1, 5] = np.nan
    got = attend(dev, q, kc, vc, D, nh, nkv, 0.125, n_kv, mask=mask)
    R.check(got[1:T - 1], want[:T - 2], tol[:T - 2], "beside a NaN query")
    assert np.isnan(got[T - 1, 0]).all() and np.isfinite(got[T - 1, 1]).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("q_scale,v_scale,scale", [(1e-20, 1e-6, 1e19), (1e30, 3e4, 1e-31), (30.0, 1.0, 0.125),
                                                   (0.0, 1e-3, 1.0)])
def test_ranges(dev, typ, q_scale, v_scale, scale):
    """Queries and values far from 1, scores that single cells win, queries of zero."""
    nh, nkv, D, T, n_kv = 4, 2, 64, 5, 600
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 51, v_scale=v_scale)
    q = (S.normal(53, T * nh * D) * np.float32(q_scale)).reshape(T, nh * D).astype(np.float32)
    want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, np.float64(np.float32(scale)))
    R.check(attend(dev, q, kc, vc, D, nh, nkv, scale, n_kv), want, tol, "ranges")


def test_a_huge_value_written_before(dev):
    """What a plane held once does not cost later results their precision beyond the bound."""
    nh, nkv, D, n_kv = 4, 2, 64, 200
    E = nkv * D
    ki, kc, vi, vc = caches(dev, H.KV_Q4_0, n_kv, E, 61)
    dev.kv_set_rows(vc, 1, dev.upload(np.full((1, E), 5e5, np.float32)), 1, E, dev.upload(np.array([3], np.int64)))
    vc.set_bytes(1, vi[3], 3 * vc.row_bytes)
    q = S.normal(63, nh * D).reshape(1, nh * D)
    want, tol = R.attention(q, ki, vi, H.KV_Q4_0, D, nh, nkv, 0.125)
    R.check(attend(dev, q, kc, vc, D, nh, nkv, 0.125, n_kv), want, 4 * tol, "after a huge value")


def test_graph_replays_follow_runs_and_cells(dev):
    """A captured call with a workspace of its own, replayed with eager work between: each replay attends over the runs and
    cells of its time; a second graph with a workspace of its own in turn with it."""
    nh, nkv, D, kv_size = 32, 8, 128, 3000
    typ = H.KV_Q4_0
    E, scale = nkv * D, 1.0 / math.sqrt(D)
    ki, kc, vi, vc = caches(dev, typ, kv_size, E, 71)
    n_ws = dev.flash_attn_kv4_ws(1, D, nh, nkv, kv_size)
    assert n_ws > 0
    q = S.normal(73, 8 * nh * D).reshape(8, nh * D)
    bq, br = dev.upload(q[0]), dev.upload(causal(1, 0))
    outs, graphs, wss = [], [], []
    for i in range(2):
        out, ws = dev.alloc(4 * nh * D), dev.alloc(n_ws)
        dev.graph_begin()
        try:
            dev.flash_attn_kv4(bq, 1, nh * D, kc, vc, D, nh, nkv, scale, kv_size, out, nh * D, runs=br, ws=ws)
        finally:
            graphs.append(dev.graph_end())
        outs.append(out)
        wss.append(ws)
    for step, hist in enumerate((0, 40, 2999, 31, 1500)):
        row = S.normal(90 + step, E).reshape(1, E)
        cell = np.array([hist], np.int64)
        for c, which, img in ((kc, 0, ki), (vc, 1, vi)):
            dev.kv_set_rows(c, which, dev.upload(row), 1, E, dev.upload(cell))
            img[hist] = R.quantize(row, typ)[0]
        bq.write(q[step])
        br.write(causal(1, hist))
        for g in graphs:
            g.launch()
        dev.sync()
        want, tol = R.attention(q[step:step + 1], ki[:hist + 1], vi[:hist + 1], typ, D, nh, nkv, scale)
        eager = attend(dev, q[step:step + 1], kc, vc, D, nh, nkv, scale, kv_size, causal(1, hist))
        for out in outs:
            got = out.read(np.float32, (1, nh, D))
            assert (got.view(np.uint32) == eager.view(np.uint32)).all()
            R.check(got, want, tol, f"replay {step}")
    # without a workspace of its own a captured call is refused, and records nothing
    dev.graph_begin()
    try:
        with pytest.raises(H.TsrHipError) as e:
            dev.flash_attn_kv4(bq, 1, nh * D, kc, vc, D, nh, nkv, scale, kv_size, outs[0], nh * D, runs=br)
        assert e.value.code == -1
    finally:
        dev.graph_end().free()
    for g in graphs:
        g.free()


def test_same_bits_every_time(dev):
    """Splits join in a fixed order: repeated calls, with a workspace or the context's scratch, give the same bits."""
    nh, nkv, D, n_kv = 32, 8, 128, 5000
    ki, kc, vi, vc = caches(dev, H.KV_Q4_1, n_kv, nkv * D, 81)
    q = S.normal(83, 3 * nh * D).reshape(3, nh * D)
    ws = dev.alloc(dev.flash_attn_kv4_ws(3, D, nh, nkv, n_kv))
    first = attend(dev, q, kc, vc, D, nh, nkv, 0.1, n_kv)
    for i in range(5):
        got = attend(dev, q, kc, vc, D, nh, nkv, 0.1, n_kv, ws=ws if i & 1 else None)
        assert (got.view(np.uint32) == first.view(np.uint32)).all()


def test_no_cells(dev):
    kc, vc = dev.kv(64, 32, H.KV_Q4_0), dev.kv(64, 32, H.KV_Q4_0)
    q = S.normal(1, 3 * 64).reshape(3, 64)
    assert (attend(dev, q, kc, vc, 64, 1, 1, 1.0, 0) == 0).all()


def test_refusals(dev):
    L, ctx = dev.L, dev.ctx
    kc, vc, k1 = dev.kv(128, 64, H.KV_Q4_0), dev.kv(128, 64, H.KV_Q4_0), dev.kv(128, 64, H.KV_Q4_1)
    k8, small, wide = dev.kv(128, 64), dev.kv(128, 32, H.KV_Q4_0), dev.kv(192, 64, H.KV_Q4_0)
    b = dev.alloc(1 << 16)
    ok = dict(ctx=ctx, q=b.ptr, T=2, qs=256, kc=kc.h, vc=vc.h, D=64, nh=4, nkv=2, scale=0.125, n_kv=64, runs=None, mask=None,
              ms=0, out=b.ptr + 8192, os=256, ws=None, wb=0, stream=None)

    def call(**kw):
        return L.tsr_hip_flash_attn_kv4(*{**ok, **kw}.values())

    assert call() == 0
    dev.sync()
    for kw in (dict(ctx=None), dict(q=None), dict(kc=None), dict(vc=None), dict(out=None), dict(T=0), dict(T=65536),
               dict(q=b.ptr + 4), dict(out=b.ptr + 8196), dict(qs=252), dict(qs=258), dict(os=252), dict(os=258),
               dict(runs=b.ptr + 4), dict(mask=b.ptr + 1, ms=64), dict(mask=b.ptr, ms=63), dict(ws=b.ptr + 4, wb=1 << 15)):
        assert call(**kw) == -1, kw
    for kw in (dict(D=32, nh=8, nkv=4), dict(D=96), dict(nkv=0), dict(nh=0), dict(nh=3), dict(nh=132, nkv=2),
               dict(D=512, nh=128, nkv=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
               dict(scale=1e-40), dict(kc=wide.h), dict(vc=wide.h), dict(vc=small.h)):
        assert call(**kw) == -2, kw
    for kw in (dict(kc=k8.h), dict(vc=k8.h), dict(kc=k8.h, vc=k8.h), dict(kc=k1.h), dict(vc=k1.h)):
        assert call(**kw) == -7, kw
    assert call(n_kv=65) == -5
    big = dev.kv(128, 4096, H.KV_Q4_0)
    n_ws = dev.flash_attn_kv4_ws(2, 64, 4, 2, 4096)
    assert n_ws > 4096
    assert call(kc=big.h, vc=big.h, n_kv=4096, ws=b.ptr, wb=n_ws - 1) == -1
    assert dev.flash_attn_kv4_ws(0, 64, 4, 2, 4096) == 0 and dev.flash_attn_kv4_ws(2, 65, 4, 2, 4096) == 0


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv,kind", [(8, 4, 128, 64, 1000, "causal"), (8, 4, 128, 64, 1000, "mask"),
                                                  (8, 4, 256, 64, 1000, "mask"), (32, 8, 128, 1, 1000, "mask"),
                                                  (32, 8, 128, 16, 20000, "batch"), (4, 1, 64, 1, 30000, "causal")])
def test_precision(dev, typ, nh, nkv, D, T, n_kv, kind):
    """The error of whole rows, where roundings of either sign add as squares and not as bounds do. On normal values a score
    of spread 1 (the sum of D products by 1 / sqrt(D)) is off by the pieces of q (2^-23 of it), the rounding of each block's
    and the running sum (D / 32 of 2^-24 on some four times the score's spread, for the zero point) and of the change of
    base (2^-24 of at most 6): below 2^-21 altogether; a weight by that, exp2 (2^-24) and its pieces (2^-22), so that a
    row, a sum of weights times values of either sign, is off by less than 2^-21 of its length on average, and 2^-19 leaves
    four times that for the worst of a few hundred rows. (One value of one cell that is rounded to 11 bits shows as 2^-16.)"""
    E, scale = nkv * D, 1.0 / math.sqrt(D)
    ki, kc, vi, vc = caches(dev, typ, n_kv, E, 1, v_scale=0.5)
    q = S.normal(9, T * nh * D).reshape(T, nh * D)
    rng = np.random.default_rng(3)
    runs = mask = None
    if kind == "mask":
        mask = np.zeros((T, n_kv), np.float16)
        mask[rng.random((T, n_kv)) < 0.2] = -np.inf
        mask[:, 0] = 0
    elif kind == "batch":
        runs = np.zeros((T, 4), np.uint32)
        runs[:, 1] = np.cumsum(rng.integers(n_kv // T // 8, n_kv // T, T))
        runs[1:, 0] = runs[:-1, 1]
    else:
        runs = causal(T, n_kv - T)
    want, _ = R.attention(q, ki, vi, typ, D, nh, nkv, scale, runs, mask)
    got = attend(dev, q, kc, vc, D, nh, nkv, scale, n_kv, runs, mask).astype(np.float64)
    rel = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert rel.max() <= 2.0 ** -19, (rel.max(), np.unravel_index(rel.argmax(), rel.shape))


def test_many_rows(dev):
    """More tokens than one launch holds."""
    D, T, n_kv, typ = 64, 16500, 70, H.KV_Q4_0
    ki, kc, vi, vc = caches(dev, typ, n_kv, D, 91)
    q = S.normal(93, T * D).reshape(T, D)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = 1 + np.arange(T) % n_kv
    got = attend(dev, q, kc, vc, D, 1, 1, 0.125, n_kv, runs)
    pick = np.r_[0:40, 15980:16020, T - 40:T]
    want, tol = R.attention(q[pick], ki, vi, typ, D, 1, 1, 0.125, runs[pick])
    R.check(got[pick], want, tol, "many rows")


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", [(32, 8, 64, 600, 75), (32, 8, 128, 520, 200), (8, 4, 256, 150, 131),
                                              (4, 2, 512, 20, 97), (12, 2, 512, 2, 300), (16, 1, 256, 1, 900)])
def test_masks_at_every_head_size(dev, typ, nh, nkv, D, T, n_kv):
    """Masks that hide and weigh cells, their rows aligned to eight bytes and not, a row that sees nothing."""
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 101)
    rng = np.random.default_rng(D + T)
    q = S.normal(103, T * nh * D).reshape(T, nh * D)
    for width in (n_kv + 1, (n_kv + 7) // 4 * 4):
        mask = rng.standard_normal((T, width)).astype(np.float16)
        mask[rng.random((T, width)) < 0.5] = -np.inf
        mask[T - 1] = -np.inf
        mask[:, n_kv:] = np.nan
        want, tol = R.attention(q, ki, vi, typ, D, nh, nkv, 0.15, None, mask)
        got = attend(dev, q, kc, vc, D, nh, nkv, 0.15, n_kv, mask=mask)
        R.check(got, want, tol, f"rows of {width}")
        assert (got[T - 1] == 0).all()


def test_two_streams(dev):
    """Calls on two streams at once: each with a workspace of its own, and both with the context's scratch; rows stored,
    read back and attended to on a stream that is not the context's."""
    other = H.Device(0)
    nh, nkv, D, n_kv, typ = 32, 8, 128, 6000, H.KV_Q4_1
    ki, kc, vi, vc = caches(dev, typ, n_kv, nkv * D, 111)
    qs = S.normal(113, 2 * nh * D).reshape(2, nh * D)
    bq = [dev.upload(qs[i]) for i in range(2)]
    streams = (None, other.stream)
    need = dev.flash_attn_kv4_ws(1, D, nh, nkv, n_kv)
    assert need > 0
    wants = [R.attention(qs[i:i + 1], ki, vi, typ, D, nh, nkv, 0.1) for i in range(2)]
    for ws in ([dev.alloc(need), dev.alloc(need)], [None, None]):
        outs = [[dev.alloc(4 * nh * D).fill(0xFF) for _ in range(6)] for _ in range(2)]
        dev.sync()
        for j in range(6):
            for i in range(2):
                dev.flash_attn_kv4(bq[i], 1, nh * D, kc, vc, D, nh, nkv, 0.1, n_kv, outs[i][j], nh * D, ws=ws[i],
                                   stream=streams[i])
        for st in streams:
            dev.sync(st)
        for i in range(2):
            for out in outs[i]:
                R.check(out.read(np.float32, (1, nh, D)), *wants[i], f"stream {i}")
    x = S.normal(117, 3 * nkv * D).reshape(3, nkv * D)
    cells = np.array([5, 17, 4000], np.int64)
    bx, bi, back = dev.upload(x), dev.upload(cells), dev.alloc(x.nbytes).fill(0xFF)
    out = dev.alloc(4 * nh * D)
    dev.sync()
    dev.kv_set_rows(vc, 1, bx, 3, nkv * D, bi, stream=streams[1])
    dev.kv_get_rows(vc, 1, bi, 3, back, nkv * D, stream=streams[1])
    dev.flash_attn_kv4(bq[0], 1, nh * D, kc, vc, D, nh, nkv, 0.1, n_kv, out, nh * D, stream=streams[1])
    dev.sync(streams[1])
    vi[cells] = R.quantize(x, typ)
    assert (back.read(np.float32, x.shape) == R.values_f32(vi[cells], typ)).all()
    R.check(out.read(np.float32, (1, nh, D)), *R.attention(qs[:1], ki, vi, typ, D, nh, nkv, 0.1), "behind the rows")
    # (the scratch goes back to the context's stream before the other one ends)
    R.check(attend(dev, qs[:1], kc, vc, D, nh, nkv, 0.1, n_kv), *R.attention(qs[:1], ki, vi, typ, D, nh, nkv, 0.1), "after it")
    other.close()


def test_offsets_past_32_bits(dev):
    """A plane of more than 4 GiB: its last cells and heads stored, read back and attended to."""
    nh = nkv = 64
    D, kv_size, n, typ = 128, 1 << 20, 45, H.KV_Q4_0
    E = nkv * D
    assert kv_size * (E // 32) * R.BLOCK[typ] > 1 << 32
    cells = kv_size - n + np.arange(n, dtype=np.int64)
    bi, imgs, cs = dev.upload(cells), [], []
    for which in (0, 1):
        x = S.normal(121 + which, n * E).reshape(n, E)
        imgs.append(R.quantize(x, typ))
        cs.append(dev.kv(E, kv_size, typ))
        dev.kv_set_rows(cs[which], which, dev.upload(x), n, E, bi)
        back = dev.alloc(4 * n * E)
        dev.kv_get_rows(cs[which], which, bi, n, back, E)
        dev.sync()
        assert (back.read(np.float32, (n, E)) == R.values_f32(imgs[which], typ)).all()
        assert (cs[which].get_bytes(which, int(cells[0]) * cs[which].row_bytes, imgs[which].nbytes) == imgs[which].reshape(-1)).all()
    T = 3
    q = S.normal(125, T * nh * D).reshape(T, nh * D)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 0], runs[:, 1] = cells[0], cells[0] + [1, 20, n]
    want, tol = R.attention(q, imgs[0], imgs[1], typ, D, nh, nkv, 0.1, runs - np.array([cells[0], cells[0], 0, 0], np.uint32))
    R.check(attend(dev, q, cs[0], cs[1], D, nh, nkv, 0.1, kv_size, runs), want, tol, "the last cells")
    for c in cs:
        c.free()
