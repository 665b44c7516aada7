"""GPU KV caches of 4-bit blocks (q4_0, q4_1): the ggml image round trip, rows stored bit for bit as ggml's rule gives them,
cells read back, ROPE + SET_ROWS_KV, refusals."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R
import tsr_hip as H
import tsr_synth as S
from helpers import assert_bits_equal

pytestmark = pytest.mark.gpu
TYPES = [H.KV_Q4_0, H.KV_Q4_1]


def hard_rows(n, E, seed):
    """Rows with the blocks where the rule can go wrong: zeros, one value, ties of +-max, constants, tiny, huge, NaN."""
    x = S.normal(seed, n * E).reshape(n, E).copy()
    b = x.reshape(-1, 32)
    k = len(b)
    b[0 % k] = 0.0
    b[1 % k, :] = 0.0
    b[1 % k, 7] = -3.0
    b[2 % k, 5], b[2 % k, 20] = -9.0, 9.0            # the first of two equal magnitudes gives the sign
    b[3 % k, 5], b[3 % k, 20] = 9.0, -9.0
    b[4 % k] = 2.5
    b[5 % k] *= np.float32(1e-41)
    b[6 % k] *= np.float32(1e5)
    b[7 % k, 3] = np.nan
    b[8 % k] = np.nan
    b[9 % k] = np.linspace(-8, 7.5, 32)              # quotients on the borders between codes
    b[10 % k] = -0.0
    b[11 % k] *= np.float32(1e-7)
    return x


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("E,kv_size", [(1024, 256), (192, 100), (64, 33), (64, 1)])
def test_image_round_trip(dev, typ, E, kv_size):
    rng = np.random.default_rng(E + kv_size)
    for which in (0, 1):
        kv = dev.kv(E, kv_size, typ)
        assert (kv.get_bytes(which) == 0).all()
        img = rng.integers(0, 256, kv_size * kv.row_bytes, dtype=np.uint8)
        kv.set_bytes(which, img)
        assert (kv.get_bytes(which) == img).all()
        off, n = 13 % img.size, min(700, img.size - 13)          # ranges that cut blocks and scales
        patch = rng.integers(0, 256, n, dtype=np.uint8)
        kv.set_bytes(which, patch, off)
        img[off:off + n] = patch
        assert (kv.get_bytes(which) == img).all()
        assert (kv.get_bytes(which, 5, 11) == img[5:16]).all()
        with pytest.raises(H.TsrHipError) as e:
            kv.set_bytes(which, patch, img.size - 1)
        assert e.value.code == -5
        kv.free()


@pytest.mark.parametrize("typ", [H.KV_Q8_0, H.KV_Q4_0, H.KV_Q4_1])
def test_image_in_pieces(dev, typ):
    """An image of more bytes than one piece of the conversion (64 MiB), from the middle of a row to the middle of one."""
    E, kv_size = 1024, 150_000
    kv = dev.kv(E, kv_size, typ)
    img = np.random.default_rng(typ).integers(0, 256, kv_size * kv.row_bytes, dtype=np.uint8)
    off, end = 5 * kv.row_bytes + 77, img.size - 300
    assert end - off > 80 << 20
    kv.set_bytes(H.KV_K, img[off:end], off)
    assert (kv.get_bytes(H.KV_K, off, end - off) == img[off:end]).all()
    img[:off], img[end:] = 0, 0
    assert (kv.get_bytes(H.KV_K) == img).all()
    kv.free()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("E,kv_size,n,stride", [(1024, 64, 1, 1024), (128, 300, 33, 132), (64, 40, 40, 64),
                                                (320, 1000, 257, 1600)])
def test_set_rows_bits_and_read_back(dev, typ, which, E, kv_size, n, stride):
    kv = dev.kv(E, kv_size, typ)
    rng = np.random.default_rng(n)
    before = R.quantize(S.normal(5, kv_size * E).reshape(kv_size, E), typ)
    kv.set_bytes(which, before)
    src = np.zeros((n, stride), np.float32)
    src[:, :E] = hard_rows(n, E, 7)
    idx = rng.permutation(kv_size)[:n].astype(np.int64)
    want = before.copy()
    want[idx] = R.quantize(src[:, :E], typ)
    bad = dev.upload(np.zeros(1, np.int32))
    dev.kv_set_rows(kv, which, dev.upload(src), n, stride, dev.upload(idx), bad)
    assert (kv.get_bytes(which).reshape(kv_size, -1) == want).all()
    # read back, the same cells more than once, into rows wider than E
    ids = np.concatenate([idx, idx[:1], rng.integers(0, kv_size, 50)]).astype(np.int64)
    dst = dev.alloc(4 * ids.size * (E + 8)).fill(0xFF)
    dev.kv_get_rows(kv, which, dev.upload(ids), ids.size, dst, E + 8, bad)
    dev.sync()
    got = dst.read(np.float32, (ids.size, E + 8))
    v = R.values_f32(want, typ)[ids]
    assert_bits_equal(np.where(np.isnan(got[:, :E]), 0, got[:, :E]), np.where(np.isnan(v), 0, v), "read back")
    assert (np.isnan(got[:, :E]) == np.isnan(v)).all()
    assert (got[:, E:].view(np.uint32) == 0xFFFFFFFF).all()
    assert bad.read(np.int32, (1,))[0] == 0


@pytest.mark.parametrize("typ", TYPES)
def test_infinite_values_stay_in_their_block(dev, typ):
    E = 64
    kv = dev.kv(E, 4, typ)
    x = S.normal(3, 2 * E).reshape(2, E).copy()
    x[0, 3] = np.inf
    x[1, 40] = -np.inf
    dst = dev.alloc(8 * E)
    idx = dev.upload(np.array([2, 1], np.int64))
    dev.kv_set_rows(kv, 0, dev.upload(x), 2, E, idx)
    dev.kv_get_rows(kv, 0, idx, 2, dst, E)
    dev.sync()
    got = dst.read(np.float32, (2, E))
    want = R.values_f32(R.quantize(x, typ), typ)
    assert not np.isfinite(got[0, 3]) and not np.isfinite(got[1, 40])
    for r, s in ((0, slice(32, 64)), (1, slice(0, 32))):
        assert_bits_equal(got[r, s], want[r, s], "the other block")


@pytest.mark.parametrize("typ", [H.KV_Q8_0] + TYPES)
def test_out_of_range_cells(dev, typ):
    E, kv_size = 64, 16
    kv = dev.kv(E, kv_size, typ)
    bad = dev.upload(np.zeros(1, np.int32))
    x = dev.upload(np.ones((4, E), np.float32))
    idx = dev.upload(np.array([3, 16, -1, 1 << 40], np.int64))
    dev.kv_set_rows(kv, 0, x, 4, E, idx, bad)
    dev.sync()
    assert bad.read(np.int32, (1,))[0] == 1
    img = kv.get_bytes(0).reshape(kv_size, -1)
    assert (img[[r for r in range(kv_size) if r != 3]] == 0).all() and (img[3] != 0).any()
    bad.fill(0)
    dst = dev.alloc(4 * 4 * E).fill(0xFF)
    dev.kv_get_rows(kv, 0, idx, 4, dst, E, bad)
    dev.sync()
    assert bad.read(np.int32, (1,))[0] == 1
    got = dst.read(np.float32, (4, E))
    # q8_0: f16(1/127) 127, off by the half step of f16 at most; q4_0: -1/8 (0 - 8) and q4_1: 0 n + 1, exact
    assert (np.abs(got[0] - 1.0) <= (2.0 ** -11 if typ == H.KV_Q8_0 else 0.0)).all() and (got[1:].view(np.uint32) == 0xFFFFFFFF).all()
    # without a word of its own the call raises the context's
    dev.get_flags()
    dev.kv_get_rows(kv, 0, idx, 4, dst, E)
    assert dev.get_flags() & 1


@pytest.mark.parametrize("which", [0, 1])
def test_q8_0_cells_read_back(dev, which):
    E, kv_size = 192, 50
    kv = dev.kv(E, kv_size)
    rng = np.random.default_rng(1)
    img = rng.integers(0, 256, (kv_size, E // 32, 34), dtype=np.uint8)
    img[..., 1] &= 0x3B                               # finite scales
    kv.set_bytes(which, img)
    d = np.ascontiguousarray(img[..., :2]).view(np.float16).astype(np.float32)
    want = (d * img[..., 2:].view(np.int8)).reshape(kv_size, E)
    ids = rng.permutation(kv_size).astype(np.int64)
    dst = dev.alloc(4 * kv_size * E)
    dev.kv_get_rows(kv, which, dev.upload(ids), kv_size, dst, E)
    dev.sync()
    assert_bits_equal(dst.read(np.float32, (kv_size, E)), want[ids], "q8_0 read back")


@pytest.mark.parametrize("tk,tv", [(1, 1), (2, 2), (0, 1), (2, 0)])
def test_rope_kv_is_its_three_ops(dev, tk, tv):
    T, D, nh, nkv, kv_size = 5, 64, 4, 2, 40
    E, w = nkv * D, (nh + 2 * nkv) * D
    x = S.normal(9, T * w).reshape(T, w)
    pos = dev.upload(np.arange(3, 3 + T, dtype=np.int32))
    cell = dev.upload(np.array([7, 0, 39, 12, 20], np.int64))
    a, b = dev.upload(x), dev.upload(x)
    kv = [dev.kv(E, kv_size, t) for t in (tk, tv, tk, tv)]
    dev.rope_kv(a, T, w, D, nh, nkv, D, H.ROPE_NORMAL, pos, 10000.0, kv[0], kv[1], cell)
    dev.rope(b, T, w, D, nh + nkv, D, H.ROPE_NORMAL, pos, 10000.0, b, w)
    dev.kv_set_rows(kv[2], 0, b.ptr + 4 * nh * D, T, w, cell)
    dev.kv_set_rows(kv[3], 1, b.ptr + 4 * (nh + nkv) * D, T, w, cell)
    dev.sync()
    assert_bits_equal(a.read(np.float32, (T, w)), b.read(np.float32, (T, w)), "rotated rows")
    assert (kv[0].get_bytes(0) == kv[2].get_bytes(0)).all() and (kv[1].get_bytes(1) == kv[3].get_bytes(1)).all()
    assert (kv[0].get_bytes(0) != 0).any() and (kv[1].get_bytes(1) != 0).any()


def test_refusals(dev):
    L, ctx = dev.L, dev.ctx
    h = C.c_void_p()
    assert L.tsr_hip_kv_create_type(ctx, 3, 64, 16, C.byref(h)) == -7 and h.value is None
    for E, n in ((0, 16), (32, 16), (96, 16), (32832, 16), (64, 0), (64, 1 << 31)):
        assert L.tsr_hip_kv_create_type(ctx, 1, E, n, C.byref(h)) == -2
    kv = dev.kv(64, 16, H.KV_Q4_0)
    x, idx = dev.alloc(4096), dev.upload(np.zeros(4, np.int64))
    p, i = x.ptr, idx.ptr
    for call in (L.tsr_hip_kv_get_rows,):
        assert call(ctx, kv.h, 0, i, 0, p, 64, None, None) == 0
        for args in ((None, kv.h, 0, i, 1, p, 64), (ctx, None, 0, i, 1, p, 64), (ctx, kv.h, 2, i, 1, p, 64),
                     (ctx, kv.h, 0, None, 1, p, 64), (ctx, kv.h, 0, i, 1, None, 64), (ctx, kv.h, 0, i, 2, p + 4, 64),
                     (ctx, kv.h, 0, i, 2, p, 66), (ctx, kv.h, 0, i, 2, p, 60), (ctx, kv.h, 0, i, 65536, p, 64)):
            assert call(*args, None, None) == -1, args
    # the q8_0 attention does not take a 4-bit cache
    k8 = dev.kv(64, 16)
    msum = H.msum_build_f16(np.zeros((1, 16), np.float16))
    q, o = dev.alloc(256), dev.alloc(256)
    for kc, vc in ((kv, kv), (k8, kv), (kv, k8)):
        for fn in (dev.flash_attn, dev.flash_attn_noalloc):
            with pytest.raises(H.TsrHipError) as e:
                fn(q, 1, 64, kc, vc, 64, 1, 1, 0.125, msum, o, 64)
            assert e.value.code == -7
    plan = dev.fa_plan(64, 1, 1, 1, 16)
    plan.set(msum)
    with pytest.raises(H.TsrHipError) as e:
        dev.flash_attn_plan(plan, q, 64, kv, kv, 0.125, o, 64)
    assert e.value.code == -7
    plan.free()
