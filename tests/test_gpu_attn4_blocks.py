"""Attention over listed blocks of a 4-bit KV cache (tsr_hip_flash_attn_kv4_blocks) against 64 bits."""
import math

import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P

pytestmark = pytest.mark.gpu


def caches(dev, seed, n, E, typ, size=None):
    k, v = P.cache_rows(seed, n, E), (0.5 * P.cache_rows(seed + 1, n, E)).astype(np.float32)
    ki, vi = R.quantize(k, typ), R.quantize(v, typ)
    kc, vc = dev.kv(E, size or n, typ), dev.kv(E, size or n, typ)
    kc.set_bytes(0, ki)
    vc.set_bytes(1, vi)
    return kc, vc, ki, vi


def lists(rng, T, nkv, n_sel, nb):
    """Ascending block lists, some shorter than n_sel."""
    out = np.full((T, nkv, n_sel), -1, np.int32)
    for t in range(T):
        for h in range(nkv):
            n = min(nb, n_sel if rng.random() < 0.7 else int(rng.integers(0, n_sel + 1)))
            out[t, h, :n] = np.sort(rng.permutation(nb)[:n])
    return out


def run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block, runs=None, ws=None, out=None):
    T = q.shape[0]
    ob = dev.upload(np.full((T, nh * D), 9.0, np.float32))
    dev.flash_attn_kv4_blocks(dev.upload(q), T, nh * D, kc, vc, D, nh, nkv, 1 / math.sqrt(D), n_kv, dev.upload(blocks), blocks.shape[2],
                              block, ob, nh * D, runs=None if runs is None else dev.upload(np.asarray(runs, np.uint32)), ws=ws)
    return ob.read(np.float32, (T, nh, D))


SHAPES = [
    # n_head, n_head_kv, D, T, n_kv, block, n_sel
    (14, 2, 64, 1, 900, 32, 16), (32, 8, 128, 1, 3000, 64, 32), (32, 8, 128, 3, 1000, 32, 9), (8, 8, 128, 2, 500, 32, 3),
    (16, 1, 128, 2, 700, 64, 5), (12, 2, 128, 2, 700, 96, 5), (40, 2, 64, 2, 600, 32, 30), (8, 4, 256, 5, 900, 64, 7),
    (16, 2, 256, 2, 600, 32, 25), (20, 1, 256, 1, 300, 32, 9), (2, 2, 512, 3, 400, 128, 2), (8, 1, 512, 1, 2000, 32, 60),
    (9, 1, 512, 2, 300, 32, 4), (64, 1, 64, 2, 300, 32, 5), (4, 4, 64, 40, 257, 32, 4), (1, 1, 64, 1, 1, 32, 1),
]


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv,block,n_sel", SHAPES)
def test_shapes(dev, typ, nh, nkv, D, T, n_kv, block, n_sel):
    rng = np.random.default_rng(nh * D + T)
    kc, vc, ki, vi = caches(dev, nh + D, n_kv, nkv * D, typ)
    q = rng.standard_normal((T, nh * D)).astype(np.float32)
    blocks = lists(rng, T, nkv, n_sel, -(-n_kv // block))
    want, tol = P.attention(q, ki, vi, typ, D, nh, nkv, 1 / math.sqrt(D), blocks, block, n_kv)
    R.check(run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block), want, tol)
    runs = np.sort(rng.integers(0, n_kv + 30, (T, 2, 2)), -1).reshape(T, 4)
    want, tol = P.attention(q, ki, vi, typ, D, nh, nkv, 1 / math.sqrt(D), blocks, block, n_kv, runs)
    R.check(run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block, runs), want, tol, "runs")


def test_all_blocks_are_dense_attention(dev):
    """Every block listed, and many more tiles than a wave takes at a time: dense attention within both errors."""
    nh, nkv, D, T, n_kv, block = 4, 1, 64, 300, 9000, 32
    kc, vc, ki, vi = caches(dev, 3, n_kv, D, R.Q4_0)
    q = np.random.default_rng(0).standard_normal((T, nh * D)).astype(np.float32)
    runs = np.zeros((T, 4), np.uint32)
    runs[:, 1] = np.linspace(0, n_kv, T).astype(np.uint32)
    nb = -(-n_kv // block)
    blocks = np.broadcast_to(np.arange(nb, dtype=np.int32), (T, 1, nb)).copy()
    got = run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block, runs)
    out = dev.alloc(4 * T * nh * D)
    dev.flash_attn_kv4(dev.upload(q), T, nh * D, kc, vc, D, nh, nkv, 1 / math.sqrt(D), n_kv, out, nh * D, runs=dev.upload(runs))
    dense = out.read(np.float32, (T, nh, D))
    some = [1, 7, 100, 299]
    want, tol = R.attention(q[some], ki, vi, R.Q4_0, D, nh, nkv, 1 / math.sqrt(D), runs[some])
    R.check(got[some], want, tol)
    assert (got[0] == 0).all() and (dense[0] == 0).all()
    size = np.abs(dense).max(-1, keepdims=True)
    assert (np.abs(got - dense) <= 2e-5 * size).all()               # (two kernels, each some 1e-6 of the row's largest)


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
def test_entries_that_are_passed_over(dev, typ):
    """Blocks behind the cells in use, negative ones and such as no int32 block can be: nothing is read of them, and a list of
    nothing else is an empty row."""
    nh, nkv, D, T, n_kv, size, block = 4, 2, 64, 4, 100, 500, 32
    kc, vc, ki, vi = caches(dev, 1, size, nkv * D, typ)
    bad = R.quantize(np.full((size - n_kv, nkv * D), np.inf, np.float32), typ)
    kc.set_bytes(0, bad, off=n_kv * kc.row_bytes)
    vc.set_bytes(1, bad, off=n_kv * kc.row_bytes)
    q = np.random.default_rng(4).standard_normal((T, nh * D)).astype(np.float32)
    blocks = np.array([[[3, 0, -1], [2, 5, 1]], [[-1, -2, 4], [2 ** 31 - 1, -2 ** 31, 15]], [[1, 3, 2], [0, 15, 16]],
                       [[67108863, 67108864, 1], [3, 1, 0]]], np.int32)
    fine = np.where((blocks < 0) | (blocks > 3), -1, blocks)
    want, tol = P.attention(q, ki, vi, typ, D, nh, nkv, 0.125, fine, block, n_kv)
    got = run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block)
    R.check(got, want, tol)
    assert (got[1] == 0).all()


def test_a_block_that_is_listed_twice_counts_twice(dev):
    nh, nkv, D, n_kv, block = 2, 1, 64, 200, 32
    kc, vc, ki, vi = caches(dev, 6, n_kv, D, R.Q4_0)
    q = np.random.default_rng(5).standard_normal((1, nh * D)).astype(np.float32)
    blocks = np.array([[[1, 4, 1]]], np.int32)
    got = run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block)
    K, V = R.values(ki, R.Q4_0), R.values(vi, R.Q4_0)
    cells = np.concatenate([np.arange(32, 64), np.arange(128, 160), np.arange(32, 64)])
    s = q.reshape(nh, D).astype(np.float64) @ K[cells].T * 0.125
    p = np.exp(s - s.max(1, keepdims=True))
    want = (p / p.sum(1, keepdims=True)) @ V[cells]
    _, tol = P.attention(q, ki, vi, R.Q4_0, D, nh, nkv, 0.125, np.array([[[1, 4]]]), block, n_kv)
    R.check(got[0], want, 2 * tol[0])                               # (weights up to twice as large)


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
def test_cells_that_are_not_seen_reach_nothing(dev, typ):
    """Infinities and NaNs in blocks that are not listed, and in listed blocks behind a row's runs."""
    nh, nkv, D, n_kv, block = 8, 2, 128, 320, 64
    k, v = P.cache_rows(1, n_kv, nkv * D), P.cache_rows(2, n_kv, nkv * D)
    k[64:128], v[64:128], k[300:], v[300:] = np.inf, np.nan, np.nan, np.inf
    k[200, 5], v[210, 9] = np.inf, -np.inf
    ki, vi = R.quantize(k, typ), R.quantize(v, typ)
    kc, vc = dev.kv(nkv * D, n_kv, typ), dev.kv(nkv * D, n_kv, typ)
    kc.set_bytes(0, ki)
    vc.set_bytes(1, vi)
    q = np.random.default_rng(7).standard_normal((2, nh * D)).astype(np.float32)
    blocks = np.array([[[0, 2, 4], [0, 4, -1]], [[0, 2, 3], [0, 3, 4]]], np.int32)
    runs = np.array([[0, 64, 128, 300], [0, 20, 240, 300]], np.uint32)
    want, tol = P.attention(q, ki, vi, typ, D, nh, nkv, 1 / math.sqrt(D), blocks, block, n_kv, runs)
    assert np.isfinite(want).all()
    R.check(run(dev, q, kc, vc, D, nh, nkv, n_kv, blocks, block, runs), want, tol)


def test_strides_and_what_lies_behind_the_rows(dev):
    nh, nkv, D, T, n_kv, block = 4, 2, 64, 5, 300, 32
    kc, vc, ki, vi = caches(dev, 8, n_kv, nkv * D, R.Q4_1)
    rng = np.random.default_rng(3)
    qs, os_ = nh * D + 20, nh * D + 8
    q = rng.standard_normal((T, qs)).astype(np.float32)
    blocks = lists(rng, T, nkv, 5, 10)
    out = dev.upload(np.full((T + 1, os_), 3.5, np.float32))
    dev.flash_attn_kv4_blocks(dev.upload(q), T, qs, kc, vc, D, nh, nkv, 0.125, n_kv, dev.upload(blocks), 5, block, out, os_)
    got = out.read(np.float32, (T + 1, os_))
    want, tol = P.attention(q[:, :nh * D], ki, vi, R.Q4_1, D, nh, nkv, 0.125, blocks, block, n_kv)
    R.check(got[:T, :nh * D], want, tol)
    assert (got[:T, nh * D:] == 3.5).all() and (got[T] == 3.5).all()


def test_selected_and_attended_in_a_graph(dev):
    """A decode token's calls as they are used: the new cell's bounds, the selection and the attention, captured once with one
    workspace and replayed while the context grows."""
    nh, nkv, D, size, block, n_sel = 8, 2, 128, 2500, 32, 21
    E = nkv * D
    k, v = P.cache_rows(21, size, E), P.cache_rows(22, size, E)
    kc, vc = dev.kv(E, size, R.Q4_0), dev.kv(E, size, R.Q4_0)
    ki, vi = R.quantize(k, R.Q4_0), R.quantize(v, R.Q4_0)
    nb = -(-size // block)
    bounds = dev.alloc(4 * E * nb)
    have = 2000
    kc.set_bytes(0, ki[:have])
    vc.set_bytes(1, vi[:have])
    dev.kv4_bounds(kc, D, block, have, bounds)
    need = max(dev.kv4_select_ws(1, nkv, block, size), dev.flash_attn_kv4_blocks_ws(1, D, nh, nkv, n_sel, block))
    ws, qb, out = dev.alloc(need), dev.alloc(4 * nh * D), dev.alloc(4 * nh * D)
    ids, row, vrow = dev.alloc(4 * nkv * n_sel), dev.alloc(4 * E), dev.alloc(4 * E)
    ins = dev.alloc(32)                                            # runs, then the cell (int64), then {cell, cell + 1}
    with pytest.raises(Exception):
        dev.graph_begin()
        try:
            dev.flash_attn_kv4_blocks(qb, 1, nh * D, kc, vc, D, nh, nkv, 0.1, size, ids, n_sel, block, out, nh * D, runs=ins)
        finally:
            dev.graph_end().free()
    dev.graph_begin()
    dev.kv_set_rows(kc, 0, row, 1, E, ins.ptr + 16)
    dev.kv_set_rows(vc, 1, vrow, 1, E, ins.ptr + 16)
    dev.kv4_bounds(kc, D, block, size, bounds, cells=ins.ptr + 24, n_new=1)
    dev.kv4_select(qb, 1, nh * D, bounds, nb, D, nh, nkv, block, size, n_sel, 1, 2, ids, runs=ins, ws=ws)
    dev.flash_attn_kv4_blocks(qb, 1, nh * D, kc, vc, D, nh, nkv, 0.1, size, ids, n_sel, block, out, nh * D, runs=ins, ws=ws)
    g = dev.graph_end()
    values = R.values_f32(ki, R.Q4_0)
    rng = np.random.default_rng(1)
    for cell in range(have, have + 70, 1):
        q = rng.standard_normal((1, nh * D)).astype(np.float32)
        qb.write(q)
        row.write(k[cell])
        vrow.write(v[cell])
        w = np.zeros(8, np.uint32)
        w[1] = cell + 1
        w[4] = cell
        w[6], w[7] = cell, cell + 1
        ins.write(w)
        g.launch()
        if cell % 23 and cell not in (have, have + 15, have + 16):
            continue
        got_ids, got = ids.read(np.int32, (1, nkv, n_sel)), out.read(np.float32, (1, nh, D))
        lo, hi = P.bounds(values[:cell + 1], D, block)
        want_ids = P.select(q.reshape(1, nh, D), lo, hi, nh, block, cell + 1, n_sel, 1, 2)
        assert (got_ids == want_ids).all(), cell
        want, tol = P.attention(q, ki, vi, R.Q4_0, D, nh, nkv, 0.1, want_ids, block, cell + 1)
        R.check(got, want, tol, f"cell {cell}")
    g.free()
