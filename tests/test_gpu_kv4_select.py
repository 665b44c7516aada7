"""The blocks that tokens attend to (tsr_hip_kv4_select), against 64 bits: equal lists."""
import numpy as np
import pytest

import sparse4_ref as P

pytestmark = pytest.mark.gpu


def make(seed, T, n_head, nkv, D, nb):
    rng = np.random.default_rng(seed)
    mid = rng.standard_normal((nkv, nb, D))
    half = np.abs(rng.standard_normal((nkv, nb, D)))
    return rng.standard_normal((T, n_head, D)).astype(np.float32), P.bf16_down((mid - half).astype(np.float32)), P.bf16_up((mid + half).astype(np.float32))


def run(dev, q, lo, hi, n_head, block, n_kv, n_sel, nf, nl, runs=None, ws=None, stream=None):
    T, _, D = q.shape
    nkv = lo.shape[0]
    qb, bb = dev.upload(q), dev.upload(P.pack(lo, hi))
    rb = None if runs is None else dev.upload(np.asarray(runs, np.uint32))
    out = dev.upload(np.full((T, nkv, n_sel), -77, np.int32))
    dev.kv4_select(qb, T, n_head * D, bb, lo.shape[1], D, n_head, nkv, block, n_kv, n_sel, nf, nl, out, runs=rb, ws=ws, stream=stream)
    return out.read(np.int32, (T, nkv, n_sel))


CASES = [
    # T, n_head, n_head_kv, D, block, n_kv, spare blocks, n_sel, first, last
    (1, 32, 8, 128, 64, 8192, 0, 32, 1, 4), (1, 14, 2, 64, 32, 4001, 3, 16, 1, 2), (5, 14, 2, 64, 32, 1000, 0, 9, 0, 0),
    (33, 8, 4, 256, 64, 3000, 1, 8, 2, 2), (2, 8, 1, 512, 128, 20000, 0, 20, 0, 1), (3, 64, 1, 64, 32, 2000, 0, 5, 1, 0),
    (2, 34, 2, 64, 32, 700, 0, 4, 0, 4), (1, 1, 1, 64, 32, 1, 0, 1, 0, 0), (1, 4, 4, 64, 32, 134400, 5, 64, 1, 1),
    (7, 8, 8, 128, 1024, 50000, 0, 7, 1, 1), (1, 16, 1, 64, 32, 16400, 0, 511, 0, 0), (300, 4, 2, 64, 96, 2000, 0, 3, 1, 1),
    (2, 4, 2, 64, 32, 0, 2, 6, 1, 1), (2, 4, 2, 64, 32, 200, 0, 7, 3, 4), (2, 4, 2, 64, 32, 200, 0, 6, 3, 3),
]


@pytest.mark.parametrize("T,nh,nkv,D,block,n_kv,spare,n_sel,nf,nl", CASES)
def test_all_cells(dev, T, nh, nkv, D, block, n_kv, spare, n_sel, nf, nl):
    q, lo, hi = make(T + n_kv + D, T, nh, nkv, D, -(-n_kv // block) + spare)
    want = P.select(q, lo, hi, nh, block, n_kv, n_sel, nf, nl)
    assert (run(dev, q, lo, hi, nh, block, n_kv, n_sel, nf, nl) == want).all()


@pytest.mark.parametrize("T,nh,nkv,D,block,n_kv,n_sel,nf,nl", [
    (40, 14, 2, 64, 32, 3000, 6, 1, 2), (17, 32, 8, 128, 64, 5000, 8, 0, 1), (9, 40, 2, 64, 32, 900, 5, 2, 0)])
def test_runs(dev, T, nh, nkv, D, block, n_kv, n_sel, nf, nl):
    """Two runs a token in any order, that overlap, touch, are empty or end beyond n_kv; rows that see nothing."""
    q, lo, hi = make(T, T, nh, nkv, D, -(-n_kv // block))
    rng = np.random.default_rng(T)
    runs = np.sort(rng.integers(0, n_kv + 40, (T, 2, 2)), -1)
    runs[::5] = runs[::5, ::-1]
    runs[1, 0] = (50, 50)
    runs[2] = ((70, 20), (n_kv, n_kv + 9))                          # nothing
    runs[3] = ((100, 1500), (200, 300))                             # one inside the other
    runs[4] = ((10, 33), (33, 700))
    runs[6] = ((0, 4000000000), (5, 4294967295))
    runs[7] = ((63, 64), (64, 65))
    runs = runs.reshape(T, 4)
    want = P.select(q, lo, hi, nh, block, n_kv, n_sel, nf, nl, runs)
    assert (run(dev, q, lo, hi, nh, block, n_kv, n_sel, nf, nl, runs) == want).all()
    assert (want[2] == -1).all()


@pytest.mark.parametrize("n_kv", [3000, 140000])
def test_ties_go_to_the_lowest(dev, n_kv):
    q, lo, hi = make(4, 3, 4, 2, 64, -(-n_kv // 32))
    q[0] = 0.0                                                      # every score 0
    lo[:, 20:] = lo[:, 7:8]                                         # all but 20 blocks alike
    hi[:, 20:] = hi[:, 7:8]
    lo[:, ::3], hi[:, ::3] = lo[:, 1:2], hi[:, 1:2]
    want = P.select(q, lo, hi, 4, 32, n_kv, 30, 0, 2)
    assert (run(dev, q, lo, hi, 4, 32, n_kv, 30, 0, 2) == want).all()


def test_close_scores(dev):
    """Scores that differ by less than f32 tells apart, and by 17 orders of magnitude."""
    nb = 300
    q = np.ones((2, 1, 64), np.float32)
    q[0, 0, 1] = 2.0 ** -20
    lo = np.zeros((1, nb, 64))
    hi = np.zeros((1, nb, 64))
    perm = np.random.default_rng(0).permutation(nb)
    hi[0, :, 0] = 128.0
    hi[0, :, 1] = P.bf16_up(2.0 ** -13 * (1 + (perm // 3) / 128.0).astype(np.float32))
    hi[0, 5:9, 0] = 2.0 ** 57
    for n_sel in (4, 11, 100, 299):
        want = P.select(q, lo, hi, 1, 32, nb * 32, n_sel, 0, 0)
        assert (run(dev, q, lo, hi, 1, 32, nb * 32, n_sel, 0, 0) == want).all()


def test_queries_that_are_not_finite(dev):
    """A NaN score is the lowest, for its KV head alone; infinities have their order."""
    q, lo, hi = make(1, 3, 8, 2, 64, 50)
    q[0, 1, 5] = np.nan
    q[1, 6, 7] = np.inf
    hi[1, 10, 7] = 0.0                                              # inf 0
    lo[1, 10, 7] = -1.0
    want = P.select(q, lo, hi, 8, 32, 1600, 6, 1, 1)
    got = run(dev, q, lo, hi, 8, 32, 1600, 6, 1, 1)
    assert (got[[0, 0, 1, 2, 2], [0, 1, 0, 0, 1]] == want[[0, 0, 1, 2, 2], [0, 1, 0, 0, 1]]).all()
    assert want[0, 0].tolist() == [0, 1, 2, 3, 4, 49]
    assert 10 not in got[1, 1].tolist()


def test_workspace_in_a_graph(dev):
    """A captured call brings its workspace and reads queries, bounds and runs when it is replayed; without one it is refused."""
    T, nh, nkv, D, n_kv = 2, 4, 2, 64, 2000
    q, lo, hi = make(11, T, nh, nkv, D, -(-n_kv // 32))
    need = dev.kv4_select_ws(T, nkv, 32, n_kv)
    ws, qb, bb = dev.alloc(need), dev.upload(q), dev.upload(P.pack(lo, hi))
    rb, out = dev.upload(np.zeros((T, 4), np.uint32)), dev.alloc(4 * T * nkv * 8)
    args = (qb, T, nh * D, bb, lo.shape[1], D, nh, nkv, 32, n_kv, 8, 1, 1, out)
    dev.graph_begin()
    with pytest.raises(Exception):
        dev.kv4_select(*args, runs=rb)
    dev.kv4_select(*args, runs=rb, ws=ws)
    g = dev.graph_end()
    for k, end in enumerate((2000, 31, 1000, 300, 0)):
        q = make(20 + k, T, nh, nkv, D, 1)[0]
        runs = np.array([[0, end, 0, 0], [end // 2, end, 0, 5]], np.uint32)
        qb.write(q)
        rb.write(runs)
        ws.fill(0xFF)
        g.launch()
        want = P.select(q, lo, hi, nh, 32, n_kv, 8, 1, 1, runs)
        assert (out.read(np.int32, want.shape) == want).all(), end
    g.free()


def test_long_calls_go_out_in_parts(dev):
    """More tokens than the workspace's 64 MiB hold keys for."""
    T, n_kv = 2100, 131072
    q, lo, hi = make(5, T, 1, 1, 64, 4096)
    assert dev.kv4_select_ws(T, 1, 32, n_kv) == 64 << 20
    got = run(dev, q, lo, hi, 1, 32, n_kv, 5, 1, 1)
    for t in (0, 1, 2047, 2048, 2099):
        assert (got[t:t + 1] == P.select(q[t:t + 1], lo, hi, 1, 32, n_kv, 5, 1, 1)).all(), t
