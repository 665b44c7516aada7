"""Sparse attention and eviction as one run of calls: two streams at once, two graphs in turn, planes of more than 4 GiB."""
import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P
import tsr_hip as H
import weights4_ref as W

pytestmark = pytest.mark.gpu

NH, NKV, D, BLOCK, SEL, KEEP = 8, 2, 64, 32, 8, 333


class Chain:
    """A token's calls over caches of its own: bounds, selection, attention over the list, weights, pick, both moves."""

    def __init__(self, dev, typ, n, seed):
        self.dev, self.n = dev, n
        E = NKV * D
        self.images = [R.quantize(P.cache_rows(seed + i, n, E), typ) for i in range(2)]
        self.kc, self.vc = dev.kv(E, n, typ), dev.kv(E, n, typ)
        self.nb = -(-n // BLOCK)
        self.q = dev.upload(np.random.default_rng(seed).standard_normal((1, NH * D)).astype(np.float32))
        self.bounds, self.ids = dev.alloc(4 * E * self.nb), dev.alloc(4 * NKV * SEL)
        self.out, self.acc, self.idx = dev.alloc(4 * NH * D), dev.alloc(4 * n), dev.alloc(8 * KEEP)
        self.ws = [None] * 5
        self.reset()

    def own_workspaces(self):
        d = self.dev
        sizes = [d.kv4_select_ws(1, NKV, BLOCK, self.n), d.flash_attn_kv4_blocks_ws(1, D, NH, NKV, SEL, BLOCK),
                 d.attn_weights_kv4_ws(1, D, NH, NKV, self.n), d.kv_gather_ws(self.kc, KEEP), d.kv_gather_ws(self.vc, KEEP)]
        self.ws = [d.alloc(x) if x else None for x in sizes]

    def reset(self):
        for which, kv in enumerate((self.kc, self.vc)):
            kv.set_bytes(which, self.images[which])
        for b in (self.bounds, self.ids, self.out, self.acc, self.idx):
            b.fill(0xFF)
        self.dev.sync()

    def run(self, stream=None):
        d, n, ws = self.dev, self.n, self.ws
        d.kv4_bounds(self.kc, D, BLOCK, n, self.bounds, stream=stream)
        d.kv4_select(self.q, 1, NH * D, self.bounds, self.nb, D, NH, NKV, BLOCK, n, SEL, 1, 2, self.ids, ws=ws[0], stream=stream)
        d.flash_attn_kv4_blocks(self.q, 1, NH * D, self.kc, self.vc, D, NH, NKV, 0.125, n, self.ids, SEL, BLOCK, self.out, NH * D,
                                ws=ws[1], stream=stream)
        d.attn_weights_kv4(self.q, 1, NH * D, self.kc, D, NH, NKV, 0.125, n, self.acc, ws=ws[2], stream=stream)
        d.kv_pick(self.acc, n, KEEP, 4, 50, self.idx, stream=stream)
        d.kv_gather(self.kc, self.kc, 0, self.idx, KEEP, ws=ws[3], stream=stream)
        d.kv_gather(self.vc, self.vc, 1, self.idx, KEEP, ws=ws[4], stream=stream)

    def results(self):
        return [self.bounds.read(np.uint32, (NKV, self.nb, D)), self.ids.read(np.int32, (NKV, SEL)), self.out.read(np.uint32, (NH, D)),
                self.acc.read(np.uint32, (self.n,)), self.idx.read(np.int64, (KEEP,)),
                self.kc.get_bytes(0).reshape(self.n, -1), self.vc.get_bytes(1).reshape(self.n, -1)]


def same(got, want, what):
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a == b).all(), (what, i)


def test_two_streams_and_two_graphs(dev):
    other = H.Device(0)
    chains = [Chain(dev, R.Q4_0, 3000, 1), Chain(dev, R.Q4_1, 2500, 5)]
    wants = []
    for c in chains:
        c.run()
        dev.sync()
        wants.append(c.results())
        cells = wants[-1][4]
        for which in range(2):
            assert (wants[-1][5 + which][:KEEP] == c.images[which][cells]).all()
            assert (wants[-1][5 + which][KEEP:] == c.images[which][KEEP:]).all()
    streams = (None, other.stream)
    for own in (False, True):
        for i in range(3):
            for c in chains:
                c.reset()
            for c, st in zip(chains, streams):
                if own:
                    c.own_workspaces()
                c.run(st)
            for st in streams:
                dev.sync(st)
            for c, want in zip(chains, wants):
                same(c.results(), want, f"streams, {own}, {i}")
    graphs = []
    for c in chains:
        dev.graph_begin()
        c.run()
        graphs.append(dev.graph_end())
    for i in range(4):
        for c in chains:
            c.reset()
        graphs[i % 2].launch()
        graphs[1 - i % 2].launch(other.stream)
        dev.sync()
        dev.sync(other.stream)
        for c, want in zip(chains, wants):
            same(c.results(), want, f"graphs, {i}")
        chains[i % 2].reset()                                       # eager work between the replays
        chains[i % 2].run()
        dev.sync()
        same(chains[i % 2].results(), wants[i % 2], f"eager, {i}")
    for g in graphs:
        g.free()
    dev.kv4_select(chains[0].q, 1, NH * D, chains[0].bounds, chains[0].nb, D, NH, NKV, BLOCK, 3000, SEL, 1, 2, chains[0].ids)
    dev.sync()
    other.close()


def test_planes_past_32_bits(dev):
    """The last cells and heads of planes of 4.8 GB."""
    nh = nkv = 64
    hd, size, n, block, typ = 128, 1 << 20, 45, 64, R.Q4_0
    E = nkv * hd
    kc, vc = dev.kv(E, size, typ), dev.kv(E, size, typ)
    rng = np.random.default_rng(1)
    x = [rng.standard_normal((n, E)).astype(np.float32) for _ in range(2)]
    cells = np.arange(size - n, size, dtype=np.int64)
    ib = dev.upload(cells)
    for which, kv in enumerate((kc, vc)):
        dev.kv_set_rows(kv, which, dev.upload(x[which]), n, E, ib)
    ki, vi = (R.quantize(v, typ) for v in x)
    nb = size // block
    bounds = dev.alloc(4 * E * nb)
    last = (nkv * nb - 1) * hd * 4
    H.BufferPart(bounds, last, 4 * hd).fill(0)
    new = dev.upload(np.array([size - n, size], np.uint32))
    dev.kv4_bounds(kc, hd, block, size, bounds, cells=new, n_new=n)
    got = P.words(H.BufferPart(bounds, last, 4 * hd).read(np.uint32, (1, 1, hd)))
    keys = np.concatenate([untouched(dev, kc, size - block, block - n, E), R.values_f32(ki, typ)])
    for a, b in zip(got, P.bounds(keys, hd, block)):
        assert (a[0, 0] == b[-1, 0]).all()
    q = rng.standard_normal((1, nh * hd)).astype(np.float32)
    qb, runs = dev.upload(q), dev.upload(np.array([[size - n, size, 0, 0]], np.uint32))
    ids, out, acc = dev.alloc(4 * nkv * 3), dev.alloc(4 * nh * hd), dev.alloc(4 * size)
    dev.kv4_select(qb, 1, nh * hd, bounds, nb, hd, nh, nkv, block, size, 3, 1, 1, ids, runs=runs)
    assert (ids.read(np.int32, (nkv, 3)) == [nb - 1, -1, -1]).all()
    dev.flash_attn_kv4_blocks(qb, 1, nh * hd, kc, vc, hd, nh, nkv, 0.1, size, ids, 3, block, out, nh * hd, runs=runs)
    R.check(out.read(np.float32, (1, nh, hd)), *R.attention(q, ki, vi, typ, hd, nh, nkv, 0.1))
    dev.attn_weights_kv4(qb, 1, nh * hd, kc, hd, nh, nkv, 0.1, size, acc, runs=runs)
    w = acc.read(np.float32, (size,))
    assert (w[:size - n] == 0).all()
    R.check(w[size - n:], *W.weights(q, ki, typ, hd, nh, nkv, 0.1, n))
    idx = dev.alloc(8 * n)
    dev.kv_pick(acc, size, n, 0, 1, idx)
    assert (idx.read(np.int64, (n,)) == cells).all()
    back, front = dev.alloc(4 * n * E), dev.upload(np.arange(n, dtype=np.int64))
    for which, (kv, img) in enumerate(((kc, ki), (vc, vi))):
        dev.kv_gather(kv, kv, which, idx, n)
        dev.kv_get_rows(kv, which, front, n, back, E)
        assert (back.read(np.float32, (n, E)) == R.values_f32(img, typ)).all()
    for b in (bounds, kc, vc):
        b.free()


def untouched(dev, kv, first, n, E):
    """What a cache's untouched cells hold."""
    back = dev.alloc(4 * n * E)
    dev.kv_get_rows(kv, 0, dev.upload(np.arange(first, first + n, dtype=np.int64)), n, back, E)
    return back.read(np.float32, (n, E))
