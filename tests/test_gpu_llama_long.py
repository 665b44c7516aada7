"""The Llama decoder in long contexts: scaled rotary positions over both kinds of caches, sparse attention and eviction over
4-bit ones, each call checked on what the model's buffers hold at that moment."""
import numpy as np
import pytest

import kv4_ref as R
import rope_scaled_ref as RS
import sparse4_ref as P
import tsr_hip as H
import tsr_llama as LL
import weights4_ref as W
from helpers import assert_bits_equal
from test_gpu_evict import pick_ref
from test_gpu_llama_kv4 import images

pytestmark = pytest.mark.gpu

YARN = LL.RopeScale(8.0, n_ctx_orig=64)
FACTORS = LL.RopeScale(4.0, ext_factor=0.0, freq_factors=tuple(1.0 + i / 16 for i in range(32)))


@pytest.mark.parametrize("scale", [YARN, FACTORS], ids=["yarn", "factors"])
def test_scaled_positions_over_q8_0(dev, scale):
    """The fused calls, which take the angles as a table, give the bits of rope_scaled, the stores and the attention."""
    cfg = LL.tiny_config("tiny-scaled", rope_scale=scale)
    w = LL.SyntheticWeights(cfg, cache=True)
    a, b = LL.LlamaDecoder(dev, cfg, w, 300), LL.LlamaDecoder(dev, cfg, w, 300, fused=False)
    plain = LL.LlamaDecoder(dev, LL.tiny_config("tiny-scaled"), w, 300)
    prompt = np.random.default_rng(3).integers(0, cfg.n_vocab, 90).astype(np.int32)
    for m in (a, b, plain):
        m.prefill(prompt, 0, 64)
    assert_bits_equal(a.read_logits(), b.read_logits(), "prefill")
    assert (a.read_logits() != plain.read_logits()).any()
    tok = a.read_token()
    for i in range(3):
        a.step_graph(tok, 90 + i)
        b.step(tok, 90 + i)
        assert_bits_equal(a.read_logits(), b.read_logits(), f"token {i}")
        tok = b.read_next()
    for m in (a, b, plain):
        m.check()
        m.free()


@pytest.mark.parametrize("scale,mode", [(YARN, H.ROPE_NORMAL), (FACTORS, H.ROPE_NEOX)], ids=["yarn", "factors"])
def test_scaled_positions_over_4_bit_caches(dev, monkeypatch, scale, mode):
    cfg = LL.tiny_config("tiny-scaled4", rope_scale=scale, rope_mode=mode)
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 400, kv_type=H.KV_Q4_1)
    f, mul = RS.frequencies(cfg.head_dim, cfg.rope_base, 1.0 / scale.factor, scale.ext_factor, scale.n_ctx_orig, scale.freq_factors)
    calls, real = [0], dev.rope_scaled
    w3, heads = cfg.n_q + 2 * cfg.E, cfg.n_head + cfg.n_head_kv

    def checked(x, T, x_stride, hd, n, n_dims, mode_, pos, *args, **kw):
        dev.sync()
        before, at = x.read(np.float32, (T, w3)), pos
        real(x, T, x_stride, hd, n, n_dims, mode_, pos, *args, **kw)
        dev.sync()
        got = x.read(np.float32, (T, w3))
        p = at.read(np.int32, (T,)) if isinstance(at, H.Buffer) else m.params.read(np.int32, (1,))
        want, tol = RS.rope(before[:, :heads * hd].reshape(T, heads, hd), p, hd, mode != H.ROPE_NORMAL, f, mul)
        assert (np.abs(got[:, :heads * hd].reshape(want.shape) - want) <= tol).all()
        assert (got[:, heads * hd:] == before[:, heads * hd:]).all()
        calls[0] += 1

    monkeypatch.setattr(dev, "rope_scaled", checked)
    m.prefill(np.random.default_rng(1).integers(0, cfg.n_vocab, 40).astype(np.int32), 0, 32)
    m.step(None, 40)
    assert calls[0] == 3 * cfg.n_layer
    m.check()
    m.free()


SPARSE = LL.SparseAttention(block=32, n_blocks=8, first=1, last=2)


@pytest.mark.parametrize("typ,kw,sparse", [
    (H.KV_Q4_0, {}, SPARSE), (H.KV_Q4_1, dict(n_head=8, n_head_kv=1, head_dim=128, n_embd=512, n_ff=768), SPARSE),
    (H.KV_Q4_0, {}, LL.SparseAttention(block=32, n_blocks=8, first=1, last=0)),
    (H.KV_Q4_1, {}, LL.SparseAttention(block=64, n_blocks=4, first=0, last=1))], ids=["q4_0", "q4_1-gqa8", "no-last", "one-last"])
def test_sparse_decode(dev, monkeypatch, typ, kw, sparse):
    """Every layer's list and attention of eager tokens, and graph replays with the same bits across the growth of their cells."""
    cfg = LL.tiny_config("tiny-sparse", rope_scale=YARN, **kw)
    w = LL.SyntheticWeights(cfg, cache=True)
    m, g = (LL.LlamaDecoder(dev, cfg, w, 1200, kv_type=typ, sparse=sparse) for _ in range(2))
    prompt = np.random.default_rng(2).integers(0, cfg.n_vocab, 510).astype(np.int32)
    for x in (m, g):
        x.prefill(prompt, 0, 200)
    nb, calls, real = m.n_bounds, [0], dev.flash_attn_kv4_blocks

    def checked(q, T, q_stride, kc, vc, D, nh, nkv, scale, n_kv, blocks, n_sel, block, out, out_stride, **kw):
        real(q, T, q_stride, kc, vc, D, nh, nkv, scale, n_kv, blocks, n_sel, block, out, out_stride, **kw)
        dev.sync()
        L = next(x for x in m.layers if x["kc"] is kc)
        ki, vi = images(m, L)
        lo, hi = P.words(L["bounds"].read(np.uint32, (nkv, nb, D)))
        want = tuple(P.bounds(R.values_f32(ki[:n_kv], typ), D, block))
        used = (n_kv - 1) // block if sparse.last else -(-n_kv // block)   # (the token's own block is listed without its bounds)
        for a, b in zip((lo, hi), want):
            assert (a[:, :used] == b[:, :used]).all()
        lo, hi = want
        qs = q.read(np.float32, (1, q_stride))[:, :nh * D]
        ids = blocks.read(np.int32, (1, nkv, n_sel))
        assert (ids == P.select(qs.reshape(1, nh, D), lo, hi, nh, block, n_kv, n_sel, sparse.first, sparse.last)).all()
        o, tol = P.attention(qs, ki, vi, typ, D, nh, nkv, np.float64(np.float32(scale)), ids, block, n_kv)
        R.check(out.read(np.float32, (1, nh, D)), o, tol, f"{n_kv} cells")
        calls[0] += 1

    tok = m.read_token()
    for i in range(5):
        monkeypatch.setattr(dev, "flash_attn_kv4_blocks", checked)
        m.step(tok, 510 + i)
        monkeypatch.setattr(dev, "flash_attn_kv4_blocks", real)
        g.step_graph(tok, 510 + i)
        assert_bits_equal(m.read_logits(), g.read_logits(), f"token {i}")
        tok = m.read_next()
    assert calls[0] == 5 * cfg.n_layer and g.captures == 2 and g.n_kv_graph == 1024
    for x in (m, g):
        x.check()
        x.free()


@pytest.mark.parametrize("typ,sparse", [(H.KV_Q4_0, None), (H.KV_Q4_1, SPARSE)], ids=["q4_0", "q4_1-sparse"])
def test_eviction(dev, typ, sparse):
    """Weights as the tokens of a prompt and of graph replays give them, the caches thinned out by them, and tokens behind that: their
    positions go on, they see the kept cells."""
    cfg = LL.tiny_config("tiny-evict")
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 700, kv_type=typ, sparse=sparse, track=0.75)
    D, nh, nkv = cfg.head_dim, cfg.n_head, cfg.n_head_kv
    scale = np.float64(np.float32(m.scale))
    L = m.layers[-1]
    m.prefill(np.random.default_rng(4).integers(0, cfg.n_vocab, 400).astype(np.int32), 0, 400)
    q = m._pf["qkv"].read(np.float32, (400, cfg.n_q + 2 * cfg.E))[336:, :cfg.n_q]
    runs = np.zeros((64, 4), np.int64)
    runs[:, 1] = 337 + np.arange(64)
    want, tol = W.weights(np.ascontiguousarray(q), images(m, L)[0], typ, D, nh, nkv, scale, 400, runs)
    got = L["weights"].read(np.float32, (700,))
    R.check(got[:400], want, tol, "prompt")
    assert (got[400:] == 0).all()
    pos = 400
    for i in range(3):
        m.step_graph(None, pos)
        before, got = got, L["weights"].read(np.float32, (700,))
        q = m.qkv.read(np.float32, (1, cfg.n_q + 2 * cfg.E))[:, :cfg.n_q]
        want, tol = W.weights(np.ascontiguousarray(q), images(m, L)[0], typ, D, nh, nkv, scale, pos + 1, None, before[:pos + 1], 0.75)
        R.check(got[:pos + 1], want, tol, f"token {pos}")
        pos += 1
    was = [(images(m, x), x["weights"].read(np.float32, (700,))) for x in m.layers]
    m.evict(300, first=4, last=50)
    assert (m.dropped, m.n_cells) == (103, 300)
    for x, (img, w) in zip(m.layers, was):
        cells = pick_ref(w[:403], 300, 4, 50)
        now = x["weights"].read(np.float32, (700,))
        assert (now[:300] == w[cells]).all() and (now[300:] == 0).all()
        for old, new in zip(img, images(m, x)):
            assert (new[:300] == old[cells]).all() and (new[403:] == old[403:]).all()
    for i in range(3):
        m.step_graph(None, pos)
        row = m.qkv.read(np.float32, (1, cfg.n_q + 2 * cfg.E))
        ki, vi = images(m, L)
        cell = 300 + i
        assert (ki[cell] == R.quantize(row[:, cfg.n_q:cfg.n_q + cfg.E], typ)).all()
        if sparse is None:
            o, tol = R.attention(row[:, :cfg.n_q], ki[:cell + 1], vi[:cell + 1], typ, D, nh, nkv, scale)
        else:
            lo, hi = P.bounds(R.values_f32(ki[:cell + 1], typ), D, sparse.block)
            ids = P.select(row[:, :cfg.n_q].reshape(1, nh, D), lo, hi, nh, sparse.block, cell + 1, sparse.n_blocks, 1, 2)
            o, tol = P.attention(row[:, :cfg.n_q], ki, vi, typ, D, nh, nkv, scale, ids, sparse.block, cell + 1)
        R.check(m.att.read(np.float32, (1, nh, D)), o, tol, f"token {pos}")
        assert int(m.params.read(np.int32, (1,))[0]) == pos
        pos += 1
    m.prefill(np.arange(20, dtype=np.int32), 0)                     # another context starts anew
    assert (m.dropped, m.n_cells) == (0, 20) and (L["weights"].read(np.float32, (700,))[20:] == 0).all()
    m.check()
    m.free()


def test_cells_written_anew(dev):
    """A step back: what the tokens that were there got of attention is forgotten, what the others got is not."""
    cfg = LL.tiny_config("tiny-evict")
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 300, kv_type=H.KV_Q4_0, track=1.0)
    nh = cfg.n_head
    L = m.layers[0]
    m.prefill(np.arange(100, dtype=np.int32), 0)
    for i in range(4):
        m.step_graph(7 + i, 100 + i)
    before = L["weights"].read(np.float32, (300,))
    assert (before[:104] > 0).all() and (before[104:] == 0).all()
    before[102:] = 0
    m.step_graph(3, 102)
    got = L["weights"].read(np.float32, (300,))
    assert m.n_cells == 103 and (got[103:] == 0).all() and (got[:103] >= before[:103]).all()
    assert abs(float((got - before).astype(np.float64).sum()) - nh) <= 103 * nh * 2.0 ** -20
    m.prefill(np.arange(5, dtype=np.int32), 50)
    got = L["weights"].read(np.float32, (300,))
    assert m.n_cells == 55 and (got[:50] >= before[:50]).all() and (got[55:] == 0).all()
    m.check()
    m.free()


def test_refusals(dev):
    cfg = LL.tiny_config("tiny-evict")
    w = LL.SyntheticWeights(cfg, cache=True)
    for kw in (dict(sparse=SPARSE), dict(track=1.0)):
        with pytest.raises(ValueError):
            LL.LlamaDecoder(dev, cfg, w, 100, **kw)
    m = LL.LlamaDecoder(dev, cfg, w, 100, kv_type=H.KV_Q4_0)
    with pytest.raises(ValueError):
        m.evict(1)
    m.free()
    m = LL.LlamaDecoder(dev, cfg, w, 100, kv_type=H.KV_Q4_0, track=1.0)
    m.prefill(np.arange(50, dtype=np.int32), 0)
    for args in ((51,), (0,), (20, 4, 64)):
        with pytest.raises(ValueError):
            m.evict(*args)
    m.evict(30, 4, 10)
    with pytest.raises(ValueError):
        m.prefill(np.arange(5, dtype=np.int32), 10)                 # a position that was evicted
    m.free()
