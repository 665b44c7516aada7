"""The Llama decoder over 4-bit KV caches: the cache's stores, the read back and the attention as a model runs them together.
Every attention call of a prefill and of decode steps is checked against the plain computation on what the caches hold at
that moment, the caches' bytes against the format's rule on the rotated rows, and graph replays against the same."""
import numpy as np
import pytest

import kv4_ref as R
import tsr_hip as H
import tsr_llama as LL

pytestmark = pytest.mark.gpu

CONFIGS = [
    (LL.tiny_config(), H.KV_Q4_0),
    (LL.tiny_config("tiny-qwen", wfmt=H.FMT_Q8_0, ofmt=H.FMT_Q8_0, rope_mode=H.ROPE_NEOX, eps=1e-6,
                    rope_base=1000000.0), H.KV_Q4_1),
    (LL.tiny_config("tiny-gqa8", n_head=8, n_head_kv=1, head_dim=128, n_embd=512, n_ff=768, n_vocab=1000), H.KV_Q4_0),
    (LL.tiny_config("tiny-kv8", n_head=16, n_head_kv=8, head_dim=64, n_embd=512, n_ff=768, n_vocab=1000), H.KV_Q4_1),
]


def images(m, L):
    return [L[k].get_bytes(w).reshape(m.kv_size, -1) for w, k in ((0, "kc"), (1, "vc"))]


def check_attention(m, L, qkv, att, T, pos0, what):
    """Rows T of the buffers qkv (rotated) and att, at positions pos0 .., against the layer's caches."""
    c = m.cfg
    w3 = c.n_q + 2 * c.E
    rows = qkv.read(np.float32, (T, w3))
    ki, vi = images(m, L)
    cells = slice(pos0, pos0 + T)
    assert (ki[cells] == R.quantize(rows[:, c.n_q:c.n_q + c.E], m.kv_type)).all(), what
    assert (vi[cells] == R.quantize(rows[:, c.n_q + c.E:], m.kv_type)).all(), what
    runs = np.zeros((T, 4), np.int64)
    runs[:, 1] = pos0 + 1 + np.arange(T)
    want, tol = R.attention(rows[:, :c.n_q], ki[:pos0 + T], vi[:pos0 + T], m.kv_type, c.head_dim, c.n_head, c.n_head_kv,
                            np.float64(np.float32(m.scale)), runs)
    got = att.read(np.float32, (T, c.n_head, c.head_dim))
    R.check(got, want, tol, what)
    # the cells read back are what the images stand for
    ids = m.dev.upload(np.arange(pos0 + T, dtype=np.int64))
    dst = m.dev.alloc(4 * (pos0 + T) * c.E)
    for which, k, img in ((0, "kc", ki), (1, "vc", vi)):
        m.dev.kv_get_rows(L[k], which, ids, pos0 + T, dst, c.E)
        m.dev.sync()
        back = dst.read(np.float32, (pos0 + T, c.E))
        assert (back == R.values_f32(img[:pos0 + T], m.kv_type)).all(), what


@pytest.mark.parametrize("cfg,typ", CONFIGS, ids=["q4k-norm", "q80-neox", "gqa8-d128", "kv8"])
@pytest.mark.parametrize("fused", [True, False], ids=["fused", "separate"])
def test_prefill_and_decode(dev, monkeypatch, cfg, typ, fused):
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 640, fused=fused, kv_type=typ)
    calls, real = [0], dev.flash_attn_kv4

    def checked(q, T, q_stride, kc, vc, *args, **kw):
        real(q, T, q_stride, kc, vc, *args, **kw)
        dev.sync()
        L = next(x for x in m.layers if x["kc"] is kc)
        att = args[5]
        check_attention(m, L, q, att, T, args[4] - T, f"{cfg.name}: {T} rows behind {args[4] - T}, call {calls[0]}")
        calls[0] += 1

    monkeypatch.setattr(dev, "flash_attn_kv4", checked)
    prompt = np.random.default_rng(5).integers(0, cfg.n_vocab, 75).astype(np.int32)
    m.prefill(prompt, 0, 32)                                      # ubatches of 32, 32 and 11
    tok = int(m.next.read(np.int32, (1,))[0])
    for i in range(2):
        m.step(tok if i == 0 else None, 75 + i)
        assert np.isfinite(m.read_logits()).all()
    assert calls[0] == 5 * cfg.n_layer
    m.check()
    m.free()


@pytest.mark.parametrize("cfg,typ", CONFIGS, ids=["q4k-norm", "q80-neox", "gqa8-d128", "kv8"])
def test_decode_graph(dev, cfg, typ):
    """Graph replays across the growth of the graph's cells at 256: the last layer's attention after every replay, and the
    greedy token fed back on the device."""
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 640, kv_type=typ)
    prompt = np.random.default_rng(6).integers(0, cfg.n_vocab, 253).astype(np.int32)
    m.prefill(prompt, 0, 128)
    for i in range(6):
        m.step_graph(None, 253 + i)
        logits = m.read_logits()
        assert np.isfinite(logits).all() and m.read_token() == int(logits.argmax())
        check_attention(m, m.layers[-1], m.qkv, m.att, 1, 253 + i, f"{cfg.name} replay {i}")
    assert m.captures == 2 and m.n_kv_graph == 512
    m.step_async(None, 259)                                       # the same launches without a graph
    check_attention(m, m.layers[-1], m.qkv, m.att, 1, 259, cfg.name)
    m.check()
    m.free()
