"""The Llama decoder over 4-bit caches as a conversation uses it: prompts behind generated tokens, caches that are filled anew, forgetting
weights. What the model keeps of its cells (bounds, weights) is checked against its caches."""
import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P
import tsr_hip as H
import tsr_llama as LL
import weights4_ref as W
from test_gpu_llama_kv4 import images

pytestmark = pytest.mark.gpu

SPARSE = LL.SparseAttention(block=32, n_blocks=8, first=1, last=2)


def check_bounds(m, n_cells):
    """The bounds of every layer's full blocks but the newest one, which is attended to without a look at them."""
    c, block = m.cfg, m.sparse.block
    used = (n_cells - 1) // block
    for L in m.layers:
        got = P.words(L["bounds"].read(np.uint32, (c.n_head_kv, m.n_bounds, c.head_dim)))
        want = P.bounds(R.values_f32(images(m, L)[0][:used * block], m.kv_type), c.head_dim, block)
        for a, b in zip(got, want):
            assert (a[:, :used] == b).all()


@pytest.mark.parametrize("typ", [H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("end", [95, 96, 97])
def test_a_prompt_behind_generated_tokens(dev, typ, end):
    """Tokens that end before, on and behind a block's last cell, then a prompt of several ubatches, then tokens again."""
    cfg = LL.tiny_config("tiny-chat")
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 700, kv_type=typ, sparse=SPARSE)
    for L in m.layers:
        L["bounds"].fill(0x55)
    rng = np.random.default_rng(1)
    m.prefill(rng.integers(0, cfg.n_vocab, 40).astype(np.int32), 0)
    for pos in range(40, end):
        m.step_graph(None, pos)
    m.prefill(rng.integers(0, cfg.n_vocab, 200).astype(np.int32), end, 64)
    check_bounds(m, end + 200)
    for i in range(70):
        m.step_graph(None, end + 200 + i)
    check_bounds(m, end + 270)
    m.check()
    m.free()


def test_a_step_ahead(dev):
    """Cells that were passed over hold what the caches had there; their blocks have bounds all the same."""
    cfg = LL.tiny_config("tiny-chat")
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 700, kv_type=H.KV_Q4_0, sparse=SPARSE)
    for L in m.layers:
        L["bounds"].fill(0x55)
    m.prefill(np.arange(40, dtype=np.int32), 0)
    m.step_graph(None, 333)
    check_bounds(m, 334)
    m.prefill(np.arange(40, dtype=np.int32), 500)
    check_bounds(m, 540)
    m.check()
    m.free()


def test_a_history_of_another_context(dev):
    """Cells that a history fills have got no attention, nor have those behind them."""
    cfg = LL.tiny_config("tiny-evict")
    w = LL.SyntheticWeights(cfg)
    m = LL.LlamaDecoder(dev, cfg, w, 300, kv_type=H.KV_Q4_0, track=1.0)
    m.prefill(np.arange(100, dtype=np.int32), 0)
    for i in range(4):
        m.step_graph(None, 100 + i)
    m.prefill_history(w, 60)
    assert m.n_cells == 60
    for L in m.layers:
        assert (L["weights"].read(np.float32, (300,)) == 0).all()
    m.step_graph(3, 60)
    for L in m.layers:
        got = L["weights"].read(np.float32, (300,))
        assert abs(float(got.astype(np.float64).sum()) - cfg.n_head) <= 61 * cfg.n_head * 2.0 ** -20 and (got[61:] == 0).all()
    m.check()
    m.free()


def test_weights_age_by_the_token(dev):
    """A ubatch's tokens are as many as make its weights' age: earlier weights are multiplied once for each."""
    cfg = LL.tiny_config("tiny-evict")
    D, nh, nkv = cfg.head_dim, cfg.n_head, cfg.n_head_kv
    m = LL.LlamaDecoder(dev, cfg, LL.SyntheticWeights(cfg), 300, kv_type=H.KV_Q4_1, track=0.9)
    L = m.layers[-1]
    m.prefill(np.arange(60, dtype=np.int32), 0)
    before = L["weights"].read(np.float32, (300,))
    m.prefill(np.arange(8, dtype=np.int32), 60)
    q = m._pf["qkv"].read(np.float32, (8, cfg.n_q + 2 * cfg.E))[:, :cfg.n_q]
    runs = np.zeros((8, 4), np.int64)
    runs[:, 1] = 61 + np.arange(8)
    want, tol = W.weights(np.ascontiguousarray(q), images(m, L)[0], H.KV_Q4_1, D, nh, nkv, np.float64(np.float32(m.scale)), 68, runs,
                          before[:68], 0.9 ** 8)
    R.check(L["weights"].read(np.float32, (300,))[:68], want, tol, "prompt")
    m.check()
    m.free()
