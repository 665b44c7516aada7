"""LlamaDecoder's positions, cells and options of long contexts on the CPU, over a pretended device. No GPU calls."""
import numpy as np
import pytest

import tsr_llama as LL


class Piece:
    ptr, nbytes = 0, 1 << 40

    def free(self):
        pass


class Device:
    """Takes every call and does nothing."""

    def alloc(self, n):
        return Piece()

    def __getattr__(self, name):
        return lambda *args, **kw: None


def decoder(kv_size=500, n_cells=0):
    m = object.__new__(LL.LlamaDecoder)
    m.dev, m.cfg, m.kv_size, m.kv4, m.fused = Device(), LL.tiny_config(), kv_size, True, True
    m.layers, m.track, m.n_cells, m._pf = [], 1.0, n_cells, {"x": Piece()}
    m.out_norm = m.wout = m.logits = m.next = m.tok = None
    m.placed = []

    def ubatch(toks, pos0):
        m.placed.append((pos0 - m.dropped, toks.size))
        m.n_cells = pos0 - m.dropped + toks.size

    m._prefill_ubatch = ubatch
    return m


def tokens(n):
    return np.zeros(n, np.int32)


def test_a_refused_prompt_changes_nothing():
    m = decoder(n_cells=403)
    m.evict(300)
    for n, pos0 in ((501, 0), (201, 403)):
        with pytest.raises(ValueError):
            m.prefill(tokens(n), pos0)
        assert (m.dropped, m.n_cells) == (103, 300) and not m.placed
    m.prefill(tokens(7), 403)
    assert m.placed == [(300, 7)]


def test_a_prompt_of_position_0_is_another_context():
    m = decoder(n_cells=403)
    m.evict(300)
    m.prefill(tokens(500), 0)
    assert m.dropped == 0 and m.placed == [(0, 500)]
    m.prefill(tokens(10), 200)                                      # positions are cells again
    assert m.placed[-1] == (200, 10)


def test_a_token_of_position_0_is_another_context():
    m = decoder(n_cells=403)
    m.evict(300)
    m._mask(0, None)
    assert (m.dropped, m.n_cells) == (0, 0)
    m._mask(1, None)


def test_kept_cells_are_not_written_again():
    """Their positions are no longer the decoder's to tell: a step back ends where the eviction was."""
    m = decoder(n_cells=403)
    m.evict(300)
    for pos in (-1, 1, 102, 103, 250, 402):
        with pytest.raises(ValueError):
            m._mask(pos, None)
        with pytest.raises(ValueError):
            m.prefill(tokens(2), pos)
        assert (m.dropped, m.n_cells) == (103, 300) and not m.placed
    m._mask(403, None)
    m.prefill(tokens(60), 403)
    m._mask(410, None)                                              # a step back behind the kept cells
    m.evict(200)
    assert m.dropped == 103 + 107 and m.n_cells == 200
    with pytest.raises(ValueError):
        m._mask(409, None)
    m._mask(410, None)


def test_an_eviction_of_nothing_moves_nothing():
    m = decoder(n_cells=403)
    m.evict(403)
    m._mask(50, None)


@pytest.mark.parametrize("n", [0, 1, 31, 33, 64])
def test_frequency_factors_are_a_pair_s(n):
    """One for each pair of a head's values; the kernels read as many."""
    cfg = LL.tiny_config(rope_scale=LL.RopeScale(4.0, freq_factors=(1.0,) * n))
    with pytest.raises(ValueError):
        LL.LlamaDecoder(None, cfg, None, 100)
