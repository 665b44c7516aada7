"""LlamaDecoder over 4-bit KV caches on the CPU, over a pretended device: the graph's workspace. No GPU calls."""
import pytest

import tsr_llama as LL


class Piece:
    def __init__(self, nbytes):
        self.nbytes, self.freed = nbytes, False

    def free(self):
        assert not self.freed
        self.freed = True


class Device:
    def __init__(self):
        self.left, self.made = 10, []

    def flash_attn_kv4_ws(self, T, D, n_head, n_head_kv, n_kv):
        return n_kv if n_kv > 256 else 0

    def alloc(self, n):
        if self.left == 0:
            raise MemoryError
        self.left -= 1
        self.made.append(Piece(n))
        return self.made[-1]


def decoder(kv_size):
    m = object.__new__(LL.LlamaDecoder)
    m.dev, m.cfg, m.kv_size = Device(), LL.tiny_config(), kv_size
    m.graph, m.ws, m.n_kv_graph = None, None, 0
    return m


def test_the_workspace_follows_the_cells():
    m = decoder(1000)
    assert m._graph_cells(0) and (m.n_kv_graph, m.ws) == (256, None)
    assert not m._graph_cells(255)
    assert m._graph_cells(256) and m.n_kv_graph == 512 and m.ws.nbytes == 512
    m.graph = Piece(0)
    old, g = m.ws, m.graph
    assert m._graph_cells(999) and m.n_kv_graph == 1000 and m.ws.nbytes == 1000
    assert old.freed and g.freed and m.graph is None
    assert not m._graph_cells(999)


def test_a_workspace_that_could_not_be_had_is_asked_for_again():
    """Without memory the decoder holds no freed workspace, and the next token asks again."""
    m = decoder(4096)
    assert m._graph_cells(300)
    m.dev.left = 0
    for _ in range(2):
        with pytest.raises(MemoryError):
            m._graph_cells(600)
        assert m.ws is None or not m.ws.freed
    m.dev.left = 1
    assert m._graph_cells(600) and m.n_kv_graph == 1024 and m.ws.nbytes == 1024 and not m.ws.freed
    assert not m._graph_cells(600)
