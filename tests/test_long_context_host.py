"""The argument checks, cuts and workspaces of sparse attention over 4-bit KV caches and of eviction by attention weight, on the
CPU. No GPU calls."""


def test_sparse_refusals(native):
    assert "calls" in native("sparse4_refusals_check")


def test_evict_refusals(native):
    assert "calls" in native("evict_refusals_check")
