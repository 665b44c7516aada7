"""The workspace of attention over 4-bit KV caches on the CPU. No GPU calls."""


def test_workspace(native):
    """Rows and pairs of every split lie apart, inside ws_bytes and on their alignment."""
    assert "odd number" in native("kv4_ws_check")
