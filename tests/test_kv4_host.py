"""4-bit KV caches on the CPU: the planes' layout, the cuts of an attention call over them and its refusals. No GPU
calls."""


def test_layout_and_plan(native):
    """Every byte of every cell has one place inside the plane; every call's launch is one that the kernels offer."""
    assert "calls cut" in native("kv4_check")


def test_refusals(native):
    """Wrong shapes, types, strides, alignments and workspaces are refused before anything is launched; long calls go
    out in whole chunks."""
    assert "calls" in native("kv4_refusals_check")
