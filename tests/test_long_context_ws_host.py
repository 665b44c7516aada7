"""Workspaces of the calls of long contexts on the CPU: more cells never need less. No GPU calls."""


def test_weights(native):
    assert "workspaces" in native("weights_ws_check")


def test_selection(native):
    assert "workspaces" in native("select_ws_check")
