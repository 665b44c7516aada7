"""The argument checks of the scaled rotary positions on the CPU. No GPU calls."""


def test_refusals(native):
    assert "calls" in native("rope_scaled_refusals_check")
