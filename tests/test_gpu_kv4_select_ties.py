"""Blocks whose scores are equal though their bounds are not: the lowest are taken (tsr_hip_kv4_select)."""
import numpy as np
import pytest

import sparse4_ref as P
from test_gpu_kv4_select import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,nh,nkv,D,n_blocks", [
    (1, 8, 2, 128, 300), (3, 1, 1, 64, 300), (2, 12, 2, 256, 100), (80, 4, 2, 64, 300), (70, 20, 1, 128, 130), (64, 2, 2, 512, 100)])
def test_bounds_that_no_query_meets(dev, T, nh, nkv, D, n_blocks):
    """Queries of one sign a channel: of a block one bound a channel counts, and that is every block's alike."""
    rng = np.random.default_rng(T + D)
    q = np.abs(rng.standard_normal((T, nh, D))).astype(np.float32) * np.float32(10.0) ** rng.integers(-2, 2, (T, nh, D)).astype(np.float32)
    sign = np.where(rng.random((nkv, D)) < 0.5, -1.0, 1.0)
    q *= np.repeat(sign, nh // nkv, 0)[None].astype(np.float32)
    met = P.bf16_up(rng.standard_normal((nkv, 1, D)))
    apart = P.bf16_up(np.abs(rng.standard_normal((nkv, n_blocks, D))) * 3.0 ** rng.integers(0, 9, (nkv, n_blocks, D)))
    up = sign[:, None] > 0
    lo, hi = np.where(up, P.bf16_down(met - apart), met), np.where(up, met, P.bf16_up(met + apart))
    hi[:, 7, 0] += np.where(sign[:, 0] > 0, 1.0, 0.0)               # but for one
    hi[:, 7, 0] = P.bf16_up(hi[:, 7, 0])
    want = P.select(q, lo, hi, nh, 32, n_blocks * 32, 20, 0, 2)
    assert (want[:, sign[:, 0] < 0, :18] == np.arange(18)).all()
    assert (run(dev, q, lo, hi, nh, 32, n_blocks * 32, 20, 0, 2) == want).all()
