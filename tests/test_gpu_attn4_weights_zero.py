"""Attention weights of rows whose scores' unit is 0 in f32: queries of zeros or next to them under a small scale. Such a row gives all
the cells that it sees the same weight, as tsr_hip_flash_attn_kv4 does."""
import numpy as np
import pytest

import kv4_ref as R
import sparse4_ref as P
import weights4_ref as W
from test_gpu_attn4_weights import run

pytestmark = pytest.mark.gpu

# rows of one launch form each: a wave a KV head, one, two and four groups of rows, heads of 256 and 512; all with a last tile in part
SHAPES = [(4, 2, 64, 1, 45), (32, 8, 128, 1, 8197), (8, 2, 128, 9, 300), (8, 1, 128, 70, 7001), (4, 2, 256, 5, 130), (4, 1, 512, 3, 100)]


@pytest.mark.parametrize("typ", [R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("scale", [2.0 ** -9, 1e-4, 1e-30, 1e-37])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", SHAPES)
def test_queries_of_zeros(dev, typ, scale, nh, nkv, D, T, n_kv):
    rng = np.random.default_rng(nh + T)
    rows = P.cache_rows(D + T, n_kv, nkv * D)
    kc, ki = P.fill(dev, rows, typ)[0], R.quantize(rows, typ)
    scale = float(np.float32(scale))
    q = rng.standard_normal((T, nh, D)).astype(np.float32)
    q[:, ::2] = 0.0
    q[:, 1::4] *= np.float32(1e-42)                                 # subnormal
    q = q.reshape(T, nh * D)
    runs = np.sort(rng.integers(0, n_kv + 30, (T, 2, 2)), -1).reshape(T, 4)
    runs[0] = (1, n_kv - 1, 0, 0)
    for r in (None, runs):
        R.check(run(dev, q, kc, D, nh, nkv, n_kv, r, scale=scale), *W.weights(q, ki, typ, D, nh, nkv, scale, n_kv, r))
