"""GPU attention over 4-bit KV caches: scales of the scores at both ends of f32."""
import numpy as np
import pytest

import kv4_ref as R
import tsr_hip as H
import tsr_synth as S
from test_gpu_attn4_scales import BOUND, attend, attention64, check, planes, row_errors, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("scale,k_size", [(3.4e38, 1e-3), (2.0 ** 127, 3e-3), (2.0 ** -126, 1e2), (1.3e-38, 1e3)])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", [(8, 2, 64, 1, 700), (32, 8, 128, 90, 200)])
def test_scores_of_spread_one(dev, typ, scale, k_size, nh, nkv, D, T, n_kv):
    """scale (normal, finite), q and K whose products have the size of ordinary scores."""
    k, v = rows(301, n_kv, nkv * D, 0.5)
    ki, kc, vi, vc = planes(dev, typ, k * np.float32(k_size), v)
    q = S.normal(303, T * nh * D).reshape(T, nh * D).astype(np.float64)
    s = np.float64(np.float32(scale))
    q = (q / (np.sqrt(D) * s * k_size)).astype(np.float32)
    assert np.isfinite(q).all() and (q != 0).all()
    check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv), attention64(q, ki, vi, typ, nh, nkv, s))


@pytest.mark.parametrize("typ", [H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", [(8, 2, 64, 1, 700), (32, 8, 128, 90, 200), (8, 4, 256, 40, 300)])
def test_scores_that_one_cell_wins(dev, typ, nh, nkv, D, T, n_kv):
    """Scores of millions, short of 2^24: one cell takes the row (rows whose second cell is within 100 of the first, twenty times
    what f32 sums of such scores are off by, are left out)."""
    k, v = rows(311, n_kv, nkv * D, 0.5)
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = (S.normal(313, T * nh * D) * np.float32(1.5e6 / np.sqrt(D))).reshape(T, nh * D).astype(np.float32)
    K = R.values(ki, typ).reshape(n_kv, nkv, D)
    s = np.sort(np.stack([q.astype(np.float64).reshape(T, nh, D)[:, h] @ K[:, h // (nh // nkv)].T for h in range(nh)], 1), -1)
    assert np.abs(s).max() < 2.0 ** 24
    clear = s[..., -1] - s[..., -2] > 100.0
    assert clear.mean() > 0.9
    mask = np.zeros((T, n_kv), np.float16)
    want = attention64(q, ki, vi, typ, nh, nkv, 1.0)
    for m in (None, mask):
        got = attend(dev, q, kc, vc, nh, nkv, D, 1.0, n_kv, None, m)
        assert (row_errors(got, want)[clear] <= BOUND).all()
