"""GPU attention over 4-bit KV caches: the error of whole rows in every form of the kernels, against 64 bits."""
import numpy as np
import pytest

import tsr_hip as H
import tsr_synth as S
from attn4_forms import FORMS
from test_gpu_attn4_scales import attend, attention64, check, planes, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [H.KV_Q4_0, H.KV_Q4_1])
@pytest.mark.parametrize("nh,nkv,D,T,n_kv", FORMS)
@pytest.mark.parametrize("kind", ["causal", "window", "mask"])
def test_rows(dev, typ, nh, nkv, D, T, n_kv, kind):
    """Within 2^-19 of a row's length: scores of spread 1 add D / 32 blocks in f32, each off by 2^-24 of some four times the
    spread (the zero point), which over 16 blocks of either sign is 2^-20.8 of a weight; a row is a sum of weights times
    values of either sign. The mask's weights (spread 1) are exact in f16. A product rounded to 11 bits would be 2^-12."""
    k, v = rows(401, n_kv, nkv * D, 0.5)
    ki, kc, vi, vc = planes(dev, typ, k, v)
    q = S.normal(403, T * nh * D).reshape(T, nh * D)
    scale = float(np.float32(1.0 / np.sqrt(D)))
    rng = np.random.default_rng(405)
    runs = mask = None
    if kind == "mask":
        mask = rng.standard_normal((T, n_kv)).astype(np.float16)
        mask[rng.random((T, n_kv)) < 0.4] = -np.inf
        mask[:, 5] = 0.0
    else:
        runs = np.zeros((T, 4), np.uint32)
        runs[:, 1] = n_kv - (np.arange(T)[::-1] % n_kv)
        if kind == "window":
            runs[:, 2], runs[:, 3] = np.maximum(4, runs[:, 1].astype(np.int64) - 100), runs[:, 1]
            runs[:, 1] = np.minimum(4, runs[:, 1])
    check(attend(dev, q, kc, vc, nh, nkv, D, scale, n_kv, runs, mask), attention64(q, ki, vi, typ, nh, nkv, scale, runs, mask))
