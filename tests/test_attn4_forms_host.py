"""The forms that the precision tests of the attention over 4-bit caches stand for, on the CPU."""
import numpy as np

import kv4_ref as R
import tsr_synth as S
from attn4_forms import FORMS
from test_gpu_attn4_scales import BOUND, attention64, row_errors, rows


def test_each_call_is_its_form(native):
    """Every call is cut into the form that it is listed under; every kernel of every head size is among them, in splits and
    not."""
    out = native("attn4_forms_check", args=tuple(str(v) for call in FORMS for v in call))
    got = [tuple(int(v) for v in line.split()) for line in out.splitlines()]
    assert [g[:2] for g in got] == list(FORMS.values())
    forms = {(call[2],) + form for call, form in FORMS.items()}
    assert forms == ({(D, C, 1) for D in (64, 128, 256, 512) for C in (1, 2, 4) if D >= 128 or C < 4} |
                     {(64, 1, 2), (128, 1, 2)})
    assert any(g[2] == 1 for g in got) and any(g[2] > 1 for g in got)


def test_the_bound_sees_a_lost_piece():
    """A reference whose weights (or queries) are rounded to 11 bits is beyond the bound in every row, one of f32 sums within."""
    k, v = rows(1, 300, 64, 0.5)
    ki, vi = R.quantize(k, R.Q4_0), R.quantize(v, R.Q4_0)
    q = S.normal(3, 40 * 64).reshape(40, 64)
    want = attention64(q, ki, vi, R.Q4_0, 1, 1, 0.125)
    K, V = R.values(ki, R.Q4_0), R.values(vi, R.Q4_0)

    def plain(qt, pt, st):
        s = (q.astype(qt).astype(st) @ K.T.astype(st)) * st(0.125)
        p = np.exp(s - s.max(1, keepdims=True))
        return ((p.astype(pt).astype(st) @ V.astype(st)) / p.sum(1, keepdims=True))[:, None]

    f16, f32, f64 = np.float16, np.float32, np.float64
    assert (row_errors(plain(f64, f16, f64), want) > BOUND).all()
    assert (row_errors(plain(f16, f64, f64), want) > BOUND).all()
    assert (row_errors(plain(f32, f32, f32), want) <= BOUND).all()
