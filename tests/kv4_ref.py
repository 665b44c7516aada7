"""4-bit KV cache blocks (ggml's q4_0 / q4_1) and attention over them in plain numpy, 64 bits where sums are made, with
the error that the kernels' arithmetic allows derived term by term."""
import numpy as np

Q4_0, Q4_1 = 1, 2
BLOCK = {Q4_0: 18, Q4_1: 20}


def quantize(x, typ):
    """f32 [n, E] -> the ggml image uint8 [n, E / 32 * BLOCK]: every step one f32 operation, NaN stored as 0."""
    x = np.ascontiguousarray(x, np.float32)
    n, E = x.shape
    f = np.float32
    with np.errstate(all="ignore"):
        b = np.where(np.isnan(x), f(0), x).reshape(n, E // 32, 32)
        if typ == Q4_0:
            a = np.abs(b)
            top = np.take_along_axis(b, a.argmax(-1)[..., None], -1)[..., 0]
            d, m, half = top / f(-8), np.zeros_like(top), f(8.5)
            inv = np.where(d != 0, f(1) / d, f(0)).astype(f)
            y = b * inv[..., None] + half
        else:
            m = b.min(-1)
            d = (b.max(-1) - m) / f(15)
            inv = np.where(d != 0, f(1) / d, f(0)).astype(f)
            y = (b - m[..., None]) * inv[..., None] + f(0.5)
        assert y.dtype == np.float32
        q = np.clip(np.trunc(np.nan_to_num(y, nan=0.0, posinf=15.0, neginf=0.0)), 0, 15).astype(np.uint8)
        heads = [d.astype(np.float16)] + ([m.astype(np.float16)] if typ == Q4_1 else [])
    out = np.empty((n, E // 32, BLOCK[typ]), np.uint8)
    for i, h in enumerate(heads):
        out[..., 2 * i:2 * i + 2] = np.ascontiguousarray(h).view(np.uint8).reshape(n, E // 32, 2)
    out[..., 2 * len(heads):] = q[..., :16] | (q[..., 16:] << 4)
    return out.reshape(n, -1)


def split(img, typ):
    """image [n, bytes] -> codes f64 [n, nb, 32], d and m f64 [n, nb]."""
    n = img.shape[0]
    b = img.reshape(n, -1, BLOCK[typ])
    d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0].astype(np.float64)
    m = np.ascontiguousarray(b[..., 2:4]).view(np.float16)[..., 0].astype(np.float64) if typ == Q4_1 else -8.0 * d
    q = b[..., BLOCK[typ] - 16:]
    return np.concatenate([q & 15, q >> 4], -1).astype(np.float64), d, m


def values(img, typ):
    """What the image stands for, f64 [n, E]."""
    n, d, m = split(img, typ)
    with np.errstate(all="ignore"):
        v = d[..., None] * (n - 8.0) if typ == Q4_0 else d[..., None] * n + m[..., None]
    return v.reshape(img.shape[0], -1)


def values_f32(img, typ):
    """values() as the read gives it: d n + m rounded once (d (n - 8) is exact)."""
    with np.errstate(all="ignore"):
        return values(img, typ).astype(np.float32)


def visible(T, n_kv, runs=None, mask=None):
    """[T, n_kv] bool, and the additive mask f64."""
    j = np.arange(n_kv)[None]
    see = np.ones((T, n_kv), bool)
    add = np.zeros((T, n_kv))
    if runs is not None:
        r = np.asarray(runs, np.int64)
        see = ((j >= r[:, 0:1]) & (j < r[:, 1:2])) | ((j >= r[:, 2:3]) & (j < r[:, 3:4]))
    if mask is not None:
        add = mask[:T, :n_kv].astype(np.float64)
        see = see & (add != -np.inf)
    return see, add


def attention(q, kimg, vimg, typ, D, n_head, n_head_kv, scale, runs=None, mask=None):
    """f64 result [T, n_head, D] and how far an f32 result may be from it.

    Scores: q enters as two f16 pieces (2^-22 of |q|) and a product sum of 32 terms is made in f32 on top of the zero
    point, D / 32 of them added: with A = sum d (n + 8) |q| (q4_1: + |m| |q|) an error of at most
    A (2^-22 + (40 + D / 32) 2^-24), and 2^-23 |s| for the change of base. A weight p is off by twice that, relatively
    (its own score and the maximum's), and by 2^-22 for exp2 and its argument. Results: pieces of p d keep 2^-22; sums of 64
    terms a tile and one step a tile more; joining splits rounds a few times more: with B = sum p d (n + 8) (q4_1: + p |m|)
    an error of at most B (2^-21 + (2 tiles + 80) 2^-24), the same for the sum of weights."""
    T, G, n_kv = q.shape[0], n_head // n_head_kv, kimg.shape[0]
    see, add = visible(T, n_kv, runs, mask)
    kn, kd, km = split(kimg, typ)
    vn, vd, vm = split(vimg, typ)
    q64 = np.asarray(q, np.float64).reshape(T, n_head, D)
    out, tol = np.zeros((T, n_head, D)), np.zeros((T, n_head, D))
    tiles = n_kv / 32 + 1
    nb = D // 32
    with np.errstate(all="ignore"):
        for h in range(n_head):
            kv = slice(h // G * nb, (h // G + 1) * nb)
            K = (kd[:, kv, None] * kn[:, kv] + km[:, kv, None]).reshape(n_kv, D)
            V = (vd[:, kv, None] * vn[:, kv] + vm[:, kv, None]).reshape(n_kv, D)
            KA = (np.abs(kd[:, kv, None]) * kn[:, kv] + np.abs(km[:, kv, None])).reshape(n_kv, D)
            VA = (np.abs(vd[:, kv, None]) * vn[:, kv] + np.abs(vm[:, kv, None])).reshape(n_kv, D)
            for t in range(T):
                c = np.flatnonzero(see[t])
                s = K[c] @ q64[t, h] * scale + add[t, c]
                if c.size == 0 or s.max() == -np.inf:
                    continue
                ds = KA[c] @ np.abs(q64[t, h]) * scale * (2.0 ** -22 + (40 + nb) * 2.0 ** -24) + 2.0 ** -23 * (
                    np.abs(s) + np.abs(add[t, c]))
                p = np.exp(s - s.max())
                rel = ds + ds[s.argmax()] + 2.0 ** -22 + 2.0 ** -23 * np.abs(s - s.max())
                acc = 2.0 ** -21 + (2 * tiles + 80) * 2.0 ** -24
                out[t, h] = p @ V[c] / p.sum()
                tol[t, h] = ((p * rel) @ VA[c] + p @ VA[c] * 2 * acc) / p.sum() + np.abs(out[t, h]) * (
                    (p * rel).sum() / p.sum())
    return out, tol


def check(got, want, tol, what=""):
    got = np.asarray(got, np.float64).reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    fine = np.isfinite(want)
    assert (np.isfinite(got) == fine).all(), f"{what}: finite where the result is not, or not finite where it is"
    bad &= fine
    if bad.any():
        i = np.argwhere(bad)[0]
        i = tuple(i)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} beyond the bound; first at {i}: got {got[i]!r} want "
                             f"{want[i]!r} bound {tol[i]!r}; worst {np.max((np.abs(got - want) / (tol + 1e-30))[fine]):.3g}x")
