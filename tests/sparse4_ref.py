"""Block bounds, selection and attention over the selected blocks of 4-bit K caches in plain numpy."""
import numpy as np

import kv4_ref as R


def bf16_down(x):
    """The largest bf16 value that is not above x (f32 or exact f64 of f32), as f64."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.floor(m * 256.0), e - 8)


def bf16_up(x):
    return -bf16_down(-np.asarray(x, np.float64))


def bounds(values, D, block, n_kv=None):
    """f32 values [cells, E] -> f64 [E / D, blocks, D] lo and hi of the blocks of the first n_kv cells."""
    n_kv = values.shape[0] if n_kv is None else n_kv
    E = values.shape[1]
    lo, hi = [], []
    for c0 in range(0, n_kv, block):
        part = values[c0:min(n_kv, c0 + block)]
        lo.append(bf16_down(part.min(0)))
        hi.append(bf16_up(part.max(0)))
    return (np.stack(x).reshape(-1, E // D, D).transpose(1, 0, 2) for x in (lo, hi))


def words(w):
    """uint32 words -> f64 lo, hi."""
    w = np.ascontiguousarray(w, np.uint32)
    return (w << np.uint32(16)).view(np.float32).astype(np.float64), (w & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)


def pack(lo, hi):
    """The words of bf16 values."""
    lo, hi = (np.ascontiguousarray(x, np.float32).view(np.uint32) for x in (lo, hi))
    assert not ((lo | hi) & 0xFFFF).any()
    return (lo >> np.uint32(16)) | hi


def cache_rows(seed, n, E):
    """K rows with channels of different sizes and signs, exact zeros and a drift along the cells."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, E)).astype(np.float32)
    x[:, ::7] *= np.float32(5.0)
    x[:, 3::11] = np.abs(x[:, 3::11])
    x[:, 5::13] = 0.0
    x += np.float32(0.7) * np.sin(np.arange(n) / 90.0)[:, None].astype(np.float32)
    return x


def fill(dev, x, typ, which=0, cells=None):
    """A cache of the library that holds the image of x, and what it stands for (f32)."""
    img = R.quantize(x, typ)
    kv = dev.kv(x.shape[1], cells or x.shape[0], typ)
    kv.set_bytes(which, img)
    return kv, R.values_f32(img, typ)


def candidates(run, n_kv, block):
    """The blocks with a cell of a token's two runs, ascending."""
    see = np.zeros(n_kv, bool)
    for lo, hi in ((run[0], run[1]), (run[2], run[3])):
        see[int(lo):max(int(lo), min(int(hi), n_kv))] = True
    return np.unique(np.flatnonzero(see) // block)


def select(q, lo, hi, n_head, block, n_kv, n_sel, n_first, n_last, runs=None):
    """q f32 [T, n_head, D], bounds f64 [n_head_kv, blocks, D] -> int32 [T, n_head_kv, n_sel]."""
    T, nkv = q.shape[0], lo.shape[0]
    G = n_head // nkv
    out = np.full((T, nkv, n_sel), -1, np.int32)
    for t in range(T):
        c = candidates(runs[t] if runs is not None else (0, n_kv, 0, 0), n_kv, block)
        for h in range(nkv):
            mine = c
            if c.size > n_sel:
                qh = q[t, h * G:(h + 1) * G].astype(np.float64)[:, None]
                with np.errstate(invalid="ignore"):
                    s = (np.where(qh < 0, 0.0, qh) * hi[h, c] + np.where(qh > 0, 0.0, qh) * lo[h, c]).sum(-1)
                s = np.where(np.isnan(s).any(0), -np.inf, s.max(0))
                mid = np.arange(n_first, c.size - n_last)
                best = mid[np.argsort(-s[mid], kind="stable")[:n_sel - n_first - n_last]]
                mine = c[np.sort(np.concatenate([np.arange(n_first), best, np.arange(c.size - n_last, c.size)]))]
            out[t, h, :mine.size] = mine
    return out


def attention(q, kimg, vimg, typ, D, n_head, nkv, scale, blocks, block, n_kv, runs=None):
    """f64 attention over listed blocks [T, nkv, n_sel] and how far an f32 result may be from it (kv4_ref.attention's terms,
    which do not depend on the order of the tiles)."""
    T, G, nb = q.shape[0], n_head // nkv, D // 32
    out, tol = np.zeros((T, n_head, D)), np.zeros((T, n_head, D))
    per = kimg.shape[1] // (nkv * nb)
    for h in range(nkv):
        mask = np.full((T, n_kv), -np.inf, np.float16)
        for t in range(T):
            for b in blocks[t, h]:
                if b >= 0:
                    mask[t, b * block:(b + 1) * block] = 0
        part = slice(h * nb * per, (h + 1) * nb * per)
        o, x = R.attention(q.reshape(T, n_head, D)[:, h * G:(h + 1) * G], kimg[:n_kv, part], vimg[:n_kv, part], typ, D, G, 1, scale, runs, mask)
        out[:, h * G:(h + 1) * G], tol[:, h * G:(h + 1) * G] = o, x
    return out, tol
