"""The attention weight that cells get, in 64 bits, with the error that the kernels' arithmetic allows."""
import numpy as np

import kv4_ref as R


def weights(q, kimg, typ, D, n_head, nkv, scale, n_kv, runs=None, before=None, decay=1.0):
    """f64 [n_kv] and how far an f32 result may be from it.

    A score is off by ds as kv4_ref.attention derives it; so a weight p = exp(s - max) / sum, relatively, by its own ds, the
    largest ds of its row (the sum's mean of them is at most that), 2^-22 for exp2 and its argument each time (the sum's and
    its own), and the sum's roundings: 8 terms a tile and lane, one rescaling a tile, some 80 for the joins; the sum over
    rows and row sets rounds once a row (2^-24 of the sum so far each), and the addend once."""
    T, G, nb = q.shape[0], n_head // nkv, D // 32
    see, _ = R.visible(T, n_kv, runs)
    kn, kd, km = R.split(kimg[:n_kv], typ)
    q64 = np.asarray(q, np.float64).reshape(T, n_head, D)
    out, tol = np.zeros(n_kv), np.zeros(n_kv)
    tiles = n_kv / 32 + 1
    with np.errstate(all="ignore"):
        for h in range(n_head):
            kv = slice(h // G * nb, (h // G + 1) * nb)
            K = (kd[:, kv, None] * kn[:, kv] + km[:, kv, None]).reshape(n_kv, D)
            KA = (np.abs(kd[:, kv, None]) * kn[:, kv] + np.abs(km[:, kv, None])).reshape(n_kv, D)
            for t in range(T):
                c = np.flatnonzero(see[t])
                if c.size == 0:
                    continue
                s = K[c] @ q64[t, h] * scale
                if s.max() == -np.inf:
                    continue
                ds = KA[c] @ np.abs(q64[t, h]) * scale * (2.0 ** -22 + (40 + nb) * 2.0 ** -24) + 2.0 ** -23 * np.abs(s)
                p = np.exp(s - s.max())
                p /= p.sum()
                rel = ds + 2 * ds.max() + 2 * (2.0 ** -22 + 2.0 ** -23 * np.abs(s - s.max())) + (10 * tiles + 80) * 2.0 ** -24
                out[c] += p
                tol[c] += p * rel
    tol += out * (T * n_head + 40) * 2.0 ** -24
    if before is not None and decay != 0.0:
        add = np.float64(np.float32(decay)) * np.asarray(before, np.float64)
        out = out + add
        tol += 2.0 ** -24 * np.abs(out)
    return out, tol
