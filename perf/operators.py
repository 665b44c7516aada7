"""The 4-bit KV cache and the attention over it, as cases that can be timed and compared.

Three operators of the library, at sizes of its benchmark, tests and configurations or at generic ones:

  store   kv_set_rows: K and V rows quantized into a q4_0 / q4_1 cache as they are written, and kv_get_rows: the
          cells just written read back as f32 (what a program that checks, shares or shifts a prompt's cells does)
  read    kv_get_rows of a whole context, K and V (a context shift reads K back, rotates and stores it again)
  attn    flash_attn_kv4: attention of f32 query rows over a 4-bit K and V cache. `rows`: "decode" (one token behind
          `hist` cells), "batch" (one token each of `T` sequences that share the cache, ragged lengths up to `hist`),
          "prompt" (`T` tokens behind `hist` cells, causal), "window" (the same, each token sees the last `window`
          cells), "mask" (the same with an f16 mask that also hides and weighs cells). `layers` caches in turn; with
          `graph` the calls of all layers are replayed from a captured graph, as a decode token is

A block is 32 consecutive values of a cell's row: q4_0 stands for f16(d) (n - 8), q4_1 for f16(d) n + f16(m), n of 4
bits. A cache's values are returned as what they stand for.
"""
import math
import zlib

import numpy as np
import torch

own = False                     # False: elementary torch operations; True: the library's operators
_CTX = []


def _lib():
    """The library's binding and the one context that a program holds."""
    if not _CTX:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tesseract-npu_amd"))
        import tsr_hip
        _CTX.extend((tsr_hip, tsr_hip.Device(0)))
    return _CTX


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode token's K and V rows of a Llama-3-8B layer stored and read back: launches only
        {"name": "store_1x1024_q4_0", "kind": "store", "type": "q4_0", "E": 1024, "n": 1, "cells": 4096,
         "scattered": False},
        # the rows of a ragged ubatch of a small model (2 KV heads of 64), to cells all over a fragmented cache
        {"name": "store_333x128_q4_1", "kind": "store", "type": "q4_1", "E": 128, "n": 333, "cells": 8192,
         "scattered": True},
        # the rows of two 2048-token ubatches of a Llama-3-8B layer
        {"name": "store_4096x1024_q4_0", "kind": "store", "type": "q4_0", "E": 1024, "n": 4096, "cells": 8192,
         "scattered": False},
        # a short ragged context of 4 KV heads of 256 read back
        {"name": "read_777x1024_q4_1", "kind": "read", "type": "q4_1", "E": 1024, "n": 777},
        # a long context of a Llama-3-8B layer read back (context shift)
        {"name": "read_32768x1024_q4_0", "kind": "read", "type": "q4_0", "E": 1024, "n": 32768},
        # one token of a small model behind 200 cells: the latency of a chat's first tokens
        {"name": "attn_decode_200_14_2_64", "kind": "attn", "rows": "decode", "type": "q4_0", "n_head": 14,
         "n_head_kv": 2, "D": 64, "T": 1, "hist": 200, "window": 0, "layers": 4, "graph": True},
        # the benchmark's decode attention at 8192 cells
        {"name": "attn_decode_8192_32_8_128", "kind": "attn", "rows": "decode", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 1, "hist": 8192, "window": 0, "layers": 4, "graph": True},
        # a long document behind one token
        {"name": "attn_decode_131071_32_8_128", "kind": "attn", "rows": "decode", "type": "q4_1", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 1, "hist": 131071, "window": 0, "layers": 1, "graph": True},
        # 32 users' tokens decoded together, ragged contexts of up to 4000 cells in one cache
        {"name": "attn_batch32_4000_32_8_128", "kind": "attn", "rows": "batch", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 32, "hist": 4000, "window": 0, "layers": 1, "graph": False},
        # a ragged ubatch of 8 query heads over 4 KV heads of 256 with a mask that hides and weighs cells
        {"name": "attn_mask300_700_8_4_256", "kind": "attn", "rows": "mask", "type": "q4_1", "n_head": 8,
         "n_head_kv": 4, "D": 256, "T": 300, "hist": 700, "window": 0, "layers": 1, "graph": False},
        # the benchmark's prefill ubatch, 512 tokens behind 1536 cells
        {"name": "attn_prompt512_1536_32_8_128", "kind": "attn", "rows": "prompt", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 512, "hist": 1536, "window": 0, "layers": 1, "graph": False},
        # the last ubatch of a long prompt: 2048 tokens behind 6144 cells
        {"name": "attn_prompt2048_6144_32_8_128", "kind": "attn", "rows": "prompt", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 2048, "hist": 6144, "window": 0, "layers": 1, "graph": False},
    ]


_HEADS = [(32, 8, 128), (32, 8, 64), (16, 8, 128), (14, 2, 64), (8, 1, 128), (8, 4, 256), (8, 1, 512)]
_MOST = 2048 * (6144 + 1024) * 32 * 128         # (row, cell) pairs of the largest listed attention, by head values


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "store", "read", "attn", "attn", "attn", "attn", "attn"])
    typ = rng.choice(["q4_0", "q4_1"])
    if kind == "store":
        n = _log(rng, 1, 4096)
        return {"kind": kind, "type": typ, "E": 64 * rng.choice([1, 2, 4, 8, 12, 16]), "n": n,
                "cells": n + _log(rng, 16, 4096), "scattered": rng.random() < 0.5}
    if kind == "read":
        return {"kind": kind, "type": typ, "E": 64 * rng.choice([1, 2, 4, 8, 12, 16]), "n": _log(rng, 1, 32768)}
    nh, nkv, D = rng.choice(_HEADS)
    rows = rng.choice(["decode", "decode", "batch", "prompt", "window", "mask"])
    c = {"kind": kind, "rows": rows, "type": typ, "n_head": nh, "n_head_kv": nkv, "D": D, "T": 1, "hist": 0, "window": 0,
         "layers": 1, "graph": False}
    if rows == "decode":
        c["hist"], c["graph"] = _log(rng, 1, 131071), rng.random() < 0.5
        c["layers"] = 4 if c["hist"] <= 8192 else 1
    elif rows == "batch":
        c["T"], c["hist"] = _log(rng, 2, 64), _log(rng, 16, 2000)
    else:
        c["T"], c["hist"] = _log(rng, 2, 1024), 0 if rng.random() < 0.3 else _log(rng, 16, 6144)
        if rows == "window":
            c["window"] = _log(rng, 16, 2048)
        while c["T"] * (c["hist"] + c["T"]) * nh * D > _MOST:
            c["hist"], c["T"] = c["hist"] // 2, max(2, c["T"] * 2 // 3)
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed, *what):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr((int(seed), what)).encode()))


def _randn(seed, what, *shape):
    return torch.randn(*shape, generator=_gen(seed, what), device="cuda", dtype=torch.float32)


def _k_rows(seed, what, *shape):
    """Rotated key rows: normal values with a few channels larger than the rest."""
    x = _randn(seed, what, *shape)
    x[..., ::61] *= 3.0
    return x


def _v_rows(seed, what, *shape):
    return 0.5 * _randn(seed, what, *shape)


def _runs(case):
    """[T, 4] the cells [lo0, hi0) and [lo1, hi1) that each token sees, and how many cells are in use."""
    T, hist, rows = case["T"], case["hist"], case["rows"]
    r = np.zeros((T, 4), np.int64)
    if rows == "decode":
        r[0, 1] = hist + 1
        return r, hist + 1
    if rows == "batch":
        n = np.random.default_rng(hist).integers(max(1, hist // 8), hist + 1, T)
        end = np.cumsum(n)
        r[:, 0], r[:, 1] = end - n, end
        return r, int(end[-1])
    t = np.arange(T)
    r[:, 1] = hist + t + 1
    if rows == "window":                         # the first 4 cells stay visible, then the last `window` cells
        lo = np.maximum(4, hist + t + 1 - case["window"])
        r[:, 2], r[:, 3] = np.minimum(lo, r[:, 1]), r[:, 1]
        r[:, 1] = np.minimum(4, r[:, 1])
    return r, hist + T


def _mask(case, seed, runs, n_kv):
    """f16 [T, n_kv]: cells hidden here and there (documents packed together), the others weighed by distance."""
    T = case["T"]
    j = torch.arange(n_kv, device="cuda")
    hi = torch.from_numpy(runs[:, 1]).cuda()[:, None]
    m = (j[None, :] - (hi - 1)).float() * (4.0 / n_kv)
    hide = (j[None, :] >= hi) | (torch.rand(T, n_kv, generator=_gen(seed, "mask"), device="cuda") < 0.2)
    hide &= j[None, :] != hi - 1                 # a token sees itself
    return m.masked_fill(hide, float("-inf")).half()


def _type(H, name):
    return {"q4_0": H.KV_Q4_0, "q4_1": H.KV_Q4_1}[name]


def _plain_quantize(x, typ):
    """f32 [..., E] -> codes uint8 [..., E / 32, 32], f16 d and m [..., E / 32] by ggml's rule for one block."""
    b = x.unflatten(-1, (-1, 32))
    if typ == "q4_0":
        a = b.abs()
        i = torch.arange(32, device=x.device)
        first = torch.where(a == a.amax(-1, keepdim=True), i, 32).amin(-1, keepdim=True)
        d = b.gather(-1, first) / -8.0
        inv = torch.where(d == 0, d, 1.0 / d)
        n = (b * inv + 8.5).clamp(max=15.0).to(torch.uint8)
        m = torch.zeros_like(d)
    else:
        m = b.amin(-1, keepdim=True)
        d = (b.amax(-1, keepdim=True) - m) / torch.full_like(m, 15.0)      # (a division by a number multiplies by its inverse)
        inv = torch.where(d == 0, d, 1.0 / d)
        n = ((b - m) * inv + 0.5).clamp(max=15.0).to(torch.uint8)
    return n, d.squeeze(-1).half(), m.squeeze(-1).half()


def _plain_values(n, d, m, typ):
    d = d.float().unsqueeze(-1)
    if typ == "q4_0":
        return (d * (n.float() - 8.0)).flatten(-2)
    return (d * n.float() + m.float().unsqueeze(-1)).flatten(-2)


def _pack(n):
    """codes [..., nb, 32] -> ggml's nibbles [..., nb, 16]: values i and i + 16 share byte i."""
    return n[..., :16] | (n[..., 16:] << 4)


def _unpack(q):
    return torch.cat([q & 15, q >> 4], -1)


def prepare(case, seed):
    st = {"case": case, "own": own}
    kind, typ = case["kind"], case["type"]
    if own:
        H, d = _lib()
        st["d"], t = d, _type(H, typ)
    if kind in ("store", "read"):
        E, n = case["E"], case["n"]
        k, v = _k_rows(seed, "k", n, E), _v_rows(seed, "v", n, E)
        cells = case["cells"] if kind == "store" else n
        idx = torch.arange(n, device="cuda")
        if kind == "store":
            idx = torch.randperm(cells, generator=_gen(seed, "idx"), device="cuda")[:n] if case["scattered"] else \
                idx + (cells - n) // 2
        st["idx"] = idx.contiguous()
        if kind == "store":
            st["k"], st["v"] = k, v
        if own:
            st["kc"], st["vc"] = d.kv(E, cells, type=t), d.kv(E, cells, type=t)
            st["ok"], st["ov"] = torch.empty_like(k), torch.empty_like(v)
            torch.cuda.synchronize()
            if kind == "read":
                d.kv_set_rows(st["kc"], H.KV_K, k.data_ptr(), n, E, st["idx"].data_ptr())
                d.kv_set_rows(st["vc"], H.KV_V, v.data_ptr(), n, E, st["idx"].data_ptr())
                d.sync()
        elif kind == "store":
            z = torch.zeros(cells, E // 32, 16, device="cuda", dtype=torch.uint8)
            s = torch.zeros(cells, E // 32, device="cuda", dtype=torch.float16)
            st["cache"] = [(z.clone(), s.clone(), s.clone()) for _ in range(2)]
        else:
            st["cache"] = [(_pack(q), a, b) for q, a, b in (_plain_quantize(k, typ), _plain_quantize(v, typ))]
        return st
    nh, nkv, D, T, L = case["n_head"], case["n_head_kv"], case["D"], case["T"], case["layers"]
    runs, n_kv = _runs(case)
    st["n_kv"], st["scale"] = n_kv, 1.0 / math.sqrt(D)
    st["q"] = _randn(seed, "q", L, T, nh * D)
    st["runs"] = torch.from_numpy(runs.astype(np.uint32).view(np.int32)).cuda()
    st["mask"] = _mask(case, seed, runs, n_kv) if case["rows"] == "mask" else None
    k, v = _k_rows(seed, "k", L, n_kv, nkv * D), _v_rows(seed, "v", L, n_kv, nkv * D)
    if not own:
        st["cache"] = [(_pack(q), a, b) for q, a, b in (_plain_quantize(k, typ), _plain_quantize(v, typ))]
        return st
    idx = torch.arange(n_kv, device="cuda")
    st["out"] = torch.empty(L, T, nh * D, device="cuda", dtype=torch.float32)
    st["kv"] = []
    torch.cuda.synchronize()
    for i in range(L):
        kc, vc = d.kv(nkv * D, n_kv, type=t), d.kv(nkv * D, n_kv, type=t)
        for c0 in range(0, n_kv, 32768):
            c1 = min(n_kv, c0 + 32768)
            d.kv_set_rows(kc, H.KV_K, k[i, c0:c1].data_ptr(), c1 - c0, nkv * D, idx[c0:c1].data_ptr())
            d.kv_set_rows(vc, H.KV_V, v[i, c0:c1].data_ptr(), c1 - c0, nkv * D, idx[c0:c1].data_ptr())
        st["kv"].append((kc, vc))
    d.sync()
    st["graph"] = None
    if case["graph"]:                            # a decode loop's graph, its workspace with it
        n_ws = d.flash_attn_kv4_ws(T, D, nh, nkv, n_kv)
        st["ws"] = d.alloc(n_ws) if n_ws else None
        d.graph_begin()
        try:
            _attend(st)
        finally:
            st["graph"] = d.graph_end()
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _attend(st):
    """The library's attention over every layer's caches."""
    c, d = st["case"], st["d"]
    nq = c["n_head"] * c["D"]
    mask = st["mask"]
    for i, (kc, vc) in enumerate(st["kv"]):
        d.flash_attn_kv4(st["q"][i].data_ptr(), c["T"], nq, kc, vc, c["D"], c["n_head"], c["n_head_kv"], st["scale"],
                         st["n_kv"], st["out"][i].data_ptr(), nq, runs=st["runs"].data_ptr(),
                         mask=None if mask is None else mask.data_ptr(), mask_stride=st["n_kv"], ws=st.get("ws"))


def _plain_attention(st):
    c = st["case"]
    nh, nkv, D, T, L, n_kv = c["n_head"], c["n_head_kv"], c["D"], c["T"], c["layers"], st["n_kv"]
    k, v = (_plain_values(_unpack(q), d, m, c["type"]).view(L, n_kv, nkv, D).transpose(1, 2).reshape(L * nkv, n_kv, D)
            for q, d, m in st["cache"])
    q = st["q"].view(L, T, nkv, nh // nkv, D).permute(0, 2, 1, 3, 4).reshape(L * nkv, T * (nh // nkv), D)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(st["scale"]).view(L * nkv, T, nh // nkv, n_kv)
    j = torch.arange(n_kv, device="cuda", dtype=torch.int32)
    r = st["runs"][:, :, None]
    seen = ((j >= r[:, 0]) & (j < r[:, 1])) | ((j >= r[:, 2]) & (j < r[:, 3]))
    add = torch.zeros(T, n_kv, device="cuda") if st["mask"] is None else st["mask"].float()
    s += add.masked_fill(~seen, float("-inf"))[:, None, :]
    top = s.amax(-1, keepdim=True)
    s -= torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = s.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(L * nkv, T * (nh // nkv), n_kv), v).view(L * nkv, T, nh // nkv, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.view(L, nkv, T, nh // nkv, D).transpose(1, 2).reshape(L, T, nh * D)


def run(st):
    c = st["case"]
    if c["kind"] == "attn":
        if not own:
            return _plain_attention(st)
        if st["graph"] is not None:
            st["graph"].launch()
        else:
            _attend(st)
        return st["out"]
    if own:
        H, d = _lib()
        E, n, idx = c["E"], c["n"], st["idx"].data_ptr()
        if c["kind"] == "store":
            d.kv_set_rows(st["kc"], H.KV_K, st["k"].data_ptr(), n, E, idx)
            d.kv_set_rows(st["vc"], H.KV_V, st["v"].data_ptr(), n, E, idx)
        d.kv_get_rows(st["kc"], H.KV_K, idx, n, st["ok"].data_ptr(), E)
        d.kv_get_rows(st["vc"], H.KV_V, idx, n, st["ov"].data_ptr(), E)
        return st["ok"], st["ov"]
    if c["kind"] == "store":
        (kq, kd, km), (vq, vd, vm) = st["cache"]
        q, d, m = _plain_quantize(st["k"], c["type"])
        kq[st["idx"]], kd[st["idx"]], km[st["idx"]] = _pack(q), d, m
        q, d, m = _plain_quantize(st["v"], c["type"])
        vq[st["idx"]], vd[st["idx"]], vm[st["idx"]] = _pack(q), d, m
    return tuple(_plain_values(_unpack(q[st["idx"]]), d[st["idx"]], m[st["idx"]], c["type"]) for q, d, m in st["cache"])


def work(case):
    bpv = {"q4_0": 18 / 32, "q4_1": 20 / 32}[case["type"]]
    if case["kind"] in ("store", "read"):
        values = 2 * case["n"] * case["E"]
        if case["kind"] == "store":              # rows in, cells out; cells in, rows out
            return {"bytes": values * (8 + 2 * bpv) + 8 * case["n"], "flops": 4 * values}
        return {"bytes": values * (4 + bpv) + 8 * case["n"], "flops": 2 * values}
    nh, nkv, D, T, L = case["n_head"], case["n_head_kv"], case["D"], case["T"], case["layers"]
    runs, n_kv = _runs(case)
    seen = (runs[:, 1] - runs[:, 0]) + (runs[:, 3] - runs[:, 2])
    used = n_kv
    if case["rows"] == "window":                 # cells that no token sees are not read
        used = min(n_kv, 4 + max(0, n_kv - int(min(runs[0, 2], runs[0, 3]))))
    b = 2 * used * nkv * D * bpv + 8 * T * nh * D + 16 * T
    if case["rows"] == "mask":
        b += 2 * T * n_kv
    return {"bytes": float(L * b), "flops": 4.0 * L * nh * D * float(seen.sum())}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def _round(x, t):
    """One f32 (or f16) rounding of the definition, on values held in 64 bits (twice the bits and more: the sums,
    products and quotients of f32 numbers round to f32 as if they were exact)."""
    return x.to(t).to(torch.float64)


def _block_values(x, typ):
    """What a stored row stands for, f64: the format's own steps are f32 operations, each rounded once."""
    f32, f16 = torch.float32, torch.float16
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    hi, lo = x.max(-1).values, x.min(-1).values
    if typ == "q4_0":
        big = torch.maximum(hi, -lo)
        at_hi = torch.where(x == big[..., None], 1, 0).argmax(-1)      # places of +big and -big: the first one counts
        has_hi, has_lo = hi == big, -lo == big
        at_lo = torch.where(x == -big[..., None], 1, 0).argmax(-1)
        top = torch.where(has_hi & (~has_lo | (at_hi < at_lo)), big, -big)
        d = _round(top / -8.0, f32)
        inv = torch.where(d == 0, torch.zeros_like(d), _round(1.0 / torch.where(d == 0, torch.ones_like(d), d), f32))
        n = torch.floor(_round(_round(x * inv[..., None], f32) + 8.5, f32)).clamp(0, 15)
        return (_round(d, f16)[..., None] * (n - 8.0)).flatten(-2)
    d = _round(_round(hi - lo, f32) / 15.0, f32)
    inv = torch.where(d == 0, torch.zeros_like(d), _round(1.0 / torch.where(d == 0, torch.ones_like(d), d), f32))
    n = torch.floor(_round(_round(_round(x - lo[..., None], f32) * inv[..., None], f32) + 0.5, f32)).clamp(0, 15)
    return (_round(d, f16)[..., None] * n + _round(lo, f16)[..., None]).flatten(-2)


def exact(case, seed):
    typ = case["type"]
    if case["kind"] != "attn":
        k, v = _k_rows(seed, "k", case["n"], case["E"]), _v_rows(seed, "v", case["n"], case["E"])
        return _block_values(k, typ), _block_values(v, typ)
    nh, nkv, D, T, L = case["n_head"], case["n_head_kv"], case["D"], case["T"], case["layers"]
    runs, n_kv = _runs(case)
    q = _randn(seed, "q", L, T, nh * D).double().view(L, T, nh, D)
    k, v = _k_rows(seed, "k", L, n_kv, nkv * D), _v_rows(seed, "v", L, n_kv, nkv * D)
    bias = torch.full((T, n_kv), -math.inf, device="cuda", dtype=torch.float64)
    for t in range(T):
        for lo, hi in ((runs[t, 0], runs[t, 1]), (runs[t, 2], runs[t, 3])):
            bias[t, lo:hi] = 0.0
    if case["rows"] == "mask":
        bias += _mask(case, seed, runs, n_kv).double()
    out = torch.zeros(L, T, nh, D, device="cuda", dtype=torch.float64)
    for i in range(L):
        ki, vi = _block_values(k[i], typ).view(n_kv, nkv, D), _block_values(v[i], typ).view(n_kv, nkv, D)
        for h in range(nh):
            s = q[i, :, h] @ ki[:, h // (nh // nkv)].T.contiguous() / math.sqrt(D) + bias
            any_seen = (s > -math.inf).any(-1)
            out[i, any_seen, h] = torch.softmax(s[any_seen], -1) @ vi[:, h // (nh // nkv)].contiguous()
    return out.view(L, T, nh * D)
