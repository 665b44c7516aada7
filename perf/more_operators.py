"""Operators of long contexts over the 4-bit KV cache, as cases that can be timed and compared.

Three groups of operators of the library, at sizes of its benchmark, tests and configurations or at generic ones:

  rope     rope_scaled: rotary positions of q and k heads scaled for contexts longer than the trained one (YaRN, position
           interpolation, frequency factors), interleaved and half layouts, a part of the head, positions of either sign
           (a context shift turns keys back)
  bounds   kv4_bounds: the smallest and largest value of every channel over each block of a K cache's cells, in bf16,
           rounded outwards
  sparse   kv4_select and flash_attn_kv4_blocks: for every token and KV head the blocks whose bounds allow the largest
           scores, and attention over their cells alone. `rows`: "decode" (one token behind `hist` cells), "batch" (one
           token each of `T` sequences that share the cache, ragged lengths up to `hist`), "prompt" (`T` tokens behind
           `hist` cells, causal). `layers` caches in turn; with `graph` the calls of all layers are replayed from a
           captured graph, as a decode token is
  weights  attn_weights_kv4: the attention weight that each cell gets, summed over tokens and heads, on top of what it
           had before (times `decay`)
  evict    kv_pick and kv_gather: the cells with the largest weights, the first and the last ones among them, in their
           order, and their K and V cells moved into the caches of a shorter context, which is read back

A block of the cache's format is 32 consecutive values of a cell's row: q4_0 stands for f16(d) (n - 8), q4_1 for f16(d) n
+ f16(m), n of 4 bits. A cache's values are returned as what they stand for.
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
        # one decode token's q and k heads of a Llama-3-8B layer, far behind the trained context: a launch
        {"name": "rope_1x40x128_yarn", "kind": "rope", "T": 1, "heads": 40, "head_dim": 128, "n_dims": 128, "mode": 0,
         "base": 500000.0, "factor": 16.0, "ext": 1.0, "orig": 8192, "ff": False, "pos0": 131070, "shift": False},
        # the last ubatch of a long prompt, the half layout over three quarters of a head, with frequency factors
        {"name": "rope_2047x40x128_part", "kind": "rope", "T": 2047, "heads": 40, "head_dim": 128, "n_dims": 96, "mode": 2,
         "base": 10000.0, "factor": 4.0, "ext": 0.0, "orig": 4096, "ff": True, "pos0": 129024, "shift": False},
        # a short ragged context of a small model (2 KV heads of 64)
        {"name": "bounds_333_2_64_q4_1", "kind": "bounds", "type": "q4_1", "n_head_kv": 2, "D": 64, "n": 333, "block": 32},
        # a long context of a Llama-3-8B layer, made anew (after a shift or an eviction)
        {"name": "bounds_131071_8_128_q4_0", "kind": "bounds", "type": "q4_0", "n_head_kv": 8, "D": 128, "n": 131071,
         "block": 64},
        # one token of a small model: the latency of a short context
        {"name": "sparse_decode_4000_14_2_64", "kind": "sparse", "rows": "decode", "type": "q4_0", "n_head": 14,
         "n_head_kv": 2, "D": 64, "T": 1, "hist": 4000, "block": 32, "n_sel": 16, "first": 1, "last": 2, "layers": 4,
         "graph": True},
        # one token behind a long document: 2048 of its 131072 cells
        {"name": "sparse_decode_131071_32_8_128", "kind": "sparse", "rows": "decode", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 1, "hist": 131071, "block": 64, "n_sel": 32, "first": 1, "last": 4, "layers": 1,
         "graph": True},
        # 33 users' tokens decoded together, ragged contexts of up to 6000 cells in one cache
        {"name": "sparse_batch33_6000_8_4_256", "kind": "sparse", "rows": "batch", "type": "q4_1", "n_head": 8,
         "n_head_kv": 4, "D": 256, "T": 33, "hist": 6000, "block": 64, "n_sel": 16, "first": 1, "last": 2, "layers": 1,
         "graph": False},
        # the benchmark's prefill ubatch behind a context that it does not read whole
        {"name": "sparse_prompt512_7680_32_8_128", "kind": "sparse", "rows": "prompt", "type": "q4_0", "n_head": 32,
         "n_head_kv": 8, "D": 128, "T": 512, "hist": 7680, "block": 64, "n_sel": 32, "first": 1, "last": 4, "layers": 1,
         "graph": False},
        # every decode token's weights over the benchmark's context
        {"name": "weights_1_8192_32_8_128", "kind": "weights", "type": "q4_0", "n_head": 32, "n_head_kv": 8, "D": 128,
         "T": 1, "hist": 8192, "decay": 1.0},
        # a prompt's last 64 tokens look back over it once
        {"name": "weights_64_32768_32_8_128", "kind": "weights", "type": "q4_1", "n_head": 32, "n_head_kv": 8, "D": 128,
         "T": 64, "hist": 32768, "decay": 0.9},
        # a small model's cache thinned out
        {"name": "evict_777_of_1500_2_64", "kind": "evict", "type": "q4_1", "E": 128, "n": 1500, "keep": 777, "first": 4,
         "last": 64},
        # a long context of a Llama-3-8B layer thinned out to a quarter
        {"name": "evict_16384_of_65536_8_128", "kind": "evict", "type": "q4_0", "E": 1024, "n": 65536, "keep": 16384,
         "first": 4, "last": 256},
    ]


_HEADS = [(32, 8, 128), (32, 8, 64), (16, 8, 128), (14, 2, 64), (8, 1, 128), (8, 4, 256), (8, 1, 512)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "bounds", "sparse", "sparse", "sparse", "sparse", "weights", "weights", "evict"])
    typ = rng.choice(["q4_0", "q4_1"])
    if kind == "rope":
        hd = rng.choice([64, 80, 128, 256])
        T = _log(rng, 1, 2047 * 128 // hd)
        return {"kind": kind, "T": T, "heads": rng.randint(1, 40), "head_dim": hd, "n_dims": 2 * rng.randint(hd // 8, hd // 2),
                "mode": rng.choice([0, 2]), "base": rng.choice([10000.0, 500000.0]), "factor": rng.choice([1.0, 4.0, 8.0, 32.0]),
                "ext": rng.choice([0.0, 1.0, 1.0]), "orig": rng.choice([2048, 4096, 8192]), "ff": rng.random() < 0.4,
                "pos0": _log(rng, 1, 1000000), "shift": rng.random() < 0.2}
    nh, nkv, D = rng.choice(_HEADS)
    block = rng.choice([32, 64, 128])
    if kind == "bounds":
        return {"kind": kind, "type": typ, "n_head_kv": nkv, "D": D, "n": _log(rng, 1, 131071), "block": block}
    if kind == "weights":
        T, hist = _log(rng, 1, 64), _log(rng, 1, 32768)
        while T > 1 and T * (hist + T) * nh * D > 64 * 32768 * 32 * 128:
            T //= 2
        return {"kind": kind, "type": typ, "n_head": nh, "n_head_kv": nkv, "D": D, "T": T, "hist": hist,
                "decay": rng.choice([0.0, 0.9, 1.0])}
    if kind == "evict":
        n = _log(rng, 8, 65536)
        keep = rng.randint(1, min(n, 16384))
        first = rng.randint(0, min(keep, 8))
        return {"kind": kind, "type": typ, "E": 64 * rng.choice([1, 2, 4, 8, 12, 16]), "n": n, "keep": keep, "first": first,
                "last": rng.randint(0, min(keep - first, 300))}
    rows = rng.choice(["decode", "decode", "batch", "prompt"])
    n_sel = _log(rng, 4, 64)
    c = {"kind": kind, "rows": rows, "type": typ, "n_head": nh, "n_head_kv": nkv, "D": D, "T": 1, "hist": 0, "block": block,
         "n_sel": n_sel, "first": rng.randint(0, 2), "last": rng.randint(0, 2), "layers": 1, "graph": False}
    if rows == "decode":
        c["hist"], c["graph"] = _log(rng, 1, 131071), rng.random() < 0.5
        c["layers"] = 4 if c["hist"] <= 8192 else 1
        return c
    if rows == "batch":
        c["T"], c["hist"] = _log(rng, 2, 64), _log(rng, 16, 4000)
    else:
        c["T"], c["hist"] = _log(rng, 2, 512), 0 if rng.random() < 0.2 else _log(rng, 16, 7680)
    while c["T"] > 1 and c["T"] * c["n_sel"] * block * nh * D > 512 * 2048 * 32 * 128:
        c["T"] = c["T"] * 2 // 3
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed, *what):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr((int(seed), what)).encode()))


def _randn(seed, what, *shape):
    return torch.randn(*shape, generator=_gen(seed, what), device="cuda", dtype=torch.float32)


def _k_rows(seed, what, *shape):
    """Rotated key rows: normal values with a few channels larger than the rest, and a drift along the context, so that
    its blocks differ."""
    x = _randn(seed, what, *shape)
    x[..., ::61] *= 3.0
    n = shape[-2]
    at = torch.arange(n, device="cuda", dtype=torch.float32)[:, None] / 300.0
    x += 0.7 * torch.sin(at + 0.37 * torch.arange(shape[-1], device="cuda", dtype=torch.float32))
    return x


def _v_rows(seed, what, *shape):
    return 0.5 * _randn(seed, what, *shape)


def _runs(case):
    """[T, 2] the cells [lo, hi) that each token sees, and how many cells are in use."""
    T, hist, rows = case["T"], case["hist"], case.get("rows", "prompt")
    r = np.zeros((T, 2), np.int64)
    if rows == "batch":
        n = np.random.default_rng(hist).integers(max(1, hist // 8), hist + 1, T)
        end = np.cumsum(n)
        r[:, 0], r[:, 1] = end - n, end
        return r, int(end[-1])
    r[:, 1] = hist + 1 + np.arange(T)
    return r, hist + T


def _positions(case, seed):
    """int32 [T]: a ubatch's positions; a context shift turns every row by as many positions back."""
    if case["shift"]:
        return torch.full((case["T"],), -case["pos0"], device="cuda", dtype=torch.int32)
    return torch.arange(case["pos0"], case["pos0"] + case["T"], device="cuda", dtype=torch.int32)


def _factors(case, seed):
    if not case["ff"]:
        return None
    return 1.0 + 3.0 * torch.rand(case["n_dims"] // 2, generator=_gen(seed, "ff"), device="cuda", dtype=torch.float32)


def _cell_weights(case, seed):
    """f32 [n]: what cells gather: a few get most of it, some (fresh ones) nothing yet."""
    z = torch.randn(case["n"], generator=_gen(seed, "w"), device="cuda", dtype=torch.float32)
    w = torch.exp(2.0 * z) / case["n"]
    w[torch.rand(case["n"], generator=_gen(seed, "w0"), device="cuda") < 0.05] = 0.0
    return w


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


def _plain_cache(x, typ):
    n, d, m = _plain_quantize(x, typ)
    return _pack(n), d, m


def _own_cache(st, rows, which, cells=None):
    """A cache of the library that holds rows [n, E]."""
    H, d = _lib()
    n, E = rows.shape
    c = d.kv(E, cells or n, type=_type(H, st["case"]["type"]))
    idx = torch.arange(n, device="cuda")
    torch.cuda.synchronize()
    for c0 in range(0, n, 32768):
        c1 = min(n, c0 + 32768)
        d.kv_set_rows(c, which, rows[c0:c1].data_ptr(), c1 - c0, E, idx[c0:c1].data_ptr())
    d.sync()
    return c


def _own_bounds(st, kc, n):
    """The bounds of a cache's n cells: [n_head_kv, blocks, D] words, lo in the low half, hi in the high half."""
    c, (H, d) = st["case"], _lib()
    w = torch.zeros(c["n_head_kv"], -(-n // c["block"]), c["D"], device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    d.kv4_bounds(kc, c["D"], c["block"], n, w.data_ptr())
    d.sync()
    return w


def prepare(case, seed):
    st = {"case": case, "own": own}
    kind = case["kind"]
    if own:
        H, st["d"] = _lib()
    if kind == "rope":
        T, w = case["T"], case["heads"] * case["head_dim"]
        st["qkv"] = _randn(seed, "x", T, w + 2 * case["head_dim"])        # rows of a fused Q|K|V: V heads behind q and k
        st["pos"], st["ff"] = _positions(case, seed), _factors(case, seed)
        if own:
            st["y"] = torch.empty(T, w, device="cuda", dtype=torch.float32)
            st["scaling"] = H.RopeScaling(freq_base=case["base"], freq_scale=1.0 / case["factor"], ext_factor=case["ext"],
                                          n_ctx_orig=case["orig"])
        torch.cuda.synchronize()
        return st
    if kind == "evict":
        n, E = case["n"], case["E"]
        st["w"] = _cell_weights(case, seed)
        k, v = _k_rows(seed, "k", n, E), _v_rows(seed, "v", n, E)
        if not own:
            st["cache"] = [_plain_cache(k, case["type"]), _plain_cache(v, case["type"])]
            return st
        st["kv"] = [_own_cache(st, k, H.KV_K), _own_cache(st, v, H.KV_V)]
        st["to"] = [st["d"].kv(E, case["keep"], type=_type(H, case["type"])) for _ in range(2)]
        st["idx"] = torch.empty(case["keep"], device="cuda", dtype=torch.int64)
        st["kept"] = torch.empty(case["keep"], device="cuda", dtype=torch.float32)
        st["all"] = torch.arange(case["keep"], device="cuda")
        st["rows"] = [torch.empty(case["keep"], E, device="cuda", dtype=torch.float32) for _ in range(2)]
        torch.cuda.synchronize()
        return st
    nkv, D = case["n_head_kv"], case["D"]
    if kind == "bounds":
        k = _k_rows(seed, "k", case["n"], nkv * D)
        if own:
            st["kc"] = _own_cache(st, k, H.KV_K)
            st["bounds"] = _own_bounds(st, st["kc"], case["n"])
        else:
            st["cache"] = _plain_cache(k, case["type"])
        return st
    nh, T, L = case["n_head"], case["T"], case.get("layers", 1)
    runs, n_kv = _runs(case)
    st["n_kv"], st["scale"] = n_kv, 1.0 / math.sqrt(D)
    st["q"] = _randn(seed, "q", L, T, nh * D)
    four = np.concatenate([runs, np.zeros_like(runs)], 1).astype(np.uint32).view(np.int32)
    st["runs"] = torch.from_numpy(np.ascontiguousarray(four)).cuda()
    k = _k_rows(seed, "k", L, n_kv, nkv * D)
    if kind == "weights":
        st["before"] = torch.rand(n_kv, generator=_gen(seed, "before"), device="cuda", dtype=torch.float32)
        if own:
            st["kc"] = _own_cache(st, k[0], H.KV_K)
            st["acc"] = torch.empty(n_kv, device="cuda", dtype=torch.float32)
            torch.cuda.synchronize()
        else:
            st["cache"] = _plain_cache(k, case["type"])
        return st
    v = _v_rows(seed, "v", L, n_kv, nkv * D)
    if not own:
        st["cache"] = [_plain_cache(k, case["type"]), _plain_cache(v, case["type"])]
        st["bounds"] = _plain_bounds(st["cache"][0], case)
        return st
    st["kv"] = [(_own_cache(st, k[i], H.KV_K), _own_cache(st, v[i], H.KV_V)) for i in range(L)]
    st["bounds"] = [_own_bounds(st, kc, n_kv) for kc, _ in st["kv"]]
    st["out"] = torch.empty(L, T, nh * D, device="cuda", dtype=torch.float32)
    st["ids"] = torch.empty(L, T, nkv, case["n_sel"], device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    st["graph"] = None
    if case["graph"]:                            # a decode loop's graph, its workspaces with it
        d = st["d"]
        a = d.kv4_select_ws(T, nkv, case["block"], n_kv)
        b = d.flash_attn_kv4_blocks_ws(T, D, nh, nkv, case["n_sel"], case["block"])
        st["ws"] = d.alloc(max(a, b)) if max(a, b) else None
        d.graph_begin()
        try:
            _own_sparse(st)
        finally:
            st["graph"] = d.graph_end()
    return st


# ---------------------------------------------------------------------------------------------
# one pass of the library
# ---------------------------------------------------------------------------------------------
def _own_sparse(st):
    c, d = st["case"], st["d"]
    nq = c["n_head"] * c["D"]
    for i, (kc, vc) in enumerate(st["kv"]):
        q, ids, runs = st["q"][i].data_ptr(), st["ids"][i].data_ptr(), st["runs"].data_ptr()
        d.kv4_select(q, c["T"], nq, st["bounds"][i].data_ptr(), st["bounds"][i].shape[1], c["D"], c["n_head"], c["n_head_kv"],
                     c["block"], st["n_kv"], c["n_sel"], c["first"], c["last"], ids, runs=runs, ws=st.get("ws"))
        d.flash_attn_kv4_blocks(q, c["T"], nq, kc, vc, c["D"], c["n_head"], c["n_head_kv"], st["scale"], st["n_kv"], ids,
                                c["n_sel"], c["block"], st["out"][i].data_ptr(), nq, runs=runs, ws=st.get("ws"))


def _own_run(st):
    c, d = st["case"], st["d"]
    kind = c["kind"]
    if kind == "rope":
        w = c["heads"] * c["head_dim"]
        d.rope_scaled(st["qkv"].data_ptr(), c["T"], st["qkv"].shape[1], c["head_dim"], c["heads"], c["n_dims"], c["mode"],
                      st["pos"].data_ptr(), st["scaling"], st["y"].data_ptr(), w,
                      freq_factors=None if st["ff"] is None else st["ff"].data_ptr())
        return st["y"]
    if kind == "bounds":
        d.kv4_bounds(st["kc"], c["D"], c["block"], c["n"], st["bounds"].data_ptr())
        return st["bounds"].view(torch.bfloat16).view(*st["bounds"].shape, 2)
    if kind == "sparse":
        if st["graph"] is not None:
            st["graph"].launch()
        else:
            _own_sparse(st)
        return st["ids"], st["out"]
    if kind == "weights":
        d.attn_weights_kv4(st["q"].data_ptr(), c["T"], c["n_head"] * c["D"], st["kc"], c["D"], c["n_head"], c["n_head_kv"],
                           st["scale"], st["n_kv"], st["acc"].data_ptr(), before=st["before"].data_ptr(), decay=c["decay"],
                           runs=st["runs"].data_ptr())
        return st["acc"]
    n, E, idx = c["keep"], c["E"], st["idx"].data_ptr()
    d.kv_pick(st["w"].data_ptr(), c["n"], n, c["first"], c["last"], idx, kept=st["kept"].data_ptr())
    for which in range(2):
        d.kv_gather(st["to"][which], st["kv"][which], which, idx, n)
        d.kv_get_rows(st["to"][which], which, st["all"].data_ptr(), n, st["rows"][which].data_ptr(), E)
    return st["idx"], st["kept"], st["rows"][0], st["rows"][1]


# ---------------------------------------------------------------------------------------------
# one pass in plain operations
# ---------------------------------------------------------------------------------------------
def _plain_rope(st):
    c, n, hd = st["case"], st["case"]["n_dims"], st["case"]["head_dim"]
    i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
    base, scale = float(np.float32(c["base"])), float(np.float32(1.0 / c["factor"]))
    freq = base ** (-2.0 * i / n)
    if st["ff"] is not None:
        freq = freq / st["ff"].double()
    mix, m = torch.zeros_like(i), 1.0
    if c["ext"] != 0.0:
        at = [n * math.log(c["orig"] / (beta * 2.0 * math.pi)) / (2.0 * math.log(base)) for beta in (32.0, 1.0)]
        lo, hi = max(0.0, math.floor(at[0])), min(n - 1.0, math.ceil(at[1]))
        mix = c["ext"] * (1.0 - ((i - lo) / max(0.001, hi - lo)).clamp(0.0, 1.0))
        m = 1.0 + 0.1 * math.log(1.0 / scale)
    angle = st["pos"].double()[:, None] * (freq * (scale * (1.0 - mix) + mix))
    cos, sin = (m * torch.cos(angle)).float()[:, None], (m * torch.sin(angle)).float()[:, None]
    x = st["qkv"][:, :c["heads"] * hd].view(c["T"], c["heads"], hd)
    y = x.clone()
    if c["mode"] == 0:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, a * sin + b * cos
    return y.view(c["T"], -1)


def _outwards(x, up):
    """f32 -> the nearest bf16 that is not below (up) or not above x: cut towards zero, a step on where that is inwards."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    step = (cut != bits) & ((x > 0) == up)
    return (cut + 65536 * step.int()).view(torch.float32).to(torch.bfloat16)


def _plain_bounds(cache, c):
    """bf16 [..., n_head_kv, blocks, D, 2]: (lo, hi) of the cells of each block."""
    q, d, m = cache
    x = _plain_values(_unpack(q), d, m, c["type"])                # [..., n, E]
    n, B = x.shape[-2], c["block"]
    nb = -(-n // B)
    pad = x[..., -1:, :].expand(*x.shape[:-2], nb * B - n, x.shape[-1])
    x = torch.cat([x, pad], -2).unflatten(-2, (nb, B))
    lo, hi = _outwards(x.amin(-2), False), _outwards(x.amax(-2), True)
    return torch.stack([lo, hi], -1).unflatten(-2, (c["n_head_kv"], c["D"])).transpose(-4, -3).contiguous()


def _plain_select(st):
    c = st["case"]
    nh, nkv, D, T, L, B, k = c["n_head"], c["n_head_kv"], c["D"], c["T"], c["layers"], c["block"], c["n_sel"]
    q = st["q"].double().view(L, T, nkv, nh // nkv, D).transpose(1, 2).reshape(L, nkv, T * (nh // nkv), D)
    lo, hi = st["bounds"][..., 0].double(), st["bounds"][..., 1].double()
    nb = lo.shape[2]
    s = torch.matmul(q.clamp(min=0.0), hi.transpose(2, 3).contiguous())
    s += torch.matmul(q.clamp(max=0.0), lo.transpose(2, 3).contiguous())
    s = s.view(L, nkv, T, nh // nkv, nb).amax(3).transpose(1, 2)                # [L, T, nkv, nb]
    b = torch.arange(nb, device="cuda")
    r = st["runs"].long()
    cand = (r[:, 0:1] < r[:, 1:2]) & (b * B < r[:, 1:2]) & (b * B + B > r[:, 0:1])
    before, behind = cand.long().cumsum(1), cand.long().flip(1).cumsum(1).flip(1)
    forced = (before <= c["first"]) | (behind <= c["last"])
    s = s.masked_fill(forced[:, None], math.inf).masked_fill(~cand[:, None], -math.inf)
    top, ids = torch.sort(s, dim=-1, descending=True, stable=True)
    ids = ids[..., :k].masked_fill(top[..., :k] == -math.inf, nb).sort(-1).values
    ids = torch.nn.functional.pad(ids, (0, k - ids.shape[-1]), value=nb)
    return torch.where(ids == nb, -1, ids).int()


def _plain_sparse(st):
    c = st["case"]
    nh, nkv, D, T, L, B, k = c["n_head"], c["n_head_kv"], c["D"], c["T"], c["layers"], c["block"], c["n_sel"]
    ids = _plain_select(st)
    cells = (ids.long()[..., None] * B + torch.arange(B, device="cuda")).view(L, T, nkv, k * B)
    r = st["runs"].long()[None, :, None]
    seen = (cells >= r[..., 0:1]) & (cells < r[..., 1:2])
    at = cells.clamp(0, st["n_kv"] - 1)
    l, h = torch.arange(L, device="cuda").view(L, 1, 1, 1), torch.arange(nkv, device="cuda").view(1, 1, nkv, 1)

    def rows(cache):
        q, d, m = (x.view(L, st["n_kv"], nkv, D // 32, *x.shape[3:])[l, at, h] for x in cache)
        return _plain_values(_unpack(q), d, m, c["type"])         # [L, T, nkv, k B, D]

    s = torch.matmul(st["q"].view(L, T, nkv, nh // nkv, D), rows(st["cache"][0]).transpose(3, 4).contiguous()) * st["scale"]
    s = s.masked_fill(~seen[:, :, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(st["cache"][1]))
    return ids, torch.where(total > 0, o / total, torch.zeros_like(o)).view(L, T, nh * D)


def _plain_weights(st):
    c = st["case"]
    nh, nkv, D, T, n = c["n_head"], c["n_head_kv"], c["D"], c["T"], st["n_kv"]
    q, d, m = st["cache"]
    k = _plain_values(_unpack(q), d, m, c["type"]).view(n, nkv, D).permute(1, 2, 0).contiguous()
    q = st["q"].view(T, nkv, nh // nkv, D).transpose(0, 1).reshape(nkv, T * (nh // nkv), D)
    s = (torch.matmul(q, k) * st["scale"]).view(nkv, T, nh // nkv, n)
    j, r = torch.arange(n, device="cuda"), st["runs"].long()
    seen = (j >= r[:, 0:1]) & (j < r[:, 1:2])
    s = s.masked_fill(~seen[None, :, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    w = (s / s.sum(-1, keepdim=True)).sum((0, 1, 2), dtype=torch.float64)
    return (c["decay"] * st["before"].double() + w).float() if c["decay"] else w.float()


def _plain_evict(st):
    c, w, n = st["case"], st["w"], st["case"]["n"]
    key = w.clone()
    key[:c["first"]] = math.inf
    key[n - c["last"]:] = math.inf
    idx = torch.sort(key, descending=True, stable=True).indices[:c["keep"]].sort().values
    k, v = (_plain_values(_unpack(q[idx]), d[idx], m[idx], c["type"]) for q, d, m in st["cache"])
    return idx, w[idx], k, v


def run(st):
    if own:
        return _own_run(st)
    kind = st["case"]["kind"]
    if kind == "rope":
        return _plain_rope(st)
    if kind == "bounds":
        return _plain_bounds(st["cache"], st["case"])
    if kind == "sparse":
        return _plain_sparse(st)
    if kind == "weights":
        return _plain_weights(st)
    return _plain_evict(st)


def work(case):
    kind = case["kind"]
    if kind == "rope":
        v = case["T"] * case["heads"] * case["head_dim"]
        return {"bytes": 8 * v + 4 * case["T"], "flops": 3 * case["T"] * case["heads"] * case["n_dims"]}
    bpv = {"q4_0": 18 / 32, "q4_1": 20 / 32}[case["type"]]
    if kind == "evict":
        # the weights in, the list and its weights out; cells in, cells out; cells in, rows out
        return {"bytes": 4 * case["n"] + 12 * case["keep"] + 2 * case["keep"] * case["E"] * (3 * bpv + 4),
                "flops": 4 * case["keep"] * case["E"]}
    nkv, D = case["n_head_kv"], case["D"]
    if kind == "bounds":
        nb = -(-case["n"] // case["block"])
        return {"bytes": nkv * D * (case["n"] * bpv + 4 * nb), "flops": 4 * case["n"] * nkv * D}
    nh, T, L = case["n_head"], case["T"], case.get("layers", 1)
    runs, n_kv = _runs(case)
    cells = runs[:, 1] - runs[:, 0]
    if kind == "weights":
        return {"bytes": n_kv * nkv * D * bpv + 4 * T * nh * D + 8 * n_kv, "flops": 2.0 * nh * D * float(cells.sum())}
    B = case["block"]
    blocks = -(-runs[:, 1] // B) - runs[:, 0] // B
    some = np.minimum(cells, case["n_sel"] * B)
    used = min(n_kv, int(some.sum()))                             # (tokens may pick the same cells; at least one's)
    if case["rows"] == "prompt":
        used = int(some.max())
    b = 4 * nkv * D * -(-n_kv // B) + 2 * used * nkv * D * bpv + 8 * T * nh * D + 4 * T * nkv * case["n_sel"]
    return {"bytes": float(L * b), "flops": 4.0 * L * nh * D * float(some.sum() + blocks.sum())}


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


def _exact_bounds(values, case):
    """The bf16 values below and above: 8 significant bits, floor and ceil. [n_head_kv, blocks, D, 2] f64."""
    out = []
    for part in values.split(case["block"]):
        m, e = torch.frexp(torch.stack([part.amin(0), part.amax(0)]))
        m = torch.stack([torch.floor(256.0 * m[0]), torch.ceil(256.0 * m[1])])
        out.append(torch.ldexp(m, e - 8).T)
    return torch.stack(out, 1).unflatten(0, (case["n_head_kv"], case["D"])).transpose(1, 2)


def _exact_rope(case, seed):
    T, H, hd, n = case["T"], case["heads"], case["head_dim"], case["n_dims"]
    x = _randn(seed, "x", T, H * hd + 2 * hd)[:, :H * hd].double().view(T, H, hd)
    pos, ff = _positions(case, seed).double(), _factors(case, seed)
    base, scale = float(np.float32(case["base"])), float(np.float32(1.0 / case["factor"]))
    y = x.clone()
    for i in range(n // 2):
        theta = math.exp(-2.0 * i / n * math.log(base)) / (1.0 if ff is None else float(ff[i]))
        f, m = theta * scale, 1.0
        if case["ext"]:
            # pairs that turn more than 32 times in the trained context keep their angle, those below one turn are
            # interpolated, a ramp of the pair's number between
            lo = max(0, math.floor(n / 2 * math.log(case["orig"] / (64.0 * math.pi)) / math.log(base)))
            hi = min(n - 1, math.ceil(n / 2 * math.log(case["orig"] / (2.0 * math.pi)) / math.log(base)))
            kept = case["ext"] * (1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
            f, m = theta * scale * (1.0 - kept) + theta * kept, 1.0 - 0.1 * math.log(scale)
        u, w = (2 * i, 2 * i + 1) if case["mode"] == 0 else (i, i + n // 2)
        c, s = m * torch.cos(pos * f)[:, None], m * torch.sin(pos * f)[:, None]
        y[..., u], y[..., w] = x[..., u] * c - x[..., w] * s, x[..., w] * c + x[..., u] * s
    return y.view(T, H * hd)


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(case, seed)
    typ = case["type"]
    if kind == "evict":
        n = case["n"]
        w = _cell_weights(case, seed).cpu().numpy().astype(np.float64)
        rest = np.arange(case["first"], n - case["last"])
        best = rest[np.lexsort((rest, -w[rest]))][:case["keep"] - case["first"] - case["last"]]
        idx = np.unique(np.concatenate([np.arange(case["first"]), best, np.arange(n - case["last"], n)]))
        at = torch.from_numpy(idx).cuda()
        k, v = _k_rows(seed, "k", n, case["E"])[at], _v_rows(seed, "v", n, case["E"])[at]
        return at, torch.from_numpy(w[idx]).cuda(), _block_values(k, typ), _block_values(v, typ)
    nkv, D = case["n_head_kv"], case["D"]
    if kind == "bounds":
        return _exact_bounds(_round(_block_values(_k_rows(seed, "k", case["n"], nkv * D), typ), torch.float32), case)
    nh, T, L = case["n_head"], case["T"], case.get("layers", 1)
    G = nh // nkv
    runs, n_kv = _runs(case)
    q = _randn(seed, "q", L, T, nh * D).double().view(L, T, nkv, G, D)
    k = _k_rows(seed, "k", L, n_kv, nkv * D)
    if kind == "weights":
        kx = _block_values(k[0], typ).view(n_kv, nkv, D)
        total = case["decay"] * torch.rand(n_kv, generator=_gen(seed, "before"), device="cuda", dtype=torch.float32).double()
        for t in range(T):
            lo, hi = runs[t]
            for h in range(nkv):
                total[lo:hi] += torch.softmax(q[0, t, h] @ kx[lo:hi, h].T.contiguous() / math.sqrt(D), -1).sum(0)
        return total
    v = _v_rows(seed, "v", L, n_kv, nkv * D)
    B, k_sel = case["block"], case["n_sel"]
    ids = torch.full((L, T, nkv, k_sel), -1, dtype=torch.int32)
    out = torch.zeros(L, T, nkv, G, D, device="cuda", dtype=torch.float64)
    for i in range(L):
        kx, vx = _block_values(k[i], typ).view(n_kv, nkv, D), _block_values(v[i], typ).view(n_kv, nkv, D)
        bounds = _exact_bounds(_round(kx.view(n_kv, nkv * D), torch.float32), case)
        for t in range(T):
            lo, hi = (int(x) for x in runs[t])
            b0, b1 = lo // B, -(-hi // B)
            least, most = bounds[:, b0:b1, :, 0], bounds[:, b0:b1, :, 1]
            score = torch.stack([torch.maximum(q[i, t, :, g, None] * least, q[i, t, :, g, None] * most).sum(-1)
                                 for g in range(G)]).amax(0).cpu().numpy()
            for h in range(nkv):
                n = b1 - b0
                forced = set(range(min(n, case["first"]))) | set(range(max(0, n - case["last"]), n))
                rest = [x for x in np.argsort(-score[h], kind="stable") if x not in forced]
                mine = sorted((forced | set(rest[:max(0, k_sel - len(forced))])) if n > k_sel else range(n))
                ids[i, t, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32) + b0
                at = torch.cat([torch.arange(max(lo, (b0 + x) * B), min(hi, (b0 + x + 1) * B)) for x in mine]).cuda()
                p = torch.softmax(q[i, t, h] @ kx[at, h].T.contiguous() / math.sqrt(D), -1)
                out[i, t, h] = p @ vx[at, h]
    return ids.cuda(), out.view(L, T, nh * D)
