"""Operators of a layer whose cache has 4 bits and whose projections have 8: the cache as it is written, read back and
attended to, the norms of queries and keys with their rotation, and 8-bit integer products.

Five kinds of call, at the head shapes of the package's presets:

  cache4   K and V of some tokens are quantised into a 4-bit cache (e2m1 codes, a power-of-two scale per 32 dims) and
           read back.  Returns the K and V that the cache stands for.
  attn4    ragged verify / decode / prompt attention over a 4-bit cache: a query at position p reads positions 0 .. p.
  tree4    the same for trees of drafted tokens: a node reads the prefix, its ancestors and itself.
  norms    the queries and keys of a fused qkv row, normalised head by head and rotated; K and V go into the bf16 or fp32
           cache.  Returns the queries and the caches.
  linear8  activations quantised to 8-bit integers, a scale per token, times a weight of 8-bit integers, a scale per
           output channel; with the residual added or silu(gate) * up taken in the same call.

`run` is each operator's plain form where `own` is false, and the calls of this framework where it is true.  Caches are
in the framework's storage layouts in both.  A case's block structure (contexts, tokens, trees) follows from the case
alone (`shape` seeds it); the seed of `prepare` makes the values.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"

# query heads, KV heads, head_dim
HEADS = {"1b": (32, 8, 64), "8b": (32, 8, 128), "7b": (32, 32, 128)}
# output channels (gate and up together for silu), inputs, epilogue of the presets' projections
LINEAR = {"1b_o": (2048, 2048, "residual"), "1b_w13": (16384, 2048, "silu"), "1b_w2": (2048, 8192, "residual"),
          "7b_qkv": (12288, 4096, "none"), "7b_w2": (4096, 11008, "residual"), "8b_qkv": (6144, 4096, "none"),
          "8b_o": (4096, 4096, "residual"), "8b_w13": (28672, 4096, "silu"), "8b_w2": (4096, 14336, "residual")}
EPS, THETA = 1e-5, 500000.0


# ----------------------------------------------------------------------------- the cases

def _attend_case(name, kind, heads, requests, t, ctx, median=0, shape=1):
    """requests blocks of t[0]..t[1] tokens (tree nodes) at contexts ctx[0]..ctx[1]: uniform, or with median > 0
    lognormal around it."""
    c = {"kind": kind, "heads": heads, "requests": requests, "t_lo": t[0], "t_hi": t[1], "ctx_lo": ctx[0],
         "ctx_hi": ctx[1], "median": median, "shape": shape}
    return {"name": name, **c} if name else c


def _token_case(name, kind, heads, tokens, requests, dtype="bf16", shape=1):
    """tokens new tokens over requests cache rows (a run of consecutive positions in each)."""
    c = {"kind": kind, "heads": heads, "tokens": tokens, "requests": requests, "dtype": dtype, "shape": shape}
    return {"name": name, **c} if name else c


def _linear_case(name, weight, tokens, dtype="bf16"):
    c = {"kind": "linear8", "weight": weight, "tokens": tokens, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed() -> list:
    return [
        # a decode step of 32 requests writes one token each
        _token_case("cache4_8b_32", "cache4", "8b", 32, 32),
        # a long prompt of odd length goes into the cache in one call
        _token_case("cache4_8b_4001", "cache4", "8b", 4001, 1),
        # single-stream decoding: one query token, the smallest attention call
        _attend_case("attn4_1b_b1", "attn4", "1b", 1, (1, 1), (300, 400)),
        # one request with a very long context (the 1B shape's positions go to 131072), verifying a few drafts
        _attend_case("attn4_1b_long", "attn4", "1b", 1, (5, 5), (100001, 100001)),
        # verification in a large batch: contexts of median 1500 up to 8183, 1 to 9 tokens each
        _attend_case("attn4_8b_b256", "attn4", "8b", 256, (1, 9), (64, 8183), median=1500),
        # a piece of a prompt, of odd length, on top of what the cache holds already
        _attend_case("attn4_8b_prompt", "attn4", "8b", 1, (1001, 1001), (900, 1100)),
        # trees of 20 to 40 nodes over the 4-bit cache of an MHA model
        _attend_case("tree4_7b_b16", "tree4", "7b", 16, (20, 40), (256, 1100)),
        # a decode step of 32 requests
        _token_case("norms_8b_32", "norms", "8b", 32, 32),
        # a prompt of odd length
        _token_case("norms_8b_4001", "norms", "8b", 4001, 1),
        # single-stream decoding: the smallest projection
        _linear_case("linear8_1b_o_1", "1b_o", 1),
        # a decode batch's gate and up projections
        _linear_case("linear8_8b_w13_32", "8b_w13", 32),
        # a prompt of odd length
        _linear_case("linear8_8b_w2_2001", "8b_w2", 2001),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["cache4", "attn4", "attn4", "tree4", "norms", "linear8", "linear8"])
    if kind == "linear8":
        weight = rng.choice(sorted(LINEAR))
        n, k, _ = LINEAR[weight]
        fp32 = rng.random() < 0.2
        return _linear_case(None, weight, _log(rng, 1, min(4001, 2001 * 4096 * 14336 // (n * k))),
                            dtype="fp32" if fp32 else "bf16")
    heads = rng.choice(sorted(HEADS))
    shape = rng.randrange(1, 1 << 20)
    hkv = HEADS[heads][1]
    if kind in ("cache4", "norms"):
        fp32 = rng.random() < 0.25
        tokens = _log(rng, 1, 1000 if hkv == 32 or fp32 else 4001)
        return _token_case(None, kind, heads, tokens, _log(rng, 1, min(tokens, 64)), dtype="fp32" if fp32 else "bf16",
                           shape=shape)
    if kind == "tree4":
        requests = _log(rng, 1, 32 if hkv == 8 else 8)
        return _attend_case(None, kind, heads, requests, (rng.randint(1, 12), rng.randint(12, 64)),
                            (rng.randint(1, 64), _log(rng, 65, 1280)), shape=shape)
    form = rng.random()
    if form < 0.25:                                              # few requests, a long context
        hi = _log(rng, 4000, 100000 if heads == "1b" else 8000)
        return _attend_case(None, kind, heads, rng.randint(1, 2), (1, rng.randint(1, 9)), (hi // 2, hi), shape=shape)
    if form < 0.5:                                               # pieces of prompts
        return _attend_case(None, kind, heads, rng.randint(1, 3), (10, _log(rng, 11, 500)), (0, _log(rng, 1, 1000)),
                            shape=shape)
    requests = _log(rng, 1, 256 if hkv == 8 else 48)
    return _attend_case(None, kind, heads, requests, (1, rng.randint(1, 9)), (rng.randint(1, 64), _log(rng, 65, 2800)),
                        shape=shape)


# ----------------------------------------------------------------------------- what a case consists of

def _dtype(case):
    return torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16


def _blocks(case):
    """(rows, pos0, T) of a case's blocks in packed order (T ascending), int64; rows are a shuffle of the cache's."""
    r = random.Random(case["shape"])
    n = case["requests"]
    if case["median"]:
        ctx = [min(case["ctx_hi"], max(case["ctx_lo"], int(r.lognormvariate(math.log(case["median"]), 0.5))))
               for _ in range(n)]
    else:
        ctx = [r.randint(case["ctx_lo"], max(case["ctx_lo"], case["ctx_hi"])) for _ in range(n)]
    t = sorted(r.randint(case["t_lo"], max(case["t_lo"], case["t_hi"])) for _ in range(n))
    rows = list(range(n))
    r.shuffle(rows)
    return tuple(np.array(x, dtype=np.int64) for x in (rows, ctx, t))


def _max_seq(case) -> int:
    _, pos0, T = _blocks(case)
    return (int((pos0 + T).max()) + 63) // 64 * 64


def _trees(case):
    """Each block's parents (index within the block, -1 for the root; parents come before their children)."""
    r = random.Random(case["shape"] * 31 + 5)
    return [[-1] + [i - 1 if r.random() < 0.5 else r.randrange(i) for i in range(1, t)]
            for t in _blocks(case)[2].tolist()]


def _path(parents, node):
    p = [node]
    while parents[p[-1]] >= 0:
        p.append(parents[p[-1]])
    return p[::-1]


def _mask_words(case):
    """Ancestor bits, int32 [N, W]: bit j of token t's words says that t reads node j of its block."""
    trees = _trees(case)
    w = (max(len(p) for p in trees) + 31) // 32
    words = np.zeros((sum(len(p) for p in trees), w), dtype=np.uint32)
    t = 0
    for parents in trees:
        for i, a in enumerate(parents):
            if a >= 0:
                words[t + i] = words[t + a]
            words[t + i, i // 32] |= np.uint32(1 << (i % 32))
        t += len(parents)
    return words.view(np.int32)


def _tokens_of(case):
    """(rows, positions) of a case's tokens: a run of consecutive positions per cache row, its length odd or even as it
    falls."""
    r = random.Random(case["shape"])
    n, b = case["tokens"], case["requests"]
    lens = [n // b + (1 if i < n % b else 0) for i in range(b)]
    rows, pos = [], []
    for i, t in enumerate(lens):
        p0 = r.randrange(0, 200)
        rows += [i] * t
        pos += list(range(p0, p0 + t))
    return np.array(rows, dtype=np.int64), np.array(pos, dtype=np.int64)


def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + part) % (1 << 62))


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=gen)


def _gains(gen, *shape):
    """Sizes of channels: a few are several times the others, as a model's are."""
    return torch.empty(*shape, device=DEV).normal_(0.0, 0.4, generator=gen).exp_()


def _keys_values(seed, part, lead, hkv, s, d, dtype):
    """K and V [*lead, hkv, s, d]; K's channels differ in size."""
    g = _gen(seed, part)
    gain = _gains(g, hkv, 1, d).to(dtype)
    k = _normal(g, *lead, hkv, s, d, dtype=dtype)
    return k.mul_(gain), _normal(g, *lead, hkv, s, d, dtype=dtype)


def _angles(pos, d):
    """Rotation angles of positions, [n, d], in 64 bits: dim j and j + d / 2 turn by pos * THETA^(-2 j / d)."""
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=pos.device) / d)
    a = pos.double()[:, None] * inv
    return torch.cat([a, a], dim=1)


def _up(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


# ----------------------------------------------------------------------------- storage layouts
# 4-bit K: 64-position blocks of D / 32 fragments of 1 KiB; position 16 q + 4 a + r of a block, dims D / 4 * lg .. + D / 4
# - 1 are the D / 8 bytes of lane 16 lg + 4 q + r in fragment a (D = 128), or half (a % 2) of them in fragment a / 2 (D =
# 64); the lower half of a byte is the dim that comes first.  Its scales: [D / 32, 4 q + r, a] of a block.
# 4-bit V: D / 32 fragments of a block; positions 16 lg .. + 15 of dim 32 c + 16 h + l are half h of the 16 bytes of lane
# 16 lg + l in fragment c, the lower half of a byte the position that comes first.  Its scales: [D / 32, 64] of a block.
# bf16 K: 32-position blocks of 16 x 32 fragments, lane 16 lg + 4 q + r of fragment (a, j) holding position 8 q + 4 a + r
# and d = 32 j + 8 lg .. + 7.  bf16 and fp32 V: 32-position blocks, transposed.

def _nibbles(c):
    return c[..., ::2] | (c[..., 1::2] << 4)


def _codes(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)


def _k4_pack(c):
    """codes [.., s, d] -> [.., s / 64, d / 32, 64, 16] bytes"""
    *lead, s, d = c.shape
    n, h = len(lead), 128 // d
    x = _nibbles(c).reshape(*lead, s // 64, 4, 4 // h, h, 4, 4, 16 // h)      # blk, q, a / h, a % h, r, lg, byte
    x = x.permute(*range(n), *(n + i for i in (0, 2, 5, 1, 4, 3, 6)))         # blk, a / h, lg, q, r, a % h, byte
    return x.reshape(*lead, s // 64, d // 32, 64, 16).contiguous()


def _k4_unpack(b):
    *lead, nb, f, _, _ = b.shape
    n, h = len(lead), 4 // f
    x = b.reshape(*lead, nb, 4 // h, 4, 4, 4, h, 16 // h).permute(*range(n), *(n + i for i in (0, 3, 1, 5, 4, 2, 6)))
    return _codes(x.reshape(*lead, nb * 64, f * 16))


def _v4_pack(c):
    *lead, s, d = c.shape
    n = len(lead)
    x = _nibbles(c.transpose(-1, -2)).transpose(-1, -2)                       # [.., s / 2, d]
    x = x.reshape(*lead, s // 64, 4, 8, d // 32, 2, 16)                       # blk, lg, byte, c, h, l
    x = x.permute(*range(n), *(n + i for i in (0, 3, 1, 5, 4, 2)))            # blk, c, lg, l, h, byte
    return x.reshape(*lead, s // 64, d // 32, 64, 16).contiguous()


def _v4_unpack(b):
    *lead, nb, f, _, _ = b.shape
    n = len(lead)
    x = b.reshape(*lead, nb, f, 4, 16, 2, 8).permute(*range(n), *(n + i for i in (0, 2, 5, 1, 4, 3)))
    x = x.reshape(*lead, nb * 32, f * 32)
    return _codes(x.transpose(-1, -2)).transpose(-1, -2)


def _ks_pack(e):
    """biased exponents [.., s, d / 32] -> [.., s / 64, d / 32, 16, 4]"""
    *lead, s, f = e.shape
    n = len(lead)
    x = e.reshape(*lead, s // 64, 4, 4, 4, f).permute(*range(n), *(n + i for i in (0, 4, 1, 3, 2)))
    return x.reshape(*lead, s // 64, f, 16, 4).contiguous()


def _ks_unpack(e):
    *lead, nb, f, _, _ = e.shape
    n = len(lead)
    x = e.reshape(*lead, nb, f, 4, 4, 4).permute(*range(n), *(n + i for i in (0, 2, 4, 3, 1)))
    return x.reshape(*lead, nb * 64, f)


def _vs_pack(e):
    *lead, s, f = e.shape
    return e.reshape(*lead, s // 64, 64, f).transpose(-1, -2).contiguous()


def _vs_unpack(e):
    *lead, nb, f, _ = e.shape
    return e.transpose(-1, -2).reshape(*lead, nb * 64, f)


def _k_pack(k):
    *lead, s, d = k.shape
    n = len(lead)
    x = k.reshape(*lead, s // 32, 4, 2, 4, d // 32, 4, 8).permute(*range(n), *(n + i for i in (0, 2, 4, 5, 1, 3, 6)))
    return x.reshape(*lead, s // 32, d // 16, 64, 8).contiguous()


def _v_pack(v):
    *lead, s, d = v.shape
    return v.reshape(*lead, s // 32, 32, d).transpose(-1, -2).contiguous()


# ----------------------------------------------------------------------------- quantisation
# 4 bits: one scale 2^e per 32 dims, the smallest power of two >= 2^-125 with amax <= 7 * 2^e (6 is e2m1's largest value,
# and what lies between 6 and 7 is as near to it as the values above 4 are to theirs).  Held as the biased exponent e +
# 127.  Codes are x / 2^e rounded to e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), nearest even.
# 8-bit integers: a row's codes are x * r rounded to the nearest integer, ties to even, r = 127 / amax rounded to fp32;
# they stand for code * s, s = amax / 127 rounded to fp32.

def _quantise4(x):
    """x [.., d] -> (codes [.., d], biased exponents [.., d / 32])"""
    x = x.float().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)                                   # amax = m * 2^e, 0.5 <= m < 1; 7 = 0.875 * 2^3
    e = torch.where(m > 0.875, e - 2, e - 3).clamp(min=-125)
    e = torch.where(m > 0, e, torch.zeros_like(e))
    y = torch.ldexp(x, -e[..., None])
    # rounded up past a border; a tie goes to the even code, so every other border is the fp32 value below the tie
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    steps[1::2] = torch.nextafter(steps[1::2], torch.zeros_like(steps[1::2]))
    codes = torch.bucketize(y.abs(), steps, out_int32=True).to(torch.uint8)
    return (codes | (y < 0).to(torch.uint8) << 3).flatten(-2), (e + 127).to(torch.uint8)


def _values4(codes, exps):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    x = torch.cat([table, -table])[codes.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(x, exps[..., None].int() - 127).flatten(-2)


def _rows8(x):
    """x [n, k] -> (integer codes, as fp32, and scales [n, 1])"""
    amax = x.float().abs().amax(-1, keepdim=True)
    r = torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))
    return torch.round(x.double() * r.double()).float(), amax / 127.0


def _weight8(case, seed):
    """(codes int8 [n, k], scales fp32 [n]) of a projection of normal weights."""
    n, k, _ = LINEAR[case["weight"]]
    g = _gen(seed, 1)
    codes, scales = [], []
    for i in range(0, n, 4096):
        w = _normal(g, min(4096, n - i), k, dtype=torch.float32) / math.sqrt(k)
        c, s = _rows8(w)
        codes.append(c.to(torch.int8))
        scales.append(s[:, 0])
    return torch.cat(codes), torch.cat(scales)


# ----------------------------------------------------------------------------- states

def _linear_inputs(case, seed):
    """Activations, some channels of which are several times the others, and the residual."""
    n, k, epilogue = LINEAR[case["weight"]]
    g = _gen(seed, 2)
    x = _normal(g, case["tokens"], k, dtype=torch.float32).mul_(_gains(g, k)).to(_dtype(case))
    return x, _normal(g, case["tokens"], n, dtype=_dtype(case)) if epilogue == "residual" else None


def _norms_inputs(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    g = _gen(seed, 2)
    qkv = _normal(g, case["tokens"], (hq + 2 * hkv) * d, dtype=_dtype(case))
    return qkv, _gains(g, d).to(_dtype(case)), _gains(g, d).to(_dtype(case))


@torch.inference_mode()
def prepare(case: dict, seed: int):
    kind = case["kind"]
    if kind == "linear8":
        w, ws = _weight8(case, seed)
        x, r = _linear_inputs(case, seed)
        st = {"kind": kind, "epilogue": LINEAR[case["weight"]][2], "x": x, "residual": r}
        if own:  # a model's weights, laid out as they are loaded
            from thesis_amd import _lsk

            return {**st, "w": _lsk.PackedWeightI8(w, ws)}
        return {**st, "w": w, "ws": ws}
    hq, hkv, d = HEADS[case["heads"]]
    byte = dict(dtype=torch.uint8, device=DEV)
    if kind in ("cache4", "norms"):
        rows, pos = _tokens_of(case)
        s, b = (int(pos.max()) + 64) // 64 * 64, case["requests"]
        st = {"kind": kind, "heads": (hq, hkv, d), "rows": _up(rows, torch.int32), "pos": _up(pos, torch.int32)}
    if kind == "cache4":
        k, v = _keys_values(seed, 1, (), hkv, len(rows), d, _dtype(case))
        zeros = lambda *shape: torch.zeros(b, hkv, s // 64, d // 32, *shape, **byte)  # noqa: E731
        return {**st, "x_k": k.transpose(0, 1).contiguous(), "x_v": v.transpose(0, 1).contiguous(),
                "k": zeros(64, 16), "v": zeros(64, 16), "ks": zeros(16, 4) + 127, "vs": zeros(64) + 127}
    if kind == "norms":
        qkv, wq, wk = _norms_inputs(case, seed)
        a = _angles(torch.arange(s, device=DEV), d)
        k = torch.zeros(b, hkv, s, d, dtype=_dtype(case), device=DEV)
        return {**st, "qkv": qkv, "wq": wq, "wk": wk, "cos": a.cos().float(), "sin": a.sin().float(),
                "k": _k_pack(k) if case["dtype"] == "bf16" else k, "v": _v_pack(torch.zeros_like(k))}
    rows, pos0, T = _blocks(case)
    b, s = case["requests"], _max_seq(case)
    starts = np.concatenate([[0], np.cumsum(T)[:-1]])
    st = {"kind": kind, "heads": (hq, hkv, d), "rows": _up(rows, torch.int32), "pos0": _up(pos0, torch.int32),
          "lens": _up(T, torch.int32), "starts": _up(starts, torch.int32), "t_max": int(T.max()), "n": int(T.sum()),
          "end": s}
    k, v = _keys_values(seed, 1, (b,), hkv, s, d, torch.bfloat16)
    kc, ke = _quantise4(k)
    st["k"], st["ks"] = _k4_pack(kc), _ks_pack(ke)
    del k, kc
    vc, ve = _quantise4(v)
    st["v"], st["vs"] = _v4_pack(vc), _vs_pack(ve)
    del v, vc
    st["q"] = _normal(_gen(seed, 2), st["n"], hq, d)
    st["mask"] = _up(_mask_words(case)) if kind == "tree4" else None
    if own:  # the plan of a packed segment, which its layers share
        from thesis_amd import _lsk

        blocks = np.stack([np.cumsum(T) - T, pos0, T, rows], axis=1).astype(np.int32)
        cache = _lsk.KV4(st["k"], st["v"], st["ks"], st["vs"])
        st["plan"] = _lsk.AttnPlan(blocks, hq, cache, tree=kind == "tree4")
    return st


# ----------------------------------------------------------------------------- one pass

@torch.inference_mode()
def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["kind"] == "cache4":
        return _plain_cache(s)
    if s["kind"] == "norms":
        return _plain_norms(s)
    if s["kind"] == "linear8":
        return _plain_linear(s)
    return _plain_attention(s)


def _run_own(s):
    from thesis_amd import _lsk

    if s["kind"] == "linear8":
        epilogue = {"none": _lsk.EPI_NONE, "residual": _lsk.EPI_RESIDUAL, "silu": _lsk.EPI_SILU_MUL}[s["epilogue"]]
        return {"out": _lsk.gemm_i8(_lsk.quant_rows_i8(s["x"]), s["w"], residual=s["residual"], epilogue=epilogue)}
    if s["kind"] == "norms":
        hq, hkv, d = s["heads"]
        q = s["qkv"].new_empty(s["qkv"].shape[0], hq, d)
        _lsk.qk_norm_rope_append(s["qkv"], q, s["k"], s["v"], s["wq"], s["wk"], EPS, s["cos"], s["sin"], s["rows"],
                                 s["pos"], hq, hkv, d)
        return {"q": q, "k": s["k"], "v": s["v"]}
    cache = _lsk.KV4(s["k"], s["v"], s["ks"], s["vs"])
    if s["kind"] == "cache4":
        _lsk.kv4_append(s["x_k"], s["x_v"], cache, s["rows"], s["pos"])
        k, v = _lsk.kv4_read(cache, s["rows"], s["pos"], s["x_k"].dtype)
        return {"k": k, "v": v}
    return {"out": _lsk.kv4_attn(s["q"], cache, s["plan"], s["mask"])}


def _plain_cache(s):
    rows, pos = s["rows"].long(), s["pos"].long()
    kc, ke = _quantise4(s["x_k"])
    vc, ve = _quantise4(s["x_v"])
    n, hkv, d = kc.shape
    h = 128 // d
    blk, q, a, r, p = pos // 64, pos % 64 // 16, pos % 16 // 4, pos % 4, pos % 64
    k4 = s["k"].view(-1, hkv, s["k"].shape[2], 4 // h, 4, 4, 4, h, 16 // h)      # [B, H, blk, a / h, lg, q, r, a % h, 16 / h]
    k4[rows, :, blk, a // h, :, q, r, a % h] = _nibbles(kc).view(n, hkv, 4, 16 // h)
    ks = s["ks"]
    ks[rows, :, blk, :, 4 * q + r, a] = ke
    v4 = _codes(s["v"].view(*s["v"].shape[:4], 4, 16, 2, 8))                     # [B, H, blk, c, lg, l, h, 16]
    v4[rows, :, blk, :, p // 16, :, :, p % 16] = vc.view(n, hkv, d // 32, 2, 16).transpose(-1, -2)
    s["v"].copy_(_nibbles(v4).view(s["v"].shape))
    s["vs"][rows, :, blk, :, p] = ve
    kb = k4[rows, :, blk, a // h, :, q, r, a % h].reshape(n, hkv, d // 2)
    vb = _codes(s["v"].view(*s["v"].shape[:4], 4, 16, 2, 8))[rows, :, blk, :, p // 16, :, :, p % 16]
    vb = vb.transpose(-1, -2).reshape(n, hkv, d)
    return {"k": _values4(_codes(kb), ks[rows, :, blk, :, 4 * q + r, a]).to(s["x_k"].dtype),
            "v": _values4(vb, s["vs"][rows, :, blk, :, p]).to(s["x_v"].dtype)}


def _plain_norms(s):
    hq, hkv, d = s["heads"]
    rows, pos = s["rows"].long(), s["pos"].long()
    n, half = rows.numel(), d // 2
    x = s["qkv"].float().view(n, hq + 2 * hkv, d)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(h, w):
        h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w.float()
        return h * cos + torch.cat([-h[..., half:], h[..., :half]], dim=-1) * sin

    q = turned(x[:, :hq], s["wq"]).to(s["qkv"].dtype)
    k = turned(x[:, hq:hq + hkv], s["wk"]).to(s["qkv"].dtype)
    v = s["qkv"].view(n, hq + 2 * hkv, d)[:, hq + hkv:]
    if s["k"].dim() == 6:
        kc = s["k"].view(*s["k"].shape[:3], 2, d // 32, 4, 4, 4, 8)              # [B, H, blk, a, j, lg, q, r, 8]
        kc[rows, :, pos // 32, pos % 8 // 4, :, :, pos % 32 // 8, pos % 4] = k.view(n, hkv, d // 32, 4, 8)
    else:
        s["k"][rows, :, pos] = k
    s["v"][rows, :, pos // 32, :, pos % 32] = v
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_linear(s):
    c, sx = _rows8(s["x"])
    y = (c @ s["w"].float().t()) * sx * s["ws"]
    if s["epilogue"] == "silu":
        g, u = y.chunk(2, dim=-1)
        y = g / (1.0 + torch.exp(-g)) * u
    elif s["epilogue"] == "residual":
        y = y + s["residual"].float()
    return {"out": y.to(s["x"].dtype)}


def _plain_attention(s):
    hq, hkv, d = s["heads"]
    rows, pos0, t = s["rows"].long(), s["pos0"].long(), s["t_max"]
    end, b = s["end"], s["rows"].numel()
    # K and V of the blocks' cache rows, [b, hkv, end, d]
    k = _values4(_k4_unpack(s["k"][rows]), _ks_unpack(s["ks"][rows]))
    v = _values4(_v4_unpack(s["v"][rows]), _vs_unpack(s["vs"][rows]))
    # queries padded to [b, t]
    step = torch.arange(t, device=DEV)
    at = (s["starts"].long()[:, None] + step).clamp(max=s["n"] - 1)
    q = s["q"][at].float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    slot = torch.arange(end, device=DEV)[None, None] - pos0[:, None, None]          # position within the block
    allowed = (slot <= step[:, None]).expand(b, t, end)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        bits = bits.flatten(1).bool()[at]                                           # [b, t, 32 W]
        node = slot.clamp(0, bits.shape[2] - 1).expand(b, t, end)
        allowed = allowed & ((slot < 0) | bits.gather(2, node))
    scores = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(b, hkv, t, hq // hkv, end)
    scores.masked_fill_(~allowed[:, None, :, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    out = (p.view(b, hkv, -1, end) @ v).view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b * t, hq * d)
    lens = s["lens"].long()
    blk = torch.repeat_interleave(torch.arange(b, device=DEV), lens, output_size=s["n"])
    row = torch.arange(s["n"], device=DEV) - s["starts"].long()[blk] + blk * t
    return {"out": out[row].to(s["q"].dtype)}


# ----------------------------------------------------------------------------- work

def work(case: dict) -> dict:
    es = _dtype(case).itemsize
    if case["kind"] == "linear8":
        n, k, epilogue = LINEAR[case["weight"]]
        m = case["tokens"]
        outs = {"none": n, "residual": 2 * n, "silu": n // 2}[epilogue]
        return {"bytes": n * k + 4 * n + m * (k + outs) * es, "flops": 2 * m * n * k}
    hq, hkv, d = HEADS[case["heads"]]
    held = d // 2 + d // 32                                     # bytes of one position's K or V of one KV head
    if case["kind"] == "cache4":
        n = case["tokens"] * hkv
        return {"bytes": 4 * n * (d * es + held), "flops": 4 * n * d}
    if case["kind"] == "norms":
        n = case["tokens"]
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * es + 2 * n * d * 4, "flops": 8 * n * (hq + hkv) * d}
    rows, pos0, T = _blocks(case)
    pairs = int((T * pos0).sum())
    if case["kind"] == "attn4":
        pairs += int((T * (T + 1) // 2).sum())
    else:
        pairs += sum(len(_path(p, i)) for p in _trees(case) for i in range(len(p)))
    return {"bytes": int((pos0 + T).sum()) * hkv * 2 * held + 2 * int(T.sum()) * hq * d * es,
            "flops": 4 * hq * d * pairs}


# ----------------------------------------------------------------------------- the same in 64 bits

def _held4(x):
    """What the 4-bit cache holds for vectors x [.., d]."""
    x = x.double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(torch.where(amax > 0, amax, 7.0) / 7.0)  # the smallest power of two >= this
    scale = torch.exp2((e - (m == 0.5).int()).double().clamp(min=-125.0))
    y = x / scale
    unit = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return ((torch.round(y / unit) * unit).clamp(-6.0, 6.0) * scale).flatten(-2)


def _exact_linear(case, seed):
    n, k, epilogue = LINEAR[case["weight"]]
    w, ws = _weight8(case, seed)
    x, res = _linear_inputs(case, seed)
    amax = x.double().abs().amax(1)
    to = (127.0 / amax).float().double()                        # the format's own two roundings
    back = (amax / 127.0).float().double()
    codes = torch.round(x.double() * to[:, None])
    y = torch.empty(case["tokens"], n, dtype=torch.float64, device=DEV)
    for i in range(0, n, 4096):
        y[:, i:i + 4096] = codes @ w[i:i + 4096].double().T
    y *= back[:, None]
    y *= ws.double()
    if epilogue == "silu":
        y = torch.nn.functional.silu(y[:, :n // 2]) * y[:, n // 2:]
    return {"out": y + res.double() if res is not None else y}


def _exact_norms(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    rows, pos = _tokens_of(case)
    qkv, wq, wk = _norms_inputs(case, seed)
    x = qkv.double().view(-1, hq + 2 * hkv, d)
    a = _angles(torch.arange(int(pos.max()) + 1, device=DEV), d)[:, :d // 2]
    rot = torch.polar(torch.ones_like(a), a)
    # the tables are given in fp32
    rot = torch.complex(rot.real.float().double(), rot.imag.float().double())[_up(pos)][:, None]

    def turned(h, w):
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(h[..., :d // 2].contiguous(), h[..., d // 2:].contiguous()) * rot
        return torch.cat([z.real, z.imag], dim=-1)

    s = (int(pos.max()) + 64) // 64 * 64
    k = torch.zeros(case["requests"], hkv, s, d, dtype=torch.float64, device=DEV)
    v = torch.zeros_like(k)
    at = (_up(rows), slice(None), _up(pos))
    k[at] = turned(x[:, hq:hq + hkv], wk)
    v[at] = x[:, hq + hkv:]
    return {"q": turned(x[:, :hq], wq), "k": _k_pack(k) if case["dtype"] == "bf16" else k, "v": _v_pack(v)}


@torch.inference_mode()
def exact(case: dict, seed: int):
    if case["kind"] == "linear8":
        return _exact_linear(case, seed)
    if case["kind"] == "norms":
        return _exact_norms(case, seed)
    hq, hkv, d = HEADS[case["heads"]]
    if case["kind"] == "cache4":
        k, v = _keys_values(seed, 1, (), hkv, case["tokens"], d, _dtype(case))
        return {"k": _held4(k.transpose(0, 1)), "v": _held4(v.transpose(0, 1))}
    rows, pos0, T = _blocks(case)
    kc, vc = _keys_values(seed, 1, (case["requests"],), hkv, _max_seq(case), d, torch.bfloat16)
    q = _normal(_gen(seed, 2), int(T.sum()), hq, d).double()
    trees = _trees(case) if case["kind"] == "tree4" else None
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    a = 0
    for j, (r, p, t) in enumerate(zip(rows.tolist(), pos0.tolist(), T.tolist())):
        k, v = _held4(kc[r, :, :p + t]), _held4(vc[r, :, :p + t])
        reads = torch.ones(t, p + t, dtype=torch.bool)
        if trees is None:
            reads = reads.tril(p)
        else:
            reads[:, p:] = False
            for i in range(t):
                reads[i, [p + x for x in _path(trees[j], i)]] = True
        reads = reads.to(DEV)
        for h in range(hkv):
            g = hq // hkv
            s = (q[a:a + t, h * g:(h + 1) * g].reshape(t * g, d) @ k[h].T).view(t, g, -1) / math.sqrt(d)
            w = torch.softmax(s.masked_fill(~reads[:, None], -math.inf), dim=-1)
            out[a:a + t, h * g:(h + 1) * g] = (w.view(t * g, -1) @ v[h]).view(t, g, d)
        a += t
    return {"out": out.reshape(len(out), -1)}
