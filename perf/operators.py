"""Operators over the KV cache: the 8-bit cache as it is written, read back and attended to, and trees of drafted tokens
from their verification to the accepted path.

Five kinds of call, at the head shapes of the package's presets:

  cache8   K and V of some tokens are quantised into an 8-bit cache (e4m3 codes, one power-of-two scale per token and
           KV head) and read back.  Returns the K and V that the cache stands for.
  attn8    ragged verify / decode attention over an 8-bit cache: a query at position p reads positions 0 .. p.
  tree8    the same for trees of drafted tokens: a node reads the prefix, its ancestors and itself.
  tree     trees over the bf16 or fp32 cache.
  accept   greedy acceptance of verified trees, and the accepted paths' K / V moved to consecutive positions in every
           layer.  Returns the counts, paths and committed tokens and the caches.

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


# ----------------------------------------------------------------------------- the cases

def _attend_case(name, kind, heads, requests, t, ctx, median=0, dtype="bf16", shape=1):
    """requests blocks of t[0]..t[1] tokens (tree nodes) at contexts ctx[0]..ctx[1]: uniform, or with median > 0
    lognormal around it."""
    c = {"kind": kind, "heads": heads, "requests": requests, "t_lo": t[0], "t_hi": t[1], "ctx_lo": ctx[0],
         "ctx_hi": ctx[1], "median": median, "dtype": dtype, "shape": shape}
    return {"name": name, **c} if name else c


def _cache_case(name, heads, tokens, requests, shape=1):
    """tokens new tokens over requests cache rows (a run of consecutive positions in each)."""
    c = {"kind": "cache8", "heads": heads, "tokens": tokens, "requests": requests, "shape": shape}
    return {"name": name, **c} if name else c


def _accept_case(name, heads, layers, requests, t, ctx, dtype="bf16", shape=1):
    c = {"kind": "accept", "heads": heads, "layers": layers, "requests": requests, "t_lo": t[0], "t_hi": t[1],
         "ctx_lo": ctx[0], "ctx_hi": ctx[1], "median": 0, "dtype": dtype, "shape": shape}
    return {"name": name, **c} if name else c


def listed() -> list:
    return [
        # a decode step of 32 requests writes one token each
        _cache_case("cache8_8b_32", "8b", 32, 32),
        # a long prompt of odd length goes into the cache in one call
        _cache_case("cache8_8b_4001", "8b", 4001, 1),
        # single-stream decoding: one query token, the smallest attention call
        _attend_case("attn8_1b_b1", "attn8", "1b", 1, (1, 1), (300, 400)),
        # one request with a very long context (the 1B shape's positions go to 131072), verifying a few drafts
        _attend_case("attn8_1b_long", "attn8", "1b", 1, (5, 5), (100001, 100001)),
        # a server's decode batch: 32 requests, prompts up to 1024 and 256 new tokens
        _attend_case("attn8_8b_b32", "attn8", "8b", 32, (1, 1), (128, 1280)),
        # verification in a large batch: contexts of median 1500 up to 8183, 1 to 9 tokens each
        _attend_case("attn8_8b_b256", "attn8", "8b", 256, (1, 9), (64, 8183), median=1500),
        # trees of 20 to 40 nodes over an 8-bit cache of an MHA model
        _attend_case("tree8_7b_b16", "tree8", "7b", 16, (20, 40), (256, 1100)),
        # a single stream's tree of 13 nodes
        _attend_case("tree_1b_b1", "tree", "1b", 1, (13, 13), (300, 400)),
        # a batch of trees of up to 64 nodes
        _attend_case("tree_8b_b32", "tree", "8b", 32, (25, 64), (128, 1280)),
        # the fp32 model (the token-identity configuration) with small trees
        _attend_case("tree_1b_fp32_b4", "tree", "1b", 4, (5, 12), (16, 192), dtype="fp32"),
        # a single stream's tree is accepted: 16 layers of the 1B shape
        _accept_case("accept_1b_b1", "1b", 16, 1, (13, 13), (300, 400)),
        # a batch's trees are accepted: 32 layers of the 8B shape
        _accept_case("accept_8b_b32", "8b", 32, 32, (25, 64), (128, 440)),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["cache8", "attn8", "attn8", "tree8", "tree", "tree", "accept"])
    heads = rng.choice(sorted(HEADS))
    shape = rng.randrange(1, 1 << 20)
    hkv = HEADS[heads][1]
    if kind == "cache8":
        tokens = _log(rng, 1, 4001 if hkv == 8 else 1000)
        return _cache_case(None, heads, tokens, _log(rng, 1, min(tokens, 64)), shape=shape)
    if kind == "accept":
        fp32 = rng.random() < 0.25
        return _accept_case(None, heads, rng.randint(1, 32 if hkv == 8 else 8), _log(rng, 1, 16 if fp32 else 32),
                            (rng.randint(1, 12), rng.randint(12, 64)), (rng.randint(1, 64), _log(rng, 65, 440)),
                            dtype="fp32" if fp32 else "bf16", shape=shape)
    if kind == "attn8":
        if rng.random() < 0.25:                                  # few requests, a long context
            hi = _log(rng, 4000, 100000 if heads == "1b" else 8000)
            return _attend_case(None, kind, heads, rng.randint(1, 2), (1, rng.randint(1, 9)), (hi // 2, hi),
                                shape=shape)
        requests = _log(rng, 1, 256 if hkv == 8 else 48)
        return _attend_case(None, kind, heads, requests, (1, rng.randint(1, 9)),
                            (rng.randint(1, 64), _log(rng, 65, 2800)), shape=shape)
    fp32 = kind == "tree" and rng.random() < 0.3
    requests = _log(rng, 1, 4 if fp32 else 32 if hkv == 8 else 8)
    return _attend_case(None, kind, heads, requests, (rng.randint(1, 12), rng.randint(12, 24 if fp32 else 64)),
                        (rng.randint(1, 64), _log(rng, 65, 200 if fp32 else 1280)), dtype="fp32" if fp32 else "bf16",
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
    """Each block's parents (index within the block, -1 for the root; parents come before their children) and the
    node whose path is accepted."""
    r = random.Random(case["shape"] * 31 + 5)
    out = []
    for t in _blocks(case)[2].tolist():
        parents = [-1] + [i - 1 if r.random() < 0.5 else r.randrange(i) for i in range(1, t)]
        out.append((parents, r.randrange(t)))
    return out


def _path(parents, node):
    p = [node]
    while parents[p[-1]] >= 0:
        p.append(parents[p[-1]])
    return p[::-1]


def _mask_words(case):
    """Ancestor bits, int32 [N, W]: bit j of token t's words says that t reads node j of its block."""
    trees = [p for p, _ in _trees(case)]
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
    """(rows, positions) of a cache8 case's tokens: a run of consecutive positions per cache row, its length odd or
    even as it falls."""
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


def _keys_values(seed, part, lead, hkv, s, d, dtype):
    """K and V [*lead, hkv, s, d]; K's channels differ in size (a few are several times the others), as a model's do."""
    g = _gen(seed, part)
    gain = torch.empty(hkv, 1, d, device=DEV).normal_(0.0, 0.4, generator=g).exp_().to(dtype)
    k = _normal(g, *lead, hkv, s, d, dtype=dtype)
    return k.mul_(gain), _normal(g, *lead, hkv, s, d, dtype=dtype)


def _up(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


# ----------------------------------------------------------------------------- storage layouts
# bf16 K: 32-position blocks of 16 x 32 fragments, lane 16 lg + 4 q + r of fragment (a, j) holding position
# 8 q + 4 a + r and d = 32 j + 8 lg .. + 7.  8-bit K: 64-position blocks of 16 x 64 fragments, lane 16 lg + 4 q + r of
# (a, j) holding position 16 q + 4 a + r and d = 64 j + 16 lg .. + 15.  V: 32- (64-) position blocks, transposed.

def _k_pack(k):
    *lead, s, d = k.shape
    n = len(lead)
    x = k.reshape(*lead, s // 32, 4, 2, 4, d // 32, 4, 8).permute(*range(n), *(n + i for i in (0, 2, 4, 5, 1, 3, 6)))
    return x.reshape(*lead, s // 32, d // 16, 64, 8).contiguous()


def _k_unpack(kf):
    *lead, nb, nf, _, _ = kf.shape
    n = len(lead)
    x = kf.reshape(*lead, nb, 2, nf // 2, 4, 4, 4, 8).permute(*range(n), *(n + i for i in (0, 4, 1, 5, 2, 3, 6)))
    return x.reshape(*lead, nb * 32, nf * 16)


def _v_pack(v, block=32):
    *lead, s, d = v.shape
    return v.reshape(*lead, s // block, block, d).transpose(-1, -2).contiguous()


def _v_unpack(vb):
    *lead, nb, d, block = vb.shape
    return vb.transpose(-1, -2).reshape(*lead, nb * block, d)


def _k8_pack(k):
    *lead, s, d = k.shape
    n = len(lead)
    x = k.reshape(*lead, s // 64, 4, 4, 4, d // 64, 4, 16).permute(*range(n), *(n + i for i in (0, 2, 4, 5, 1, 3, 6)))
    return x.reshape(*lead, s // 64, 4, d // 64, 64, 16).contiguous()


def _k8_unpack(kf):
    *lead, nb, _, j, _, _ = kf.shape
    n = len(lead)
    x = kf.reshape(*lead, nb, 4, j, 4, 4, 4, 16).permute(*range(n), *(n + i for i in (0, 4, 1, 5, 2, 3, 6)))
    return x.reshape(*lead, nb * 64, j * 64)


# ----------------------------------------------------------------------------- quantisation
# One scale 2^e per token and head: the smallest power of two with amax <= 448 * 2^e (448: e4m3's largest value), and
# e >= -117, so that every value is a normal bf16 number.  Held as the biased exponent e + 127 in 8 bits.  Codes are x / 2^e rounded to e4m3, nearest even.

def _quantise(x):
    """x [.., d] -> (codes as bytes [.., d], biased exponents [..])."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))                       # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(m > 0, e, torch.zeros_like(e)).clamp(-117, 127)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, exps):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), exps[..., None].int() - 127)


# ----------------------------------------------------------------------------- states

def _cache_state(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    rows, pos0, T = _blocks(case)
    b, s = case["requests"], _max_seq(case)
    if case["kind"] in ("attn8", "tree8"):
        k, v = _keys_values(seed, 1, (b,), hkv, s, d, torch.bfloat16)
        kc, ks = _quantise(k)
        del k
        vc, vs = _quantise(v)
        del v
        return {"k": _k8_pack(kc).view(torch.float8_e4m3fn), "v": _v_pack(vc, 64).view(torch.float8_e4m3fn),
                "ks": ks, "vs": vs}
    k, v = _keys_values(seed, 1, (b,), hkv, s, d, _dtype(case))
    return {"k": _k_pack(k) if case["dtype"] == "bf16" else k, "v": _v_pack(v)}


def _block_state(case):
    rows, pos0, T = _blocks(case)
    starts = np.concatenate([[0], np.cumsum(T)[:-1]])
    return {"rows": _up(rows, torch.int32), "pos0": _up(pos0, torch.int32), "lens": _up(T, torch.int32),
            "starts": _up(starts, torch.int32), "t_max": int(T.max()), "n": int(T.sum()),
            "end": (int((pos0 + T).max()) + 63) // 64 * 64}


@torch.inference_mode()
def prepare(case: dict, seed: int):
    hq, hkv, d = HEADS[case["heads"]]
    kind = case["kind"]
    if kind == "cache8":
        rows, pos = _tokens_of(case)
        s = (int(pos.max()) + 64) // 64 * 64
        k, v = _keys_values(seed, 1, (), hkv, len(rows), d, torch.bfloat16)
        b = case["requests"]
        byte = dict(dtype=torch.uint8, device=DEV)
        return {"kind": kind, "x_k": k.transpose(0, 1).contiguous(), "x_v": v.transpose(0, 1).contiguous(),
                "rows": _up(rows, torch.int32), "pos": _up(pos, torch.int32),
                "k": torch.zeros(b, hkv, s // 64, 4, d // 64, 64, 16, **byte).view(torch.float8_e4m3fn),
                "v": torch.zeros(b, hkv, s // 64, d, 64, **byte).view(torch.float8_e4m3fn),
                "ks": torch.full((b, hkv, s), 127, **byte), "vs": torch.full((b, hkv, s), 127, **byte)}
    st = {"kind": kind, "heads": (hq, hkv, d), **_block_state(case)}
    if kind == "accept":
        k, v = _accept_caches(case, seed)
        tokens, y = _accept_tokens(case, seed)
        trees = _trees(case)
        parents = np.concatenate([np.array(p) for p, _ in trees])
        return {**st, "k": k, "v": v, "tokens": _up(tokens), "y": _up(y), "parents": _up(parents, torch.int32),
                "mask": _up(_mask_words(case))}
    st.update(_cache_state(case, seed), q=_normal(_gen(seed, 2), st["n"], hq, d, dtype=_dtype(case)))
    st["mask"] = _up(_mask_words(case)) if kind in ("tree", "tree8") else None
    if own:  # the plan of a packed segment, which its layers share
        from thesis_amd import _lsk

        rows, pos0, T = _blocks(case)
        blocks = np.stack([np.cumsum(T) - T, pos0, T, rows], axis=1).astype(np.int32)
        cache = _lsk.KV8(st["k"], st["v"], st["ks"], st["vs"]) if kind != "tree" else st["k"]
        st["plan"] = _lsk.AttnPlan(blocks, hq, cache)
    return st


def _accept_caches(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    k, v = _keys_values(seed, 1, (case["layers"], case["requests"]), hkv, _max_seq(case), d, _dtype(case))
    return (_k_pack(k) if case["dtype"] == "bf16" else k), _v_pack(v)


def _accept_tokens(case, seed):
    """Drafted tokens and the verifier's greedy tokens: the accepted node's path matches and nothing after it does;
    siblings now and then carry the same token."""
    r = np.random.default_rng([int(seed) % (1 << 31), case["shape"]])
    tokens, y = [], []
    for parents, node in _trees(case):
        t = r.integers(0, 1000, len(parents))
        g = r.integers(1000, 2000, len(parents))
        path = _path(parents, node)
        for a, b in zip(path, path[1:]):
            g[a] = t[b]
            for c in range(1, b):                                # the first sibling with the token is the accepted one
                if parents[c] == a and t[c] == t[b]:
                    t[c] += 2000
        tokens.append(t)
        y.append(g)
    return np.concatenate(tokens), np.concatenate(y)


# ----------------------------------------------------------------------------- one pass

@torch.inference_mode()
def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["kind"] == "cache8":
        return _plain_cache(s)
    if s["kind"] == "accept":
        return _plain_accept(s)
    return _plain_attention(s)


def _run_own(s):
    from thesis_amd import _lsk

    if s["kind"] == "cache8":
        cache = _lsk.KV8(s["k"], s["v"], s["ks"], s["vs"])
        _lsk.kv8_append(s["x_k"], s["x_v"], cache, s["rows"], s["pos"])
        k, v = _lsk.kv8_read(cache, s["rows"], s["pos"])
        return {"k": k, "v": v}
    if s["kind"] == "accept":
        acc, path, out = _lsk.tree_accept(s["y"], s["tokens"], s["parents"], s["starts"], s["lens"], s["t_max"])
        _lsk.kv_compact(s["k"], s["v"], s["rows"], s["pos0"], acc, path)
        return {"accepted": acc, "path": path, "tokens": out, "k": s["k"], "v": s["v"]}
    if s["kind"] == "tree":
        return {"out": _lsk.tree_attn(s["q"], s["k"], s["v"], s["plan"], s["mask"])}
    cache = _lsk.KV8(s["k"], s["v"], s["ks"], s["vs"])
    return {"out": _lsk.kv8_attn(s["q"], cache, s["plan"], s["mask"])}


def _plain_cache(s):
    rows, pos = s["rows"].long(), s["pos"].long()
    kc, ke = _quantise(s["x_k"])
    vc, ve = _quantise(s["x_v"])
    n, hkv, d = kc.shape
    blk, q, a, r = pos // 64, pos % 64 // 16, pos % 16 // 4, pos % 4
    k8 = s["k"].view(torch.uint8).unflatten(5, (4, 4, 4))       # [B, H, blk, a, j, lg, q, r, 16]
    v8 = s["v"].view(torch.uint8)
    k8[rows, :, blk, a, :, :, q, r] = kc.view(n, hkv, d // 64, 4, 16)
    v8[rows, :, blk, :, pos % 64] = vc
    s["ks"][rows, :, pos] = ke
    s["vs"][rows, :, pos] = ve
    return {"k": _values(k8[rows, :, blk, a, :, :, q, r].reshape(n, hkv, d), s["ks"][rows, :, pos]).bfloat16(),
            "v": _values(v8[rows, :, blk, :, pos % 64], s["vs"][rows, :, pos]).bfloat16()}


def _plain_attention(s):
    hq, hkv, d = s["heads"]
    rows, pos0, t = s["rows"].long(), s["pos0"].long(), s["t_max"]
    end, b = s["end"], s["rows"].numel()
    # K and V of the blocks' cache rows, [b, hkv, end, d]
    if s["kind"] == "tree":
        k = s["k"][rows, :, :end // 32] if s["k"].dim() == 6 else s["k"][rows, :, :end]
        k = (_k_unpack(k) if s["k"].dim() == 6 else k).float()
        v = _v_unpack(s["v"][rows, :, :end // 32]).float()
    else:
        k8 = _k8_unpack(s["k"].view(torch.uint8)[rows, :, :end // 64])
        v8 = _v_unpack(s["v"].view(torch.uint8)[rows, :, :end // 64])
        k = _values(k8, s["ks"][rows, :, :end])
        v = _values(v8, s["vs"][rows, :, :end])
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


def _plain_accept(s):
    b, t = s["lens"].numel(), s["t_max"]
    lens, starts = s["lens"].long(), s["starts"].long()
    step = torch.arange(t, device=DEV)
    real = step < lens[:, None]
    at = (starts[:, None] + step).clamp(max=s["n"] - 1)
    tok, y, parent = s["tokens"][at], s["y"][at], s["parents"][at].long()
    same = (parent[:, :, None] == parent[:, None]) & (tok[:, :, None] == tok[:, None]) & (step[None] < step[:, None])
    good = (y.gather(1, parent.clamp(min=0)) == tok) & ~(same & real[:, None]).any(-1) | (parent < 0)
    bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    bits = bits.flatten(1).bool()[at][:, :, :t]
    taken = ~(bits & ~good[:, None]).any(-1) & real                                 # every ancestor matches
    acc = taken.sum(-1) - 1
    path = torch.where(taken, step, t).sort(-1).values
    on = step <= acc[:, None]
    path = torch.where(on, path, -1)
    out = torch.where(on, y.gather(1, path.clamp(min=0)), -1)
    # node path[j]'s slot moves to slot j; the others move onto themselves
    rows = s["rows"].long()[:, None].expand(b, t)[real]
    dst = (s["pos0"].long()[:, None] + step)[real]
    src = (s["pos0"].long()[:, None] + torch.where(on, path, step))[real]
    k, v = s["k"], s["v"]
    if k.dim() == 7:
        k = k.unflatten(4, (2, -1)).unflatten(6, (4, 4, 4))     # [L, B, H, blk, a, j, lg, q, r, 8]
        take = lambda p: (slice(None), rows, slice(None), p // 32, p % 8 // 4, slice(None), slice(None),  # noqa: E731
                          p % 32 // 8, p % 4)
        k[take(dst)] = k[take(src)]
    else:
        k[:, rows, :, dst] = k[:, rows, :, src]
    v[:, rows, :, dst // 32, :, dst % 32] = v[:, rows, :, src // 32, :, src % 32]
    return {"accepted": acc, "path": path.int(), "tokens": out, "k": s["k"], "v": s["v"]}


# ----------------------------------------------------------------------------- work

def work(case: dict) -> dict:
    hq, hkv, d = HEADS[case["heads"]]
    if case["kind"] == "cache8":
        n = case["tokens"] * hkv
        return {"bytes": 2 * n * (2 * d + d + 1) + 2 * n * (d + 1 + 2 * d), "flops": 4 * n * d}
    rows, pos0, T = _blocks(case)
    es = _dtype(case).itemsize
    if case["kind"] == "accept":
        moved = sum(sum(j != i for j, i in enumerate(_path(p, node))) for p, node in _trees(case))
        return {"bytes": moved * case["layers"] * hkv * 2 * d * es * 2 + int(T.sum()) * 20, "flops": int(T.sum())}
    kv = 2 * d + 2 if case["kind"] != "tree" else 2 * d * es    # bytes of one position of one KV head
    pairs = int((T * pos0).sum())
    if case["kind"] == "attn8":
        pairs += int((T * (T + 1) // 2).sum())
    else:
        pairs += sum(len(_path(p, i)) for p, _ in _trees(case) for i in range(len(p)))
    return {"bytes": int((pos0 + T).sum()) * hkv * kv + 2 * int(T.sum()) * hq * d * es, "flops": 4 * hq * d * pairs}


# ----------------------------------------------------------------------------- the same in 64 bits

def _e4m3(x):
    """x rounded to the nearest e4m3 value, ties to even; 64 bits, |x| <= 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    unit = torch.exp2(e - 3.0)
    return torch.round(x / unit) * unit


def _held(x):
    """What the 8-bit cache holds for vectors x [.., d]."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 448.0) / 448.0)).clamp(min=-117.0)
    return _e4m3(x / torch.exp2(e)) * torch.exp2(e)


@torch.inference_mode()
def exact(case: dict, seed: int):
    hq, hkv, d = HEADS[case["heads"]]
    if case["kind"] == "cache8":
        k, v = _keys_values(seed, 1, (), hkv, case["tokens"], d, torch.bfloat16)
        return {"k": _held(k.transpose(0, 1)), "v": _held(v.transpose(0, 1))}
    rows, pos0, T = _blocks(case)
    if case["kind"] == "accept":
        return _exact_accept(case, seed, rows, pos0, T)
    kc, vc = _keys_values(seed, 1, (case["requests"],), hkv, _max_seq(case), d, _dtype(case))
    q = _normal(_gen(seed, 2), int(T.sum()), hq, d, dtype=_dtype(case)).double()
    trees = _trees(case) if case["kind"] != "attn8" else None
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    a = 0
    for j, (r, p, t) in enumerate(zip(rows.tolist(), pos0.tolist(), T.tolist())):
        k, v = kc[r, :, :p + t], vc[r, :, :p + t]
        k, v = (_held(k), _held(v)) if case["kind"] != "tree" else (k.double(), v.double())
        reads = torch.ones(t, p + t, dtype=torch.bool)
        if trees is None:
            reads = reads.tril(p)
        else:
            reads[:, p:] = False
            for i in range(t):
                reads[i, [p + x for x in _path(trees[j][0], i)]] = True
        reads = reads.to(DEV)
        for h in range(hkv):
            g = hq // hkv
            s = torch.einsum("tgd,pd->tgp", q[a:a + t, h * g:(h + 1) * g], k[h]) / math.sqrt(d)
            w = torch.softmax(s.masked_fill(~reads[:, None], -math.inf), dim=-1)
            out[a:a + t, h * g:(h + 1) * g] = torch.einsum("tgp,pd->tgd", w, v[h])
        a += t
    return {"out": out.reshape(len(out), -1)}


def _exact_accept(case, seed, rows, pos0, T):
    hq, hkv, d = HEADS[case["heads"]]
    k, v = _keys_values(seed, 1, (case["layers"], case["requests"]), hkv, _max_seq(case), d, _dtype(case))
    tokens, y = _accept_tokens(case, seed)
    t_max, a = int(T.max()), 0
    acc, paths, out = [], [], []
    for (parents, _), r, p, t in zip(_trees(case), rows.tolist(), pos0.tolist(), T.tolist()):
        path = [0]
        while True:
            nxt = [c for c in range(path[-1] + 1, t) if parents[c] == path[-1] and tokens[a + c] == y[a + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        at = torch.tensor([p + i for i in path], device=DEV)
        k[:, r, :, p:p + len(path)] = k[:, r][:, :, at]
        v[:, r, :, p:p + len(path)] = v[:, r][:, :, at]
        acc.append(len(path) - 1)
        paths.append(path + [-1] * (t_max - len(path)))
        out.append([int(y[a + i]) for i in path] + [-1] * (t_max - len(path)))
        a += t
    k = _k_pack(k) if case["dtype"] == "bf16" else k
    return {"accepted": torch.tensor(acc), "path": torch.tensor(paths, dtype=torch.int32), "tokens": torch.tensor(out),
            "k": k, "v": _v_pack(v)}
