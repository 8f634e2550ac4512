"""The 8-bit KV cache (write, read, attention) and trees of drafted tokens (masks, attention, acceptance, compaction)
against plain 64-bit implementations; refusals on the CPU.

Tolerances.  The cache: exact.  Attention: with w the exact normalised weights and A = sum w |v| (per output element),
the kernel rounds each weight to bf16 (relative 2^-8 at most, eps / 2) and the output to bf16 (2^-8 |out|); the fp32
score of a position is off by at most (D + 4) 2^-24 sum |q k| scale, which moves its weight by that much relatively (and
the sum of the weights likewise): below 2^-12 for every case here.  So |got - ref| <= 1.01 * 2^-8 (|ref| + A) + 2^-12 A.
fp32: the sums of n positions and D products, one after the other: (n + D + 64) 2^-24 (1 + max sum |q k| scale) 2 A.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn


def _lsk():
    from thesis_amd import _lsk

    _lsk.load()
    return _lsk


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)


def _cat(xs, dtype, dev):
    return torch.as_tensor(np.concatenate([np.asarray(x, dtype=np.int64) for x in xs]), dtype=dtype).to(dev)


# ----------------------------------------------------------------------------- plain forms

def exponents(x):
    """e of the cache's rule for vectors x [.., d] (64 bits): the smallest integer >= -117 with amax <= 448 * 2^e."""
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1).double()
    e = torch.ceil(torch.log2(torch.where(a > 0, a, 448.0) / 448.0)).clamp(min=-117)
    assert (a <= 448.0 * torch.exp2(e)).all()
    return e.to(torch.int64)


def held(x):
    """What the 8-bit cache stands for (64 bits), from e4m3's definition: units of 2^(max(floor log2, -6) - 3)."""
    s = torch.exp2(exponents(x).double())[..., None]
    y = x.double() / s
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -40))).clamp(min=-6.0) - 3.0)
    r = torch.round(y / unit) * unit * s
    return torch.where(torch.isfinite(x), r, torch.full_like(r, math.nan))


def ancestors(parents):
    """Index sets a node reads: its ancestors and itself (a parent outside [0, i) is none)."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else frozenset()) | {i})
    return out


def random_tree(rng, t):
    return [-1] + [int(i - 1 if rng.random() < 0.5 else rng.integers(i)) for i in range(1, t)]


def words_of(sets, w):
    m = np.zeros((len(sets), w), dtype=np.uint32)
    for i, s in enumerate(sets):
        for j in s:
            if j < 32 * w:
                m[i, j // 32] |= np.uint32(1 << (j % 32))
    return m.view(np.int32)


def attention(q, k, v, blocks, scale, sets=None):
    """q [N, Hq, D], k / v [B, Hkv, S, D] (64 bits) -> (out [N, Hq D], A [N, Hq D], largest sum |q k| scale)."""
    N, Hq, D = q.shape
    g = Hq // k.shape[1]
    out = torch.zeros(N, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    big = 0.0
    for (qs, p0, T, row) in blocks:
        for t in range(T):
            reads = list(range(p0 + t + 1)) if sets is None else \
                list(range(p0)) + [p0 + j for j in sorted(sets[qs + t]) if j <= t]
            if not reads:
                continue
            kr, vr = k[row][:, reads], v[row][:, reads]
            qt = q[qs + t].view(-1, g, D)
            s = (qt[:, :, None] * kr[:, None]).sum(-1) * scale
            qk = (qt.abs()[:, :, None] * kr.abs()[:, None]).sum(-1) * scale
            big = max(big, float(qk.nan_to_num(0, 0, 0).max()))
            w = torch.softmax(s, dim=-1)
            out[qs + t] = (w[..., None] * vr[:, None]).sum(2).view(Hq, D)
            mag[qs + t] = (w[..., None] * vr.abs()[:, None]).sum(2).view(Hq, D)
    return out.view(N, -1), mag.view(N, -1), big


def assert_close_bf16(got, ref, mag):
    got, ref, mag = got.double().cpu(), ref.cpu(), mag.cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    tol = 1.01 * 2.0 ** -8 * (ref.abs() + mag) + 2.0 ** -12 * mag + 1e-30
    err = (got - ref).abs()
    assert (err[fine] <= tol[fine]).all(), (err[fine] / tol[fine]).max()
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])


def assert_close_f32(got, ref, mag, n, d, big):
    tol = (n + d + 64) * 2.0 ** -24 * (1 + big) * 2 * mag + 1e-30
    assert ((got.double().cpu() - ref).abs() <= tol).all()


def pack_blocks(blocks):
    """[(row, pos0, T)] -> [(q_start, pos0, T, row)]"""
    out, off = [], 0
    for (row, p0, t) in blocks:
        out.append((off, p0, t, row))
        off += t
    return out, off


def kv8_from(lsk, cuda, k, v):
    """An 8-bit cache written by kv8_append with dense k, v [B, Hkv, S, D] (bf16)."""
    B, H, S, D = k.shape
    cache = lsk.KV8.zeros(B, H, S, D, cuda)
    rows = torch.arange(B).repeat_interleave(S)
    pos = torch.arange(S).repeat(B)
    flat = lambda x: x.permute(0, 2, 1, 3).reshape(B * S, H, D).contiguous().to(cuda)  # noqa: E731
    lsk.kv8_append(flat(k), flat(v), cache, _i32(rows, cuda), _i32(pos, cuda))
    return cache


def k8_dense(codes):
    """K codes [.., S/64, 4, D/64, 64, 16] -> [.., S, D], index by index from the documented layout."""
    *lead, nb, _, J, _, _ = codes.shape
    S, D = nb * 64, J * 64
    p, d = np.meshgrid(np.arange(S), np.arange(D), indexing="ij")
    pp = p % 64
    a, l16 = pp // 4 % 4, pp // 16 * 4 + pp % 4
    j, lg = d // 64, d // 16 % 4
    off = p // 64 * 64 * D + ((a * J + j) * 64 + lg * 16 + l16) * 16 + d % 16
    flat = codes.view(torch.uint8).reshape(*lead, S * D)
    return flat[..., torch.as_tensor(off.reshape(-1))].reshape(*lead, S, D)


# ----------------------------------------------------------------------------- the 8-bit cache

def _awkward(g, n, h, d, dtype):
    """Vectors of every size: all-zero, tiny, subnormal, huge, with the largest value at and next to 448 * 2^e, ties."""
    x = torch.randn(n, h, d, generator=g) * torch.exp2(torch.randint(-30, 30, (n, h, 1), generator=g).float())
    flat = x.view(-1, d)
    m = flat.shape[0]
    flat[0 % m] = 0.0
    flat[1 % m] = torch.randn(d, generator=g) * 1e-39
    flat[2 % m] = torch.randn(d, generator=g).clamp(-1, 1) * 3e38
    flat[3 % m, 0], flat[3 % m, 1:] = 448.0, torch.arange(1, d).float() / 8          # ties between e4m3 values
    flat[4 % m, 0], flat[4 % m, 1:] = 450.0, torch.arange(1, d).float()              # just past 448: the next scale
    flat[5 % m] = 0.0
    flat[5 % m, d - 1] = -2.0 ** -133
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,h", [(1, 1), (7, 3), (16, 8), (33, 2), (200, 8)])
def test_kv8_append_and_read_are_exact(cuda, dtype, D, n, h):
    """Codes, exponents and storage layout are the definition's; what is read back is code * 2^e; everything else of
    the cache stays as it was, and tokens outside the cache leave it alone."""
    lsk = _lsk()
    g = _gen(n * 7 + D)
    B, S = 3, 192
    k, v = _awkward(g, n, h, D, dtype), _awkward(g, n, h, D, dtype).flip(0)
    slot = torch.randperm(B * S, generator=g)[:n]
    rows, pos = slot // S, slot % S
    if n > 8:                                                         # padding and stray tokens
        rows[3], pos[5], rows[6], pos[7] = -1, S, B, -2
    ok = (rows >= 0) & (rows < B) & (pos >= 0) & (pos < S)
    cache = lsk.KV8.zeros(B, h, S, D, cuda)
    before = torch.randint(0, 120, cache.k.view(torch.uint8).shape, generator=g, dtype=torch.uint8)
    cache.k.view(torch.uint8).copy_(before)
    lsk.kv8_append(k.to(cuda), v.to(cuda), cache, _i32(rows, cuda), _i32(pos, cuda))
    kd = k8_dense(cache.k.cpu())
    vd = cache.v.cpu().view(torch.uint8).transpose(-1, -2).reshape(B, h, S, D)
    want_k, want_v = k8_dense(before.view(E4M3)), torch.zeros(B, h, S, D, dtype=torch.uint8)
    want_ks = torch.full((B, h, S), 127, dtype=torch.uint8)
    want_vs = want_ks.clone()
    for x, codes, exps in ((k, want_k, want_ks), (v, want_v, want_vs)):
        e = exponents(x.double())
        c = (held(x) / torch.exp2(e.double())[..., None]).to(torch.float32).to(E4M3).view(torch.uint8)  # exact values
        codes[rows[ok], :, pos[ok]] = c[ok]
        exps[rows[ok], :, pos[ok]] = (e + 127).to(torch.uint8)[ok]
    neg0 = lambda t: torch.where(t == 128, torch.zeros_like(t), t)    # noqa: E731  (the sign of a zero is free)
    assert torch.equal(cache.ks.cpu(), want_ks) and torch.equal(cache.vs.cpu(), want_vs)
    assert torch.equal(neg0(kd), neg0(want_k)) and torch.equal(neg0(vd), neg0(want_v))
    for out in (BF16, F32):
        kr, vr = lsk.kv8_read(cache, _i32(rows, cuda), _i32(pos, cuda), out)
        for got, x in ((kr, k), (vr, v)):
            want = torch.where(ok[:, None, None], held(x), torch.zeros(1, dtype=torch.float64))
            assert torch.equal(got.cpu().double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv8_runs_of_positions_from_any_start(cuda, D):
    """Prompts from any position, next to each other, across 64-position blocks and up to the cache's end, between
    single tokens: every token's values, and nothing of its neighbours."""
    lsk = _lsk()
    g = _gen(31)
    B, h, S = 6, 2, 256
    runs = [(0, 1, 16), (1, 2, 33), (2, 57, 31), (2, 88, 40), (3, 240, 16), (4, 3, 1), (0, 61, 5), (5, 255, 1),
            (5, 0, 96), (4, 130, 29)]
    rows = torch.cat([torch.full((n,), r) for (r, _, n) in runs])
    pos = torch.cat([torch.arange(p, p + n) for (_, p, n) in runs])
    for shift in (0, 3):                              # (the second time the workgroups hold other runs)
        rows, pos = rows.roll(shift), pos.roll(shift)
        n = len(rows)
        k, v = (torch.randn(n, h, D, generator=g).to(BF16) for _ in range(2))
        cache = lsk.KV8.zeros(B, h, S, D, cuda)
        for x in (cache.k, cache.v):
            x.view(torch.uint8).fill_(57)             # (1.125 everywhere else)
        lsk.kv8_append(k.to(cuda), v.to(cuda), cache, _i32(rows, cuda), _i32(pos, cuda))
        allrows, allpos = torch.arange(B).repeat_interleave(S), torch.arange(S).repeat(B)
        for got, x in zip(lsk.kv8_read(cache, _i32(allrows, cuda), _i32(allpos, cuda), F32), (k, v)):
            want = torch.full((B, S, h, D), 1.125, dtype=torch.float64)
            want[rows, pos] = held(x)
            assert torch.equal(got.cpu().double().view(B, S, h, D), want)
        for got, x in zip(lsk.kv8_read(cache, _i32(rows, cuda), _i32(pos, cuda), F32), (k, v)):
            assert torch.equal(got.cpu().double(), held(x))


@pytest.mark.gpu
def test_kv8_rounds_every_bf16_value_to_the_nearest_code(cuda):
    """All finite bf16 values with a fixed largest value in the vector: the code is the nearest e4m3 value, ties to
    even (torch's own conversion of the scaled value)."""
    lsk = _lsk()
    bits = torch.arange(0, 0x43E0, dtype=torch.int32)                 # 0 .. 448 in bf16
    vals = bits.to(torch.int16).view(BF16)
    n = (len(vals) + 62) // 63
    x = torch.zeros(n, 1, 64, dtype=BF16)
    x[:, 0, 0] = 448.0
    body = torch.zeros(n * 63, dtype=BF16)
    body[:len(vals)] = vals * torch.where(torch.arange(len(vals)) % 2 == 0, 1.0, -1.0).to(BF16)
    x[:, 0, 1:] = body.view(n, 63)
    S = (n + 63) // 64 * 64
    cache = lsk.KV8.zeros(1, 1, S, 64, cuda)
    rows, pos = _i32(np.zeros(n), cuda), _i32(np.arange(n), cuda)
    lsk.kv8_append(x.to(cuda), x.to(cuda), cache, rows, pos)
    assert (cache.ks.cpu()[0, 0, :n] == 127).all()
    want = x.float().to(E4M3).float()
    for got in lsk.kv8_read(cache, rows, pos, F32):
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_kv8_append_takes_strides_and_non_finite_values(cuda):
    """k and v as views of a fused qkv row (at any bf16 address); NaN and infinities become NaN and leave the scale to
    the finite values."""
    lsk = _lsk()
    g = _gen(5)
    n, h, D, S = 9, 2, 64, 64
    buf = torch.randn(n * 2 * (h * D) + n + 1, generator=g).to(BF16)
    buf[1 + 5], buf[1 + 70], buf[1 + 130 + h * D] = math.nan, math.inf, -math.inf
    dev = buf.to(cuda)
    view = lambda t, o: torch.as_strided(t, (n, h, D), (2 * h * D + 1, D, 1), o)  # noqa: E731
    cache = lsk.KV8.zeros(1, h, S, D, cuda)
    rows, pos = _i32(np.zeros(n), cuda), _i32(np.arange(n), cuda)
    lsk.kv8_append(view(dev, 1), view(dev, 1 + h * D), cache, rows, pos)
    for got, x in zip(lsk.kv8_read(cache, rows, pos, F32), (view(buf, 1), view(buf, 1 + h * D))):
        want = held(x)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().double().nan_to_num(0), want.nan_to_num(0))
    assert torch.isnan(held(view(buf, 1))).sum() == 3


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_largest_finite_values_stay_finite(cuda, dtype, D):
    """At e = 120 the e4m3 value 256 would stand for 2^128: codes end at 240, within 2^-4 of the value.  A query of
    zeros weighs such keys equally."""
    lsk = _lsk()
    top = torch.finfo(dtype).max
    x = torch.randn(6, 2, D, generator=_gen(7)).to(dtype)
    x[0, :, :4] = torch.tensor([top, -top, top / 2, top / 300], dtype=dtype)
    x[1, :, 5], x[2, :, 5], x[3, :, 5] = 248 * 2.0 ** 120, -247 * 2.0 ** 120, 2.0 ** 127
    x[4] = top * torch.linspace(-1, 1, D, dtype=torch.float64).to(dtype)
    v = torch.randn(6, 2, D, generator=_gen(8)).to(dtype)
    cache = lsk.KV8.zeros(1, 2, 64, D, cuda)
    rows, pos = _i32(np.zeros(6), cuda), _i32(np.arange(6), cuda)
    for k_, v_ in ((x, v), (v, x)):
        lsk.kv8_append(k_.to(cuda), v_.to(cuda), cache, rows, pos)
        want = held(x).clamp(-240 * 2.0 ** 120, 240 * 2.0 ** 120)
        assert ((want - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * 2.0 ** 120).all()
        for out in (F32, BF16):
            got = lsk.kv8_read(cache, rows, pos, out)[0 if k_ is x else 1]
            assert torch.equal(got.double().cpu(), want)
        if k_ is x:
            assert cache.ks[0, :, 0].tolist() == [247, 247]
            tab = [(0, 5, 1, 0)]
            got = lsk.kv8_attn(torch.zeros(1, 2, D, dtype=BF16, device=cuda), cache, lsk.AttnPlan(tab, 2, cache))
            dense = lambda t: held(t).permute(1, 0, 2)[None]          # noqa: E731
            zero = torch.zeros(1, 2, D, dtype=torch.float64)
            ref, mag, _ = attention(zero, torch.zeros_like(dense(v)), dense(v), tab, 1.0)
            assert_close_bf16(got, ref, mag)


# ----------------------------------------------------------------------------- attention

def _heads(case):
    return {"gqa128": (8, 2, 128), "gqa64": (8, 2, 64), "mha64": (3, 3, 64), "mqa128": (5, 1, 128)}[case]


# (row, pos0, T) blocks: single tokens at the first position and far along, blocks that start or end inside a step or
# at its edge, contexts over several splits, repeated cache rows, blocks without tokens
BLOCKS = {
    "first": [(0, 0, 1)],
    "decode": [(2, 0, 1), (0, 63, 1), (1, 64, 1), (3, 300, 1)],
    "verify": [(1, 0, 5), (0, 60, 9), (3, 127, 2), (2, 1000, 7)],
    "wide": [(0, 10, 40), (2, 500, 23), (1, 0, 64)],
    "empty": [(0, 5, 0), (1, 700, 3), (2, 0, 0)],
    "shared": [(1, 90, 3), (1, 40, 2), (0, 1023, 1)],
}


def _attn_inputs(seed, heads, blocks, dtype=BF16, S=1088, B=4):
    Hq, Hkv, D = heads
    g = _gen(seed)
    tab, n = pack_blocks(blocks)
    q = torch.randn(n, Hq, D, generator=g).to(dtype)
    k = (torch.randn(B, Hkv, S, D, generator=g) * torch.exp(0.4 * torch.randn(1, Hkv, 1, D, generator=g))).to(dtype)
    v = torch.randn(B, Hkv, S, D, generator=g).to(dtype)
    return tab, q, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("split", [None, 64, 256])
@pytest.mark.parametrize("blocks", BLOCKS)
@pytest.mark.parametrize("heads", ["gqa128", "gqa64", "mha64", "mqa128"])
def test_kv8_attention_matches_64_bits(cuda, heads, blocks, split):
    lsk = _lsk()
    Hq, Hkv, D = _heads(heads)
    tab, q, k, v = _attn_inputs(11, (Hq, Hkv, D), BLOCKS[blocks])
    cache = kv8_from(lsk, cuda, k, v)
    plan = lsk.AttnPlan(tab, Hq, cache, split=split)
    got = lsk.kv8_attn(q.to(cuda), cache, plan)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("split", [64, 128, 512])
def test_attention_merges_up_to_128_splits(cuda, D, split):
    """A long context in as many splits as a plan takes (and one that ends with the last of them), beside short ones."""
    lsk = _lsk()
    Hq, Hkv = 4, 1
    blocks = [(0, 8187, 5), (1, 8000, 1), (2, 1020, 9), (3, 63, 2)]
    tab, q, k, v = _attn_inputs(61, (Hq, Hkv, D), blocks, S=8192)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
    cache = kv8_from(lsk, cuda, k, v)
    plan = lsk.AttnPlan(tab, Hq, cache, split=split)
    assert plan.causal.n_parts >= 8192 // split
    assert_close_bf16(lsk.kv8_attn(q.to(cuda), cache, plan), ref, mag)
    mask = torch.from_numpy(words_of([set(range(i + 1)) for (_, _, t, _) in tab for i in range(t)], 1)).to(cuda)
    ref, mag, _ = attention(q.double(), k.double(), v.double(), tab, 1 / math.sqrt(D))
    kf, vf = lsk.k_to_frag(k).to(cuda), lsk.v_to_blocked(v).to(cuda)
    assert_close_bf16(lsk.tree_attn(q.to(cuda), kf, vf, lsk.AttnPlan(tab, Hq, kf, split=split), mask), ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [None, 128])
@pytest.mark.parametrize("heads", ["gqa128", "gqa64"])
def test_kv8_attention_of_prompts(cuda, heads, split):
    """Whole prompts and a prompt behind a committed prefix, several hundred tokens a block, beside a decode step."""
    lsk = _lsk()
    Hq, Hkv, D = _heads(heads)
    tab, q, k, v = _attn_inputs(107, (Hq, Hkv, D), [(1, 0, 333), (0, 97, 250), (2, 400, 1)], S=448, B=3)
    cache = kv8_from(lsk, cuda, k, v)
    got = lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(tab, Hq, cache, split, tree=False))
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)


def _tree_blocks(blocks, seed):
    rng = np.random.default_rng(seed)
    parents = [random_tree(rng, t) if t else [] for (_, _, t) in blocks]
    return parents, [s for p in parents for s in ancestors(p)]


@pytest.mark.gpu
@pytest.mark.parametrize("split,row_groups", [(None, None), (64, 1), (64, 4), (1024, 2), (128, 4)])
@pytest.mark.parametrize("blocks", BLOCKS)
@pytest.mark.parametrize("kind,heads", [("bf16", "gqa128"), ("bf16", "gqa64"), ("bf16", "mqa128"), ("kv8", "gqa128"),
                                        ("kv8", "mha64"), ("fp32", "gqa64"), ("fp32", "mqa128")])
def test_tree_attention_matches_64_bits(cuda, kind, heads, blocks, split, row_groups):
    lsk = _lsk()
    Hq, Hkv, D = _heads(heads)
    dtype = F32 if kind == "fp32" else BF16
    tab, q, k, v = _attn_inputs(13, (Hq, Hkv, D), BLOCKS[blocks], dtype)
    parents, sets = _tree_blocks(BLOCKS[blocks], 3)
    mask = torch.from_numpy(words_of(sets, (max(t for _, _, t in BLOCKS[blocks]) + 31) // 32)).to(cuda)
    if kind == "kv8":
        cache = kv8_from(lsk, cuda, k, v)
        got = lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(tab, Hq, cache, split, row_groups), mask)
        k, v = held(k), held(v)
    else:
        ks = (lsk.k_to_frag(k) if kind == "bf16" else k).to(cuda)
        plan = lsk.AttnPlan(tab, Hq, ks, split, row_groups)
        got = lsk.tree_attn(q.to(cuda), ks, lsk.v_to_blocked(v).to(cuda), plan, mask)
    ref, mag, big = attention(q.double(), k.double(), v.double(), tab, 1 / math.sqrt(D), sets)
    if kind == "fp32":
        assert_close_f32(got, ref, mag, 1088, D, big)
    else:
        assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "kv8", "fp32"])
def test_masks_of_any_kind_and_rows_that_read_nothing(cuda, kind):
    """Masks that are no tree: rows without a set bit at position 0 give zeros, bits of later nodes and words that a
    long block does not have count as 0, trees of more than 32 and 64 nodes."""
    lsk = _lsk()
    Hq, Hkv, D = 4, 2, 64
    blocks = [(0, 0, 70), (1, 3, 130), (2, 0, 1)]
    dtype = F32 if kind == "fp32" else BF16
    tab, q, k, v = _attn_inputs(17, (Hq, Hkv, D), blocks, dtype, S=192, B=3)
    n = len(q)
    rng = np.random.default_rng(2)
    bits = rng.random((n, 96)) < 0.2                                  # 3 words: nodes from 96 on are never read
    bits[:5] = False                                                  # block 0's first rows read nothing
    bits[n - 1] = False
    sets = [set(np.flatnonzero(r).tolist()) for r in bits]
    mask = torch.from_numpy(words_of(sets, 3)).to(cuda)
    if kind == "kv8":
        cache = kv8_from(lsk, cuda, k, v)

        def run(split, rg):
            return lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(tab, Hq, cache, split, rg), mask)

        k, v = held(k), held(v)
    else:
        ks = (lsk.k_to_frag(k) if kind == "bf16" else k).to(cuda)
        vs = lsk.v_to_blocked(v).to(cuda)

        def run(split, rg):
            return lsk.tree_attn(q.to(cuda), ks, vs, lsk.AttnPlan(tab, Hq, ks, split, rg), mask)

    ref, mag, big = attention(q.double(), k.double(), v.double(), tab, 1 / math.sqrt(D), sets)
    for split, rg in ((None, 1), (64, 1), (None, 4), (64, 4)):
        got = run(split, rg)
        assert (got[:5] == 0).all() and (got[n - 1] == 0).all()
        if kind == "fp32":
            assert_close_f32(got, ref, mag, 192, D, big)
        else:
            assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("row_groups", [1, 4])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["bf16", "kv8", "kv8 causal", "fp32"])
def test_values_that_a_row_does_not_read_never_reach_it(cuda, kind, bad, row_groups):
    """NaN and infinities in nodes that a row does not read, in the slots behind the block and in those of other rows
    leave its bits as they are; a row that reads such a V gets what the formula gives."""
    lsk = _lsk()
    Hq, Hkv, D = 4, 2, 128
    blocks = [(0, 70, 12), (2, 0, 30), (1, 131, 1)]
    dtype = F32 if kind == "fp32" else BF16
    tab, q, k, v = _attn_inputs(19, (Hq, Hkv, D), blocks, dtype, S=192, B=3)
    v[0, :, 77, 100] = 5.0                                            # (the largest also without the dims below)
    parents, sets = _tree_blocks(blocks, 5)
    if kind == "kv8 causal":
        sets = [set(range(i + 1)) for (_, _, t) in blocks for i in range(t)]
    mask = torch.from_numpy(words_of(sets, 1)).to(cuda)

    def run(k, v):
        if kind.startswith("kv8"):
            cache = kv8_from(lsk, cuda, k, v)
            if bad != bad:                                            # slots never written: any byte as a scale
                for b, (_, p0, t, row) in enumerate(tab):
                    cache.ks[row, :, p0 + t:], cache.vs[row, :, p0 + t:] = 255, 255
            plan = lsk.AttnPlan(tab, Hq, cache, None, row_groups)
            return lsk.kv8_attn(q.to(cuda), cache, plan, mask if kind == "kv8" else None).cpu()
        ks = (lsk.k_to_frag(k) if kind == "bf16" else k).to(cuda)
        plan = lsk.AttnPlan(tab, Hq, ks, None, row_groups)
        return lsk.tree_attn(q.to(cuda), ks, lsk.v_to_blocked(v).to(cuda), plan, mask).cpu()

    clean = run(k, v)
    k2, v2 = k.clone(), v.clone()
    for (_, p0, t, row) in tab:
        k2[row, :, p0 + t:], v2[row, :, p0 + t:] = bad, bad
    assert torch.equal(run(k2, v2), clean)
    node = 7                                                          # of block 0, and its V's dims 0 .. 9 and 40
    k2[0, :, 70 + node], v2[0, :, 70 + node, :10], v2[0, :, 70 + node, 40] = bad, bad, bad
    got = run(k2, v2)
    reads = torch.tensor([b == 0 and node in sets[q0 + i] for b, (q0, _, t, _) in enumerate(tab) for i in range(t)])
    assert torch.equal(got[~reads], clean[~reads]) and reads.any() and not reads.all()
    assert torch.isnan(got[reads]).all()                              # (a score that is not finite)
    v3 = v2.clone()
    got = run(torch.where(torch.isfinite(k2), k2, k), v3).view(len(q), Hq, D)
    assert torch.equal(got[~reads], clean.view(len(q), Hq, D)[~reads])
    hit = torch.zeros(D, dtype=torch.bool)
    hit[:10], hit[40] = True, True
    assert torch.equal(got[reads][..., ~hit], clean.view(len(q), Hq, D)[reads][..., ~hit])
    want = torch.full_like(got[reads][..., hit], math.nan if kind.startswith("kv8") else bad)
    assert torch.equal(got[reads][..., hit].nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["bf16", "kv8"])
def test_bad_values_in_trees_of_many_rows_stay_with_their_readers(cuda, kind, bad, D):
    """The same for trees of 80 to 180 rows, whose waves share K and V."""
    lsk = _lsk()
    Hq, Hkv = 8, 2
    blocks = [(0, 70, 20), (2, 64, 45), (1, 131, 33)]
    tab, q, k, v = _attn_inputs(47, (Hq, Hkv, D), blocks, S=256, B=3)
    v[0, :, 77, D - 1] = 5.0                                          # (the largest also without the dims below)
    v[2, :, 104, D - 1] = 5.0
    parents, sets = _tree_blocks(blocks, 5)
    mask = torch.from_numpy(words_of(sets, 2)).to(cuda)

    def run(k, v):
        if kind == "kv8":
            cache = kv8_from(lsk, cuda, k, v)
            for (_, p0, t, row) in tab:                               # slots never written: any byte as a scale
                cache.ks[row, :, p0 + t:], cache.vs[row, :, p0 + t:] = 255, 255
            plan = lsk.AttnPlan(tab, Hq, cache, None, 4)
            assert plan.tree.n_shared == 5 * Hkv and plan.tree.n_rounds == 0
            return lsk.kv8_attn(q.to(cuda), cache, plan, mask).cpu()
        ks = lsk.k_to_frag(k).to(cuda)
        plan = lsk.AttnPlan(tab, Hq, ks, None, 4)
        return lsk.tree_attn(q.to(cuda), ks, lsk.v_to_blocked(v).to(cuda), plan, mask).cpu()

    clean = run(k, v)
    k2, v2 = k.clone(), v.clone()
    for (_, p0, t, row) in tab:
        k2[row, :, p0 + t:], v2[row, :, p0 + t:] = bad, bad
    assert torch.equal(run(k2, v2), clean)
    reads = torch.zeros(len(q), dtype=torch.bool)
    for (b, node) in ((0, 7), (1, 40)):
        q0, p0, t, row = tab[b]
        v2[row, :, p0 + node, :10], v2[row, :, p0 + node, 40] = bad, bad
        reads |= torch.tensor([q0 <= i < q0 + t and node in sets[i] for i in range(len(q))])
    assert reads[:20].any() and reads[20:65].any() and not reads[:20].all() and not reads[20:65].all()
    hit = torch.zeros(D, dtype=torch.bool)
    hit[:10], hit[40] = True, True
    got, clean = run(torch.where(torch.isfinite(k2), k2, k), v2).view(-1, Hq, D), clean.view(-1, Hq, D)
    assert torch.equal(got[~reads], clean[~reads])
    assert torch.equal(got[reads][..., ~hit], clean[reads][..., ~hit])
    want = torch.full_like(got[reads][..., hit], math.nan if kind == "kv8" else bad)
    assert torch.equal(got[reads][..., hit].nan_to_num(7.0), want.nan_to_num(7.0))
    for (b, node) in ((0, 7), (1, 40)):
        k2[tab[b][3], :, tab[b][1] + node] = bad
    got = run(k2, v).view(-1, Hq, D)
    assert torch.equal(got[~reads], clean[~reads]) and torch.isnan(got[reads]).all()


def _run_kind(lsk, cuda, kind, q, k, v, tab, mask, split=None, row_groups=None):
    """One attention launch of a kind (bf16, fp32: trees; kv8: a tree; kv8 causal: no mask) over dense k, v."""
    Hq = q.shape[1]
    if kind.startswith("kv8"):
        cache = kv8_from(lsk, cuda, k, v)
        plan = lsk.AttnPlan(tab, Hq, cache, split, row_groups)
        return lsk.kv8_attn(q.to(cuda), cache, plan, mask if kind == "kv8" else None).cpu()
    ks = (lsk.k_to_frag(k) if kind == "bf16" else k).to(cuda)
    plan = lsk.AttnPlan(tab, Hq, ks, split, row_groups)
    return lsk.tree_attn(q.to(cuda), ks, lsk.v_to_blocked(v).to(cuda), plan, mask).cpu()


def _compare(kind, got, ref, mag, big, D, rows=slice(None)):
    if kind == "fp32":
        assert torch.equal(torch.isnan(got[rows]), torch.isnan(ref[rows]))
        assert_close_f32(got[rows].nan_to_num(0), ref[rows].nan_to_num(0), mag[rows].nan_to_num(0), 1088, D, big)
    else:
        assert_close_bf16(got[rows], ref[rows], mag[rows])


def _minus_infinity(kind, q, k, at):
    """Makes the scores of the slots at [(row, slice)] -infinity: one dim of K, against queries of a fixed sign there.
    An 8-bit cache holds no infinity: there q . k overflows fp32."""
    q[..., 3] = 1000.0 if kind.startswith("kv8") else q[..., 3].abs() + 0.5
    k[..., 3] = 0.0                                                   # (elsewhere the dim adds nothing)
    for row, slots in at:
        if kind.startswith("kv8"):
            k[row, :, slots] = 0.0
        k[row, :, slots, 3] = -3e38 if kind.startswith("kv8") else -math.inf


def _rising(seed, heads, blocks, S=1088, B=4):
    """Inputs whose scores (in log2 units, scale ln 2) climb along the context by steps of 3 to 12, each row at its own
    rate: downwards, not at all, slowly and fast, so that the rows of a tile pass their maxima at different steps."""
    Hq, Hkv, D = heads
    tab, q, k, v = _attn_inputs(seed, heads, blocks, S=S, B=B)
    g, n = _gen(seed + 1), len(q)
    q, k = q * 0.1, k * 0.5
    climb = torch.where(torch.rand(B, Hkv, S, generator=g) < 0.02, 3.0 + 9.0 * torch.rand(B, Hkv, S, generator=g), 0.0)
    k[..., 3] = (climb.cumsum(-1) - climb.sum(-1, keepdim=True) / 2).to(BF16)
    rate = torch.tensor([1.0, -0.5, 0.0, 0.25, 0.75, 1.5])[torch.arange(n * Hq).view(n, Hq) % 6]
    q[..., 3] = rate.to(BF16)
    return tab, q, k, v


def _passes(q, k, tab, sets, step, ways, split, limit):
    """For every row (64 bits): how often a step's maximum passes a finite running one by more than `limit` (log2
    units), and how often by less, with the steps of each split taken by `ways` waves in turn."""
    N, Hq, D = q.shape
    G = Hq // k.shape[1]
    far, near = torch.zeros(N, Hq, dtype=torch.int64), torch.zeros(N, Hq, dtype=torch.int64)
    for (qs, p0, T, row) in tab:
        for t in range(T):
            s = (q[qs + t].view(-1, G, D) @ k[row, :, :p0 + t + 1].transpose(-1, -2)).reshape(Hq, -1)
            if sets is not None:
                skip = [p0 + j for j in range(t + 1) if j not in sets[qs + t]]
                s[:, skip] = -math.inf
            for lo in range(0, s.shape[1], split):
                tiles = [x.amax(-1) for x in s[:, lo:lo + split].split(step, -1)]
                for w in range(ways):
                    m = torch.full((Hq,), -math.inf, dtype=torch.float64)
                    for x in tiles[w::ways]:
                        over = x - m
                        far[qs + t] += torch.isfinite(m) & (over > limit)
                        near[qs + t] += torch.isfinite(m) & (over > 0) & (over <= limit)
                        m = torch.where((over > limit) | torch.isneginf(m), x, m)
    return far, near


@pytest.mark.gpu
@pytest.mark.parametrize("split", [64, 512, 2048])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind,row_groups", [("kv8 causal", None), ("kv8", 1), ("kv8", 2), ("kv8", 4), ("bf16", 1),
                                             ("bf16", 2), ("bf16", 4)])
def test_running_maxima_that_are_passed_again_and_again(cuda, kind, row_groups, D, split):
    """The running maximum moves when it is passed by more than 2^8, and stays when by less: scores that climb by both,
    waves and splits whose maxima lie tens apart.  A score is off by (D + 4) 2^-24 sum |q k| scale at most, which moves
    its weight and the sum of the weights by as much relatively (the sum is `big`)."""
    lsk = _lsk()
    Hq, Hkv = 8, 2
    blocks = [(0, 600, 9), (1, 900, 1), (2, 700, 40), (3, 333, 12), (0, 1050, 20)]
    tab, q, k, v = _rising(101, (Hq, Hkv, D), blocks)
    sets = None if kind == "kv8 causal" else _tree_blocks(blocks, 13)[1]
    mask = None if sets is None else torch.from_numpy(words_of(sets, 2)).to(cuda)
    if kind == "bf16":
        ks, vs = lsk.k_to_frag(k).to(cuda), lsk.v_to_blocked(v).to(cuda)
        got = lsk.tree_attn(q.to(cuda), ks, vs, lsk.AttnPlan(tab, Hq, ks, split, row_groups), mask, math.log(2.0))
    else:
        cache = kv8_from(lsk, cuda, k, v)
        got = lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(tab, Hq, cache, split, row_groups), mask, math.log(2.0))
        if sets is None:                              # the same rows as single tokens: the same bits
            one = [(i, p0 + t, 1, row) for (qs, p0, T, row) in tab for t, i in enumerate(range(qs, qs + T))]
            alone = lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(one, Hq, cache, split), None, math.log(2.0))
            assert torch.equal(alone, got)
        k, v = held(k), held(v)
    q, k, v = q.double(), k.double(), v.double()
    ref, mag, big = attention(q, k, v, tab, math.log(2.0), sets)
    got = got.double().cpu()
    tol = 1.01 * 2.0 ** -8 * (ref.abs() + mag) + (2.0 ** -12 + 2 * (D + 4) * 2.0 ** -24 * big) * mag + 1e-30
    assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).max()
    if split > 64:                                    # (at 64 positions a wave has one step or two)
        step, ways = 32 if row_groups == 4 or kind == "bf16" else 64, 4 // (row_groups or 1)   # of blocks of many rows
        far, near = _passes(q, k, tab, sets, step, ways, split, 8.0)
        tile = far[10:14].reshape(-1)                 # 16 query rows per KV head and tile: four tokens
        assert (far > 0).sum() > 100 and (near > 0).sum() > 100 and len(set(tile.tolist())) > 1


@pytest.mark.gpu
@pytest.mark.parametrize("split", [None, 64])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "kv8", "kv8 causal", "fp32"])
def test_scores_of_minus_infinity_have_weight_zero(cuda, kind, D, split):
    """Slots with a score of -infinity where a row reads no other slot of a wave's step, of its first step or of a
    split: before the block, and as the block's first nodes."""
    lsk = _lsk()
    Hq, Hkv = 8, 2
    dtype = F32 if kind == "fp32" else BF16
    blocks = [(0, 32, 3), (1, 64, 3), (2, 128, 45), (3, 96, 7), (0, 200, 20)]
    tab, q, k, v = _attn_inputs(71, (Hq, Hkv, D), blocks, dtype, S=256)
    _minus_infinity(kind, q, k, [(0, slice(32, 33)), (1, slice(64, 65)), (2, slice(0, 64)), (3, slice(0, 96))])
    # each node reads the root and itself
    sets = [set(range(i + 1)) if kind == "kv8 causal" else {0, i} for (_, _, t) in blocks for i in range(t)]
    mask = torch.from_numpy(words_of(sets, 2)).to(cuda)
    got = _run_kind(lsk, cuda, kind, q, k, v, tab, mask, split, 4)
    if kind.startswith("kv8"):
        k, v = held(k), held(v)
    ref, mag, big = attention(q.double(), k.double(), v.double(), tab, 1 / math.sqrt(D), sets)
    assert torch.isfinite(ref).all()
    _compare(kind, got, ref, mag, big, D)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [None, 64])
@pytest.mark.parametrize("row_groups", [1, 4])
@pytest.mark.parametrize("kind", ["bf16", "kv8", "fp32"])
def test_rows_of_minus_infinity_only_and_rows_that_read_nothing(cuda, kind, row_groups, split):
    """A row that reads nothing gives zeros; one whose scores are all -infinity NaN, as the formula does (over an 8-bit
    cache, where fp32 overflows: the same); nodes whose parent scores -infinity their own V."""
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 64
    dtype = F32 if kind == "fp32" else BF16
    blocks = [(0, 0, 100), (1, 0, 9), (2, 0, 70)]
    tab, q, k, v = _attn_inputs(73, (Hq, Hkv, D), blocks, dtype, S=128)
    sets = [{0, i} for (_, _, t) in blocks for i in range(t)]
    _minus_infinity(kind, q, k, [(0, slice(0, 1)), (1, slice(0, 1)), (2, slice(0, 1))])
    first = [a for (a, _, _, _) in tab]
    nothing = [first[0] + 5, first[0] + 99, first[1] + 8, first[2] + 66]
    for i in nothing:
        sets[i] = set()
    mask = torch.from_numpy(words_of(sets, 4)).to(cuda)
    mask[first[2] + 66, 2] = 1 << 3                                   # (a later node's bit does not count)
    got = _run_kind(lsk, cuda, kind, q, k, v, tab, mask, split, row_groups)
    assert (got[nothing] == 0).all() and torch.isnan(got[first]).all()
    if kind.startswith("kv8"):
        k, v = held(k), held(v)
    ref, mag, big = attention(q.double(), k.double(), v.double(), tab, 1 / math.sqrt(D), sets)
    rest = [i for i in range(len(q)) if i not in first]
    assert torch.isfinite(ref[rest]).all()
    _compare(kind, got, ref, mag, big, D, rest)


@pytest.mark.gpu
def test_an_fp32_chain_of_minus_infinity_is_the_ragged_attentions(cuda):
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 64
    tab, q, k, v = _attn_inputs(79, (Hq, Hkv, D), [(0, 0, 5), (1, 40, 2)], F32, S=128)
    _minus_infinity("fp32", q, k, [(0, slice(0, 2)), (1, slice(0, 42))])
    kd, vd = k.to(cuda), lsk.v_to_blocked(v).to(cuda)
    mask = torch.from_numpy(words_of([set(range(i + 1)) for t in (5, 2) for i in range(t)], 1)).to(cuda)
    p = lsk.AttnPlan(tab, Hq, kd)
    want = torch.empty(len(q), Hq * D, device=cuda)
    b = torch.tensor(tab, dtype=torch.int32, device=cuda)
    lsk.ragged_attn(q.to(cuda), kd, vd, b, p.works, p.n_works, None, 0, 0, want, Hq, 1 / math.sqrt(D),
                    rows_cap=p.rows_cap)
    got = lsk.tree_attn(q.to(cuda), kd, vd, p, mask)
    assert torch.isnan(want[[0, 1, 5, 6]]).all() and torch.isfinite(want[2:5]).all()
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 64, 128])
def test_an_fp32_chain_gives_the_ragged_attentions_bits(cuda, D):
    lsk = _lsk()
    Hq, Hkv = 8, 2
    blocks = [(0, 0, 5), (2, 63, 9), (1, 700, 40), (3, 1000, 1)]
    tab, q, k, v = _attn_inputs(23, (Hq, Hkv, D), blocks, F32)
    kd, vd = k.to(cuda), lsk.v_to_blocked(v).to(cuda)
    sets = [set(range(i + 1)) for (_, _, t) in blocks for i in range(t)]
    mask = torch.from_numpy(words_of(sets, 2)).to(cuda)
    p = lsk.AttnPlan(tab, Hq, kd)
    want = torch.empty(len(q), Hq * D, device=cuda)
    b = torch.tensor(tab, dtype=torch.int32, device=cuda)
    lsk.ragged_attn(q.to(cuda), kd, vd, b, p.works, p.n_works, None, 0, 0, want, Hq, 1 / math.sqrt(D),
                    rows_cap=p.rows_cap)
    assert torch.equal(lsk.tree_attn(q.to(cuda), kd, vd, p, mask), want)


@pytest.mark.gpu
def test_trees_of_one_node_and_causal_launches_agree(cuda):
    """A launch with a mask gives, for blocks of up to 32 rows whose mask is the causal rule, the causal launch's bits:
    a root without drafts is a decode step."""
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 128
    blocks = [(0, 0, 1), (2, 63, 8), (1, 700, 1), (3, 1000, 5)]
    tab, q, k, v = _attn_inputs(43, (Hq, Hkv, D), blocks)
    cache = kv8_from(lsk, cuda, k, v)
    mask = torch.from_numpy(words_of([set(range(i + 1)) for (_, _, t) in blocks for i in range(t)], 1)).to(cuda)
    plan = lsk.AttnPlan(tab, Hq, cache, split=256, row_groups=4)
    assert torch.equal(lsk.kv8_attn(q.to(cuda), cache, plan, mask), lsk.kv8_attn(q.to(cuda), cache, plan))


@pytest.mark.gpu
@pytest.mark.parametrize("row_groups", [1, 4])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["kv8", "kv8 tree", "tree"])
def test_a_rows_result_depends_on_its_block_only(cuda, kind, D, row_groups):
    """The same rows alone, in another order, next to others (in launches of 1, 2 and 3 tiles) and as single tokens
    (causal) give the same bits."""
    lsk = _lsk()
    Hq, Hkv = 8, 2
    blocks = [(0, 37, 9), (3, 500, 30), (1, 0, 3), (2, 900, 60)]
    tab, q, k, v = _attn_inputs(29, (Hq, Hkv, D), blocks)
    _, sets = _tree_blocks(blocks, 7)
    words = torch.from_numpy(words_of(sets, 2)).to(cuda)
    qd = q.to(cuda)
    cache = kv8_from(lsk, cuda, k, v)
    kf, vf = lsk.k_to_frag(k).to(cuda), lsk.v_to_blocked(v).to(cuda)

    def run(sel):
        """sel: [(row, pos0, T, first token)]"""
        tab, _ = pack_blocks([s[:3] for s in sel])
        idx = torch.cat([torch.arange(s[3], s[3] + s[2]) for s in sel]).to(cuda)
        plan = lsk.AttnPlan(tab, Hq, kf if kind == "tree" else cache, split=256, row_groups=row_groups)
        m = words[idx].contiguous()
        if kind == "tree":
            return lsk.tree_attn(qd[idx], kf, vf, plan, m), idx
        return lsk.kv8_attn(qd[idx], cache, plan, m if kind == "kv8 tree" else None), idx

    whole = [(r, p, t, a) for (a, p, t, r) in tab]
    full, _ = run(whole)
    for sel in ([whole[1]], [whole[2]], [whole[3], whole[0]], whole[::-1]):
        got, idx = run(sel)
        assert torch.equal(got, full[idx])
    if kind == "kv8":
        r, p, t, a = whole[1]
        got, idx = run([(r, p + i, 1, a + i) for i in range(t)])
        assert torch.equal(got, full[idx])


@pytest.mark.gpu
def test_attention_takes_strided_queries_at_any_address(cuda):
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 64
    blocks = [(0, 37, 9), (1, 0, 3), (2, 200, 20)]
    tab, q, k, v = _attn_inputs(31, (Hq, Hkv, D), blocks, S=256)
    n = len(q)
    _, sets = _tree_blocks(blocks, 9)
    mask = torch.from_numpy(words_of(sets, 1)).to(cuda)
    cache = kv8_from(lsk, cuda, k, v)
    kf, vf = lsk.k_to_frag(k).to(cuda), lsk.v_to_blocked(v).to(cuda)
    buf = torch.zeros(n * 1001 + 1, dtype=BF16, device=cuda)
    strided = torch.as_strided(buf, (n, Hq, D), (1001, D + 3, 1), 1)
    strided.copy_(q)
    heads_first = q.transpose(0, 1).contiguous().to(cuda).transpose(0, 1)
    odd = torch.zeros(n * Hq * D + 1, dtype=BF16, device=cuda)
    out = odd[1:].view(n, Hq * D)                                     # an output that is only 2-byte aligned
    p8, pt = lsk.AttnPlan(tab, Hq, cache, split=64), lsk.AttnPlan(tab, Hq, kf, split=64)
    for run in (lambda x, o: lsk.kv8_attn(x, cache, p8, out=o), lambda x, o: lsk.kv8_attn(x, cache, p8, mask, out=o),
                lambda x, o: lsk.tree_attn(x, kf, vf, pt, mask, out=o)):
        want = run(q.to(cuda), None)
        for x in (strided, heads_first):
            assert torch.equal(run(x, None), want)
        assert run(q.to(cuda), out) is out and torch.equal(out, want) and odd[0] == 0
    same = q[:, :1].expand(n, Hq, D)                                  # one query for every head (stride 0)
    assert torch.equal(lsk.kv8_attn(same.to(cuda)[:, :1].expand(n, Hq, D), cache, p8),
                       lsk.kv8_attn(same.contiguous().to(cuda), cache, p8))


@pytest.mark.gpu
def test_attention_scale_streams_and_graph_replays(cuda):
    """A scale of the caller's; calls on a side stream; a captured call replayed with new queries and cache contents
    between eager calls (each call's split partials are its own)."""
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 128
    blocks = [(0, 700, 9), (1, 900, 3)]
    tab, q, k, v = _attn_inputs(37, (Hq, Hkv, D), blocks)
    _, sets = _tree_blocks(blocks, 9)
    mask = torch.from_numpy(words_of(sets, 1)).to(cuda)
    cache = kv8_from(lsk, cuda, k, v)
    kf, vf = lsk.k_to_frag(k).to(cuda), lsk.v_to_blocked(v).to(cuda)
    p8, pt = lsk.AttnPlan(tab, Hq, cache, split=256), lsk.AttnPlan(tab, Hq, kf, split=256)
    assert p8.causal.n_parts > 0 and pt.tree.n_parts > 0
    qd = q.to(cuda)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 0.03)
    assert_close_bf16(lsk.kv8_attn(qd, cache, p8, scale=0.03), ref, mag)

    def both():
        return lsk.kv8_attn(qd, cache, p8), lsk.tree_attn(qd, kf, vf, pt, mask)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = both()
        graphs.append((g, outs))
    for i in range(4):
        qd.copy_((torch.randn(q.shape, generator=_gen(100 + i))).to(BF16))
        want = both()
        for g, outs in graphs:
            g.replay()
            _ = both()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["kv8", "kv8 causal", "bf16", "fp32"])
def test_a_plan_serves_launches_on_other_streams(cuda, kind):
    """A plan whose upload waits behind its stream's work, used on another stream at once, and dropped before that
    stream's launch has run, while its own stream takes new memory: the launch's records stay what they are."""
    lsk = _lsk()
    Hq, Hkv, D = 8, 2, 64
    blocks = [(0, 200, 9), (1, 130, 40), (2, 0, 1)]
    tab, q, k, v = _attn_inputs(83, (Hq, Hkv, D), blocks, F32 if kind == "fp32" else BF16, S=256, B=3)
    mask = torch.from_numpy(words_of(_tree_blocks(blocks, 9)[1], 2)).to(cuda)
    if kind.startswith("kv8"):
        cache = kv8_from(lsk, cuda, k, v)
        call = lambda plan: lsk.kv8_attn(qd, cache, plan, mask if kind == "kv8" else None)  # noqa: E731
    else:
        cache = (lsk.k_to_frag(k) if kind == "bf16" else k).to(cuda)
        vs = lsk.v_to_blocked(v).to(cuda)
        call = lambda plan: lsk.tree_attn(qd, cache, vs, plan, mask)  # noqa: E731
    qd = q.to(cuda)
    want = call(lsk.AttnPlan(tab, Hq, cache, None if kind == "fp32" else 64))
    torch.cuda.synchronize()
    own, other = torch.cuda.Stream(), torch.cuda.Stream()
    for late_upload in (True, False):
        with torch.cuda.stream(own):
            if late_upload:
                torch.cuda._sleep(20_000_000)
            plan = lsk.AttnPlan(tab, Hq, cache, None if kind == "fp32" else 64)
        sizes = [t.numel() for t in plan._buffers]
        with torch.cuda.stream(other):
            if not late_upload:
                torch.cuda._sleep(20_000_000)
            got = call(plan)
            again = call(plan)
        del plan
        with torch.cuda.stream(own):
            fresh = [torch.zeros(n, dtype=torch.int32, device=cuda) for n in sizes for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want) and len(fresh) == 4 * len(sizes)


@pytest.mark.gpu
def test_plans_and_captures(cuda):
    """A plan is not made inside a capture, nor used there while its upload may still be on its way."""
    lsk = _lsk()
    tab, q, k, v = _attn_inputs(89, (8, 2, 64), [(0, 200, 9), (1, 130, 4)], S=256, B=2)
    cache, qd = kv8_from(lsk, cuda, k, v), q.to(cuda)
    plan = lsk.AttnPlan(tab, 8, cache)
    want = lsk.kv8_attn(qd, cache, plan)

    class Pending:
        def query(self):
            return False

    uploaded, g = plan._uploaded, torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(lsk.LskError):
            lsk.AttnPlan(tab, 8, cache)
        plan._uploaded = Pending()
        with pytest.raises(lsk.LskError):
            lsk.kv8_attn(qd, cache, plan)
        plan._uploaded = uploaded
        got = lsk.kv8_attn(qd, cache, plan)
    for i in range(3):
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(lsk.kv8_attn(qd, cache, plan), want)


@pytest.mark.gpu
def test_attention_of_offsets_past_32_bits(cuda):
    """Cache rows whose first byte lies past 4 GiB: appended, read and attended to."""
    lsk = _lsk()
    Hq, Hkv, D, S = 2, 1, 128, 65536
    B = (5 << 30) // (S * D)                                          # K codes of 5 GiB
    cache = lsk.KV8.zeros(B, Hkv, S, D, cuda)
    g = _gen(41)
    n, row = 300, B - 1
    k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
    pos = torch.arange(n)
    rows = _i32(np.full(n, row), cuda)
    lsk.kv8_append(k.to(cuda), v.to(cuda), cache, rows, _i32(pos, cuda))
    assert torch.equal(lsk.kv8_read(cache, rows, _i32(pos, cuda), F32)[0].cpu().double(), held(k))
    tab, q = [(0, n - 4, 4, row)], torch.randn(4, Hq, D, generator=g).to(BF16)
    got = lsk.kv8_attn(q.to(cuda), cache, lsk.AttnPlan(tab, Hq, cache))
    dense = lambda x: held(x).permute(1, 0, 2)[None].expand(row + 1, -1, -1, -1)  # noqa: E731
    ref, mag, _ = attention(q.double(), dense(k), dense(v), tab, 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
def test_trees_and_compaction_past_32_bits(cuda):
    """A tree of many rows in a bf16 cache row whose first byte lies past 4 GiB: attended to, accepted and compacted."""
    lsk = _lsk()
    Hq, Hkv, D, S = 8, 1, 128, 32768
    B = (5 << 30) // (S * D * 2)
    kf = torch.zeros(1, B, Hkv, S // 32, D // 16, 64, 8, dtype=BF16, device=cuda)
    vb = torch.zeros(1, B, Hkv, S // 32, D, 32, dtype=BF16, device=cuda)
    g, rng = _gen(53), np.random.default_rng(53)
    p0, T, row = 100, 40, B - 1
    n = p0 + T
    k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
    lsk.kv_append(k.to(cuda), v.to(cuda), kf[0], vb[0], _i32(np.full(n, row), cuda), _i32(np.arange(n), cuda))
    parents = random_tree(rng, T)
    tab, q = [(0, p0, T, row)], torch.randn(T, Hq, D, generator=g).to(BF16)
    sets = ancestors(parents)
    mask = torch.from_numpy(words_of(sets, 2)).to(cuda)
    got = lsk.tree_attn(q.to(cuda), kf[0], vb[0], lsk.AttnPlan(tab, Hq, kf[0]), mask)
    dense = lambda x: x.double().permute(1, 0, 2)[None].expand(row + 1, -1, -1, -1)  # noqa: E731
    ref, mag, _ = attention(q.double(), dense(k), dense(v), tab, 1 / math.sqrt(D), sets)
    assert_close_bf16(got, ref, mag)
    path = [0] + sorted(rng.choice(np.arange(1, T), 12, replace=False).tolist())
    lsk.kv_compact(kf, vb, _i32([row], cuda), _i32([p0], cuda), torch.tensor([12], device=cuda), _i32([path], cuda))
    src = list(range(p0)) + [p0 + j for j in path]
    for got, x in ((lsk.k_from_frag(kf[0, row].cpu()), k), (lsk.v_from_blocked(vb[0, row].cpu()), v)):
        assert torch.equal(got[0, :len(src)], x[src, 0]) and torch.equal(got[0, len(src):n], x[len(src):, 0])
        assert (got[0, n:] == 0).all()


# ----------------------------------------------------------------------------- masks, acceptance, compaction

def accept(parents, tokens, y):
    path = [0] if parents else []
    while path:
        nxt = [c for c in range(path[-1] + 1, len(parents)) if parents[c] == path[-1] and tokens[c] == y[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


def _forest(seed, sizes, vocab=3):
    """Trees with few different tokens (siblings share some, long paths match by chance)."""
    rng = np.random.default_rng(seed)
    parents = [random_tree(rng, t) if t else [] for t in sizes]
    tokens = [rng.integers(0, vocab, t) for t in sizes]
    y = [rng.integers(0, vocab, t) for t in sizes]
    return parents, tokens, y


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [64, 1, 0, 13], [65, 33, 2], [300, 64, 7], [1] * 70])
def test_tree_masks_and_acceptance_are_exact(cuda, sizes):
    lsk = _lsk()
    parents, tokens, y = _forest(len(sizes), sizes)
    if len(sizes) == 4:
        parents[3][5], parents[3][6] = 9, -3                          # no parents: a later node, a negative index
        tokens[0][:], y[0][:] = 1, 1                                  # every child matches: the lowest is taken
    starts = np.concatenate([[0], np.cumsum(sizes)[:-1]])
    n, most = sum(sizes), max(sizes)
    flat = lambda xs, dt: _cat(xs, dt, cuda)                          # noqa: E731
    par = flat(parents, torch.int32)
    mask, depth = lsk.tree_masks(par, _i32(starts, cuda), _i32(sizes, cuda), most)
    sets = [s for p in parents for s in ancestors(p)]
    assert np.array_equal(mask.cpu().numpy(), words_of(sets, (most + 31) // 32))
    assert depth.cpu().tolist() == [len(s) - 1 for s in sets]
    for extra in (0, 5):
        acc, path, out = lsk.tree_accept(flat(y, torch.int64), flat(tokens, torch.int64), par, _i32(starts, cuda),
                                         _i32(sizes, cuda), most + extra)
        for b in range(len(sizes)):
            want = accept(parents[b], tokens[b], y[b])
            pad = [-1] * (most + extra - len(want))
            assert int(acc[b]) == len(want) - 1
            assert path[b].tolist() == want + pad
            assert out[b].tolist() == [int(y[b][i]) for i in want] + pad
    # a chain: lsk_greedy_accept's counts
    T = 9
    draft = np.array([5, 1, 2, 3, 4, 5, 6, 7, 8])
    yv = np.array([1, 2, 3, 9, 5, 6, 7, 8, 1])
    acc, path, out = lsk.tree_accept(*(torch.as_tensor(x).to(cuda) for x in (yv, draft)), _i32(np.arange(T) - 1, cuda),
                                     _i32([0], cuda), _i32([T], cuda), T)
    seq = torch.as_tensor(draft[None]).to(cuda).contiguous()
    a2, y2 = torch.empty(1, dtype=torch.long, device=cuda), torch.empty(T, dtype=torch.long, device=cuda)
    lsk.greedy_accept(torch.as_tensor(yv).to(cuda), seq, T, _i32([0], cuda), _i32([0], cuda), _i32([T], cuda), None, 1,
                      a2, y2)
    assert int(acc) == int(a2) == 3 and out[0, :4].tolist() == yv[:4].tolist()


@pytest.mark.gpu
def test_tree_acceptance_of_blocks_outside_the_tokens(cuda):
    """Blocks that reach past the tokens, and nodes past max_nodes, take no part; nothing is read out of bounds."""
    lsk = _lsk()
    n = 10
    par, tok = _i32(np.arange(n) - 1, cuda), torch.zeros(n, dtype=torch.int64, device=cuda)
    starts, lens = _i32([0, 8, -1, 11, 0], cuda), _i32([10, 3, 2, 1, -4], cuda)
    acc, path, out = lsk.tree_accept(tok, tok, par, starts, lens, 4)
    assert acc.tolist() == [3, -1, -1, -1, -1] and path[0].tolist() == [0, 1, 2, 3] and (path[1:] == -1).all()
    mask, depth = lsk.tree_masks(par, starts[:4], _i32([0, 3, 2, 1], cuda), 4)
    assert (mask == 0).all() and (depth == 0).all()


def _caches(lsk, cuda, fmt, L, B, H, S, D, g):
    dt = F32 if fmt == "fp32" else BF16
    k, v = (torch.randn(L, B, H, S, D, generator=g).to(dt) for _ in range(2))
    if fmt == "kv8":
        layers = [kv8_from(lsk, cuda, k[i], v[i]) for i in range(L)]
        cache = lsk.KV8(*(torch.stack([c[j].view(torch.uint8) for c in layers]) for j in range(4)))
        return lsk.KV8(cache.k.view(E4M3), cache.v.view(E4M3), cache.ks, cache.vs), held(k), held(v)
    return ((lsk.k_to_frag(k) if fmt == "bf16" else k).to(cuda), lsk.v_to_blocked(v).to(cuda)), k.clone(), v.clone()


def _dense(lsk, cuda, fmt, cache, dims):
    L, B, H, S, D = dims
    if fmt != "kv8":
        k, v = cache
        return (lsk.k_from_frag(k.cpu()) if fmt == "bf16" else k.cpu()), lsk.v_from_blocked(v.cpu())
    rows, pos = _i32(np.repeat(np.arange(B), S), cuda), _i32(np.tile(np.arange(S), B), cuda)
    out = [lsk.kv8_read(cache.layer(i), rows, pos, F32) for i in range(L)]
    return tuple(torch.stack([o[j] for o in out]).view(L, B, S, H, D).transpose(2, 3).cpu() for j in (0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,D", [("bf16", 128), ("bf16", 64), ("fp32", 16), ("fp32", 32), ("fp32", 128), ("kv8", 128),
                                   ("kv8", 64)])
def test_compaction_moves_the_accepted_paths_and_nothing_else(cuda, fmt, D):
    lsk = _lsk()
    L, B, H, S = 2, 5, 2, 192
    cache, k, v = _caches(lsk, cuda, fmt, L, B, H, S, D, _gen(D))
    rows, pos0 = [3, 0, 4, 1, 7, 2], [5, 60, 0, 191, 3, 100]          # row 7 is outside, row 1 ends with the cache
    paths = [[0, 2, 3, 7, 20], [0] + list(range(2, 72, 2)), [0], [0, 1], [0, 3], []]
    acc = [len(p) - 1 for p in paths]
    most = max(len(p) for p in paths) + 1
    path = np.full((len(paths), most), -1)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    args = (_i32(rows, cuda), _i32(pos0, cuda), torch.tensor(acc, device=cuda), _i32(path, cuda))
    (lsk.kv8_compact(cache, *args) if fmt == "kv8" else lsk.kv_compact(*cache, *args))
    for r, p0, p in zip(rows, pos0, paths):
        if r >= B or (r == 1):
            continue
        src = [p0 + i for i in p]
        for x in (k, v):
            x[:, r, :, p0:p0 + len(p)] = x[:, r][:, :, src].clone()
    got = _dense(lsk, cuda, fmt, cache, (L, B, H, S, D))
    assert torch.equal(got[0].double(), k.double()) and torch.equal(got[1].double(), v.double())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,D", [("bf16", 128), ("bf16", 64), ("fp32", 16), ("fp32", 128), ("kv8", 128), ("kv8", 64)])
def test_compaction_of_long_paths_from_far_nodes(cuda, fmt, D):
    """Paths of several chunks of 16 whose sources lie in many blocks, consecutive runs between them, and a count past
    the path's end (it stops there)."""
    lsk = _lsk()
    L, B, H, S = 1, 4, 1, 1024
    cache, k, v = _caches(lsk, cuda, fmt, L, B, H, S, D, _gen(D + 1))
    rng = np.random.default_rng(D)
    rows, pos0 = [2, 0, 1, 3], [3, 31, 32, 500]
    paths = [[0] + sorted(rng.choice(np.arange(1, 900), 70, replace=False).tolist()),
             [0] + list(range(1, 20)) + [300, 301, 302, 640],
             [0, 959] + [-1] * 3, [0] + list(range(5, 75)) + [523]]
    most = max(len(p) for p in paths) + 1
    path = np.full((len(paths), most), -1)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    acc = [70, 1000, 1, 71]
    args = (_i32(rows, cuda), _i32(pos0, cuda), torch.tensor(acc, device=cuda), _i32(path, cuda))
    (lsk.kv8_compact(cache, *args) if fmt == "kv8" else lsk.kv_compact(*cache, *args))
    for r, p0, p in zip(rows, pos0, paths):
        src = [p0 + i for i in p if i >= 0]
        for x in (k, v):
            x[:, r, :, p0:p0 + len(src)] = x[:, r][:, :, src].clone()
    got = _dense(lsk, cuda, fmt, cache, (L, B, H, S, D))
    assert torch.equal(got[0].double(), k.double()) and torch.equal(got[1].double(), v.double())


@pytest.mark.gpu
@pytest.mark.parametrize("L", [33, 65])
@pytest.mark.parametrize("fmt,D", [("bf16", 64), ("fp32", 16)])
def test_compaction_of_many_layers(cuda, fmt, D, L):
    """Every layer of a large batch, each with its own slots moved."""
    lsk = _lsk()
    B, H, S = 16, 8, 96
    dt = F32 if fmt == "fp32" else BF16
    g, rng = _gen(L), np.random.default_rng(L)
    k, v = (torch.randn(L, B, H, S, D, generator=g).to(dt) for _ in range(2))
    kc, vc = (lsk.k_to_frag(k) if fmt == "bf16" else k).to(cuda), lsk.v_to_blocked(v).to(cuda)
    pos0 = rng.integers(0, 40, B)
    path = np.stack([np.concatenate([[0], np.sort(rng.choice(np.arange(1, 56), 20, replace=False))]) for _ in range(B)])
    acc = rng.integers(0, 21, B)
    rows = rng.permutation(B)
    lsk.kv_compact(kc, vc, _i32(rows, cuda), _i32(pos0, cuda), torch.from_numpy(acc).to(cuda), _i32(path, cuda))
    for i, r in enumerate(rows):
        src = (pos0[i] + path[i, :acc[i] + 1]).tolist()
        for x in (k, v):
            x[:, r, :, pos0[i]:pos0[i] + len(src)] = x[:, r][:, :, src].clone()
    assert torch.equal((lsk.k_from_frag(kc.cpu()) if fmt == "bf16" else kc.cpu()), k)
    assert torch.equal(lsk.v_from_blocked(vc.cpu()), v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_compaction_of_an_engines_cache(cuda, dtype):
    """KVCache's own storage, all layers at once, and a run of them; attention over a layer of it before and after."""
    from thesis_amd.common.model import KVCache, ModelConfig

    lsk = _lsk()
    cfg = ModelConfig(64, 256, 3, 4, 2, 64, 256)
    L, B, H, S, D = 3, 2, 2, 128, cfg.head_dim
    kv = KVCache(cfg, B, S, dtype, cuda)
    g = _gen(109)
    dense = [torch.randn(L, B, H, S, D, generator=g).to(dtype) for _ in range(2)]
    kstore = kv.kf_all if dtype == BF16 else kv.k_all
    kstore.copy_(lsk.k_to_frag(dense[0]) if dtype == BF16 else dense[0])
    kv.vb_all.copy_(lsk.v_to_blocked(dense[1]))
    q = torch.randn(1, 4, D, generator=g).to(dtype)
    tab, sets = [(0, 43, 1, 1)], [{0}]
    mask = torch.from_numpy(words_of(sets, 1)).to(cuda)

    def attend(layer):
        plan = lsk.AttnPlan(tab, 4, kv.kstore[layer], tree=True)
        got = lsk.tree_attn(q.to(cuda), kv.kstore[layer], kv.vb[layer], plan, mask)
        ref, mag, big = attention(q.double(), dense[0][layer].double(), dense[1][layer].double(), tab, 1 / math.sqrt(D),
                                  sets)
        assert_close_f32(got, ref, mag, S, D, big) if dtype == F32 else assert_close_bf16(got, ref, mag)

    path = [0, 2, 5, 9]
    args = (_i32([1], cuda), _i32([40], cuda), torch.tensor([3], device=cuda), _i32([path], cuda))
    attend(1)
    lsk.kv_compact(kstore[1:], kv.vb_all[1:], *args)
    for x in dense:
        x[1:, 1, :, 40:44] = x[1:, 1][:, :, [40 + j for j in path]].clone()
    assert torch.equal(kv.k_all.cpu(), dense[0]) and torch.equal(kv.v_all.cpu(), dense[1])
    attend(1)
    lsk.kv_compact(kstore, kv.vb_all, *args)
    for x in dense:
        x[:, 1, :, 40:44] = x[:, 1][:, :, [40 + j for j in path]].clone()
    assert torch.equal(kv.k_all.cpu(), dense[0]) and torch.equal(kv.v_all.cpu(), dense[1])
    attend(0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp32", "kv8"])
def test_compaction_of_negative_counts_moves_nothing(cuda, fmt):
    """Also counts whose low 32 bits are positive."""
    lsk = _lsk()
    L, B, H, S, D = 1, 4, 2, 64, 64
    cache, _, _ = _caches(lsk, cuda, fmt, L, B, H, S, D, _gen(97))
    before = [t.clone() for t in cache]
    acc = torch.tensor([-1, -(1 << 32) + 5, -(1 << 40) + 3, -(1 << 63)], device=cuda)
    args = (_i32(range(B), cuda), _i32([0, 3, 20, 7], cuda), acc, _i32([[0, 2, 4, 6, 8, 10, 12, 14]] * B, cuda))
    lsk.kv8_compact(cache, *args) if fmt == "kv8" else lsk.kv_compact(*cache, *args)
    bits = lambda t: t.view(torch.uint8).cpu()                        # noqa: E731
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(cache, before))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "kv8"])
def test_a_tree_step_captured_in_two_graphs(cuda, fmt):
    """Masks, write, attention, acceptance and compaction as a captured step, replayed with new inputs between eager
    steps; two graphs of the same step, whose partial outputs are their own."""
    lsk = _lsk()
    L, B, Hq, Hkv, D, S = 2, 3, 8, 2, 128, 512
    sizes, pos0, rows = [40, 5, 21], [300, 64, 7], [1, 2, 0]
    tab, n = pack_blocks(list(zip(rows, pos0, sizes)))
    (cache, _, _) = _caches(lsk, cuda, fmt, L, B, Hkv, S, D, _gen(59))
    layers = [cache.layer(i) for i in range(L)] if fmt == "kv8" else [(cache[0][i], cache[1][i]) for i in range(L)]
    flat = [t.view(torch.uint8) if t.dtype == E4M3 else t for t in cache]
    saved = [t.clone() for t in flat]
    plan = lsk.AttnPlan(tab, Hq, layers[0] if fmt == "kv8" else layers[0][0], split=128, row_groups=4)
    assert plan.tree.n_parts > 0 and plan.tree.n_shared > 0 and plan.tree.n_rounds > 0
    starts, lens = _i32([b[0] for b in tab], cuda), _i32(sizes, cuda)
    trow = _i32(np.repeat(rows, sizes), cuda)
    tpos = _i32(np.concatenate([p + np.arange(t) for p, t in zip(pos0, sizes)]), cuda)
    r_t, p_t = _i32(rows, cuda), _i32(pos0, cuda)
    par, tok, y = _i32(np.zeros(n), cuda), torch.zeros(n, dtype=torch.int64, device=cuda), torch.zeros(
        n, dtype=torch.int64, device=cuda)
    q, k, v = (torch.zeros(n, h, D, dtype=BF16, device=cuda) for h in (Hq, Hkv, Hkv))

    def step():
        mask, depth = lsk.tree_masks(par, starts, lens, max(sizes))
        out = []
        for c in layers:
            if fmt == "kv8":
                lsk.kv8_append(k, v, c, trow, tpos)
                out.append(lsk.kv8_attn(q, c, plan, mask))
            else:
                lsk.kv_append(k, v, c[0], c[1], trow, tpos)
                out.append(lsk.tree_attn(q, c[0], c[1], plan, mask))
        acc, path, new = lsk.tree_accept(y, tok, par, starts, lens, max(sizes))
        lsk.kv8_compact(cache, r_t, p_t, acc, path) if fmt == "kv8" else lsk.kv_compact(*cache, r_t, p_t, acc, path)
        return [*out, mask, depth, acc, path, new]

    def fresh(i):
        parents, tokens, greedy = _forest(60 + i, sizes, vocab=2)
        for t, x in ((par, parents), (tok, tokens), (y, greedy)):
            t.copy_(_cat(x, t.dtype, cuda))
        for j, t in enumerate((q, k, v)):
            t.copy_(torch.randn(t.shape, generator=_gen(70 + 3 * i + j)).to(BF16))

    def reset():
        for t, x in zip(flat, saved):
            t.copy_(x)

    fresh(0)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for i in range(4):
        fresh(i)
        reset()
        want = step()
        held_after = [t.clone() for t in flat]
        assert (want[-3] > 0).any()
        for g, outs in graphs:
            reset()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            assert all(torch.equal(a, b) for a, b in zip(flat, held_after))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "kv8", "fp32"])
def test_a_run_of_tree_steps(cuda, fmt):
    """Steps as an engine makes them: write a tree's K / V behind the committed prefix, attend, accept, compact, move
    the length, and attend the next token over the compacted cache; against the 64-bit forms on a dense cache."""
    lsk = _lsk()
    Hq, Hkv, D, S, B = 4, 2, 64, 256, 3
    dt = F32 if fmt == "fp32" else BF16
    g = _gen(3)
    if fmt == "kv8":
        cache = lsk.KV8.zeros(B, Hkv, S, D, cuda, layers=1)
        plan_cache = cache.layer(0)
    else:
        shape = (1, B, Hkv, S // 32, D // 16, 64, 8) if fmt == "bf16" else (1, B, Hkv, S, D)
        kc = torch.zeros(shape, dtype=dt, device=cuda)
        vc = torch.zeros(1, B, Hkv, S // 32, D, 32, dtype=dt, device=cuda)
        plan_cache = kc[0]
    kd, vd = (torch.zeros(B, Hkv, S, D, dtype=torch.float64) for _ in range(2))
    kv_len = torch.zeros(B, dtype=torch.int64, device=cuda)
    length = [0] * B
    rng = np.random.default_rng(8)
    for step in range(5):
        sizes = [40, 20, 33] if step == 0 else [int(rng.integers(1, 30)) for _ in range(B)]
        parents, tokens, y = _forest(step, sizes, vocab=2)
        order = rng.permutation(B)
        tab, n = pack_blocks([(int(r), length[r], sizes[r]) for r in order])
        cat = lambda xs, t: _cat([xs[r] for r in order], t, cuda)     # noqa: E731
        k, v = (torch.randn(n, Hkv, D, generator=g).to(dt) for _ in range(2))
        q = torch.randn(n, Hq, D, generator=g).to(dt)
        rows = np.concatenate([[r] * sizes[r] for r in order])
        pos = np.concatenate([length[r] + np.arange(sizes[r]) for r in order])
        starts, lens = _i32([b[0] for b in tab], cuda), _i32([b[2] for b in tab], cuda)
        par = cat(parents, torch.int32)
        mask, _ = lsk.tree_masks(par, starts, lens, max(sizes))
        plan = lsk.AttnPlan(tab, Hq, plan_cache, split=None if step % 2 else 64)
        if fmt == "kv8":
            lsk.kv8_append(k.to(cuda), v.to(cuda), cache.layer(0), _i32(rows, cuda), _i32(pos, cuda))
            got = lsk.kv8_attn(q.to(cuda), cache.layer(0), plan, mask)
            k, v = held(k), held(v)
        else:
            lsk.kv_append(k.to(cuda), v.to(cuda), kc[0], vc[0], _i32(rows, cuda), _i32(pos, cuda))
            got = lsk.tree_attn(q.to(cuda), kc[0], vc[0], plan, mask)
        kd[rows, :, pos], vd[rows, :, pos] = k.double(), v.double()
        sets = [s for r in order for s in ancestors(parents[r])]
        ref, mag, big = attention(q.double(), kd, vd, tab, 1 / math.sqrt(D), sets)
        assert_close_f32(got, ref, mag, S, D, big) if fmt == "fp32" else assert_close_bf16(got, ref, mag)
        acc, path, _ = lsk.tree_accept(cat(y, torch.int64), cat(tokens, torch.int64), par, starts, lens, max(sizes))
        r_t, p_t = _i32(order, cuda), _i32([length[r] for r in order], cuda)
        if fmt == "kv8":
            lsk.kv8_compact(cache, r_t, p_t, acc, path)
        else:
            lsk.kv_compact(kc, vc, r_t, p_t, acc, path)
        lsk.kv_rollback(kv_len, r_t, acc, B)
        for i, r in enumerate(order):
            p = accept(parents[r], tokens[r], y[r])
            assert int(acc[i]) == len(p) - 1
            src = [length[r] + j for j in p]
            kd[r, :, length[r]:length[r] + len(p)] = kd[r][:, src].clone()
            vd[r, :, length[r]:length[r] + len(p)] = vd[r][:, src].clone()
            length[r] += len(p)
        assert kv_len.cpu().tolist() == length


# ----------------------------------------------------------------------------- refusals (no GPU needed)

def test_entry_points_refuse_bad_arguments():
    lib = _lsk().load()
    P = 16
    a = lib.lsk_kv8_append
    ok = [1, P, P, 128, 64, P, P, P, P, P, P, 4, 2, 64, 3, 128, None]
    bad = lambda i, x: a(*(ok[:i] + [x] + ok[i + 1:]))                # noqa: E731
    for i in (1, 2, 5, 6, 7, 8, 9, 10):
        assert bad(i, None) == -1
    assert bad(0, 7) == -3 and bad(13, 96) == -3 and bad(15, 96) == -2 and bad(11, -1) == -2 and bad(3, -1) == -2
    assert bad(5, 24) == -1 and bad(14, 0) == -2                      # a cache off 16 bytes; no rows
    assert bad(11, 0) == 0                                            # no tokens: no launch
    r = lib.lsk_kv8_read
    assert r(1, P, P, P, P, P, P, P, None, 4, 2, 64, 3, 128, None) == -1
    assert r(1, P, P, P, P, P, P, P, P, 4, 2, 32, 3, 128, None) == -3
    assert r(1, P, P, P, P, P, P, P, P, 0, 2, 64, 3, 128, None) == 0
    # q, strides, k8, v8, exponents, mask, words | groups, n_groups, n_parts, recs, rounds, slots, shared, tiles, row
    # groups, part rows | out, heads, KV heads, D, S, scale, workspace, bytes, stream
    ok = [P, 512, 64, P, P, P, P, None, 0, None, 0, 0, P, 1, 1, 0, 1, 1, 16, P, 8, 2, 64, 128, 0.125, None, 0, None]
    k8 = lambda **kw: lib.lsk_kv8_attn(*[kw.get(f"a{i}", x) for i, x in enumerate(ok)])  # noqa: E731
    assert k8(a0=None) == -1 and k8(a5=None) == -1 and k8(a12=None) == -1 and k8(a7=P) == -1 and k8(a19=None) == -1
    assert k8(a16=4) == -1 and k8(a16=3, a22=128) == -1 and k8(a16=3, a7=P, a8=1) == -1 and k8(a17=2) == -1
    assert k8(a15=1) == -1 and k8(a15=-1) == -1 and k8(a24=-0.5) == -1 and k8(a24=math.nan) == -1
    assert k8(a14=0) == -1 and k8(a10=1) == -1 and k8(a13=-1) == -1
    assert k8(a20=7) == -2 and k8(a23=96) == -2 and k8(a22=32) == -3 and k8(a3=24) == -1 and k8(a1=-1) == -2
    assert k8(a10=1, a11=3) == -4 and k8(a10=1, a11=3, a9=P, a25=P, a26=100) == -4   # partials without their workspace
    assert k8(a10=1, a11=3, a9=P, a25=P, a26=1 << 20, a18=8) == -1                   # rows per partial below a tile
    assert k8(a23=1 << 25) == -2                                                     # a stripe of 2 GiB and more
    assert k8(a13=0) == 0
    ok2 = [1, P, 512, 64, P, P, P, 1, None, 0, 0, None, 0, 0, P, 1, 1, 0, 1, 1, 16, P, 8, 2, 64, 128, 0.125, None, 0,
           None]
    tr = lambda **kw: lib.lsk_tree_attn(*[kw.get(f"a{i}", x) for i, x in enumerate(ok2)])  # noqa: E731
    assert tr(a6=None) == -1 and tr(a7=0) == -1 and tr(a0=2) == -3 and tr(a14=None) == -1 and tr(a24=96) == -3
    assert tr(a0=0) == -1 and tr(a0=0, a9=1, a10=16) == -1 and tr(a0=0, a9=1, a10=24, a8=P) == -1
    assert tr(a0=0, a9=1, a10=16, a8=P, a24=80) == -3 and tr(a0=0, a10=16) == 0 and tr(a15=0) == 0
    cnt = (ctypes.c_long * 9)()
    blk = (ctypes.c_int32 * 4)(0, 700, 40, 0)
    plan = lambda **kw: lib.lsk_cache_attn_plan(*[kw.get(f"a{i}", x) for i, x in enumerate(  # noqa: E731
        [blk, 1, 4, 256, 2, 2, 128, 1, 1, 4, 256, None, 0, cnt])])
    assert plan() == 0 and list(cnt)[:3] == [40, 2, 6] and cnt[4] == 2 and cnt[7] == 4 and cnt[8] == 12
    assert plan(a9=0) == 0 and cnt[7] == 1 and plan(a9=0, a4=300) == 0 and cnt[7] == 4     # 2 x 2 x 5 tiles; 600 x 5
    assert plan(a9=8) == -2 and plan(a4=0) == -2 and plan(a8=0) == 0 and cnt[7] == 1
    assert plan(a3=100) == -2 and plan(a9=3) == -2 and plan(a6=96) == -3 and plan(a0=None) == -1
    assert plan(a13=None) == -1
    assert plan(a11=blk, a12=4) == -4 and plan(a1=0) == 0 and cnt[3] == cnt[8] == 0
    blk[2] = 1 << 20
    assert plan(a5=1 << 18) == -2 and plan(a10=1 << 30) == -2                        # more items than a plan holds
    blk[2] = 40
    blk[1] = 64 * 128
    assert plan(a3=64) == -2                                                         # more than 128 splits
    blk[1] = -1
    assert plan() == -2
    m = lib.lsk_tree_masks
    assert m(None, P, P, 1, 4, 4, P, 1, None, None) == -1 and m(P, P, P, 1, 4, 33, P, 1, None, None) == -2
    assert m(P, P, P, 0, 4, 4, P, 1, None, None) == 0 and m(P, P, P, 1, 0, 4, P, 1, None, None) == 0
    t = lib.lsk_tree_accept
    assert t(P, P, P, P, None, 1, 4, 4, P, P, P, None) == -1 and t(P, P, P, P, P, 1, 4, 0, P, P, P, None) == -2
    assert t(P, P, P, P, P, 0, 4, 4, P, P, P, None) == 0
    c = lib.lsk_kv_compact
    assert c(1, None, P, None, None, 1, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == -1
    assert c(2, P, P, None, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == -1
    assert c(3, P, P, P, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == -3
    assert c(1, P, P, None, None, 1, P, P, P, P, 1, 4, 2, 32, 3, 128, None) == -3
    assert c(2, P, P, P, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 96, None) == -2
    assert c(1, P, P, None, None, 0, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == 0


def test_the_planner_refuses_rows_outside_the_cache():
    """A launch takes a block's cache row and first token from the plan: the planner refuses what lies outside."""
    lib = _lsk().load()
    cnt = (ctypes.c_long * 9)()
    for kv8, tree in ((1, 0), (1, 1), (0, 1)):
        for q_start, row, T, want in ((0, 0, 3, 0), (7, 1, 3, 0), (0, 2, 3, -2), (0, -1, 3, -2), (-1, 0, 3, -2),
                                      (0, 1 << 30, 3, -2), ((1 << 31) - 3, 0, 3, -2), (-1, -1, 0, 0)):
            blk = (ctypes.c_int32 * 8)(0, 5, 0, 0, q_start, 40, T, row)
            assert lib.lsk_cache_attn_plan(blk, 2, 4, 256, 2, 2, 128, kv8, tree, 0, 256, None, 0, cnt) == want


def test_plans_refuse_blocks_outside_the_cache():
    lsk = _lsk()
    cache = lsk.KV8.zeros(2, 2, 128, 64, "cpu")
    plan = lsk.AttnPlan([(0, 3, 2, 1), (2, 0, 0, 0), (2, 127, 1, 0)], 4, cache)
    assert plan.n_tokens == 3 and plan.causal.n_items > 0 and plan.tree.n_items > 0 and plan.split == 512
    for b in ([(0, 3, 2, 2)], [(0, 3, 2, -1)], [(0, 127, 2, 0)], [(0, -1, 2, 0)], [(1, 0, 2, 0)], [(0, 0, -1, 0)]):
        with pytest.raises(ValueError):
            lsk.AttnPlan(b, 4, cache)
    with pytest.raises(ValueError):
        lsk.AttnPlan([(0, 0, 1, 0)], 3, cache)
    with pytest.raises(ValueError):
        lsk.AttnPlan([(0, 0, 1, 0)], 4, cache, split=100)
    with pytest.raises(ValueError):
        lsk.KV8.zeros(2, 2, 100, 64, "cpu")
    with pytest.raises(ValueError):
        lsk.KV8.zeros(2, 2, 128, 96, "cpu")
    assert lsk.AttnPlan([], 4, cache).causal.n_rounds == 0
    assert lsk.AttnPlan([], 4, cache, tree=True).causal is None and lsk.AttnPlan([], 4, cache, tree=False).tree is None
    with pytest.raises(lsk.LskError):
        lsk.AttnPlan([(0, 0, 1, 0)], 4, cache, row_groups=3)
    for b, s in ((1, 131072), (256, 8192), (32, 2048), (3, 64)):
        split = lsk.cache_attn_split(b, 8, s)
        assert split % 64 == 0 and 512 <= split <= 8192 and split * 128 >= s


def _items(plan, launch):
    """(row group rows, wave rows) of every work item of a plan: [(q_start, row0, nrows, groups, kvh, lo, hi, part)]"""
    one = launch.n_slots * launch.n_rounds * 8
    recs = launch.recs.numpy()[:one].reshape(launch.n_slots, launch.n_rounds, 8)
    shared = launch.recs.numpy()[one:].reshape(launch.n_shared, 8)     # items of four row groups
    assert all(r[2] >> 10 & 3 == 2 for r in shared)
    out = [(r[0], r[1], r[2] & 1023, 1 << (r[2] >> 10 & 3), r[2] >> 12, r[3], r[4], r[5]) for r in shared]
    for slot in recs:
        live = [r for r in slot if r[2] & 1023]
        assert all((r[2] & 1023) == 0 for r in slot[len(live):])      # a slot's items come first
        assert all(r[2] >> 10 & 3 < 2 for r in live)
        out += [(r[0], r[1], r[2] & 1023, 1 << (r[2] >> 10 & 3), r[2] >> 12, r[3], r[4], r[5]) for r in live]
    return out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("G,split,T_hi", [(4, 256, 9), (1, 64, 70), (8, 8192, 40), (3, 128, 130), (4, 512, 1)])
def test_cache_attention_plans_cover_every_row_and_position_once(G, split, T_hi, tree, D):
    lsk = _lsk()
    rng = np.random.default_rng(T_hi)
    B, Hkv, S = 6, 3, 1024
    cache = lsk.KV8.zeros(B, Hkv, S, D, "cpu")
    blocks = [(r, int(rng.integers(0, S - T_hi)), int(rng.integers(0, T_hi + 1))) for r in range(B)]
    tab, n = pack_blocks(blocks)
    plan = lsk.AttnPlan(tab, G * Hkv, cache, split=split, row_groups=4, tree=tree)
    p = plan.tree if tree else plan.causal
    items = _items(plan, p)
    most = max(t for _, _, t in blocks) * G
    assert p.tiles == (1 if most <= 16 else 2 if most <= 32 or tree or D == 128 else 3)
    parts = [i for i in items if i[7] >= 0]
    assert len({(i[4], i[7]) for i in parts}) == len(parts) == p.n_parts * Hkv
    groups = {tuple(g[:5]) for g in p.groups.numpy().reshape(-1, 8)}
    for (q0, p0, t, row) in tab:
        rows = t * G
        want = 1
        while tree and want < 4 and rows > 32 * want:
            want *= 2
        mine = [i for i in items if i[0] == q0] if t else []
        for h in range(Hkv):
            covered = np.zeros((rows, S + 1), dtype=int)
            for (_, r0, nr, g, kvh, lo, hi, part) in mine:
                if kvh == h:
                    assert g == want and nr <= 16 * p.tiles * g and lo % split == 0
                    covered[r0:r0 + nr, lo:hi] += 1
            for r in range(rows):
                assert (covered[r, :p0 + r // G + 1] == 1).all()      # what the causal rule lets the row read
        for (_, r0, nr, g, kvh, lo, hi, part) in mine:
            ns = -(-(p0 + (r0 + nr - 1) // G + 1) // split)
            assert (part >= 0) == (ns > 1)
            if part >= 0:
                assert (q0, r0, nr, part - lo // split, ns) in groups and nr <= p.part_rows


def test_wrappers_refuse_tensors_off_the_gpu():
    lsk = _lsk()
    cache = lsk.KV8.zeros(1, 1, 64, 64, "cpu")
    x, i = torch.zeros(1, 1, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    plan = lsk.AttnPlan([(0, 0, 1, 0)], 1, cache)
    for f in (lambda: lsk.kv8_append(x, x, cache, i, i), lambda: lsk.kv8_read(cache, i, i),
              lambda: lsk.kv8_attn(x, cache, plan), lambda: lsk.tree_masks(i, i, i, 1)):
        with pytest.raises(lsk.LskError):
            f()


@pytest.mark.gpu
def test_wrappers_refuse_what_does_not_fit(cuda):
    lsk = _lsk()
    cache = lsk.KV8.zeros(2, 2, 128, 64, cuda)
    x, i = torch.zeros(3, 2, 64, dtype=BF16, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    plan = lsk.AttnPlan([(0, 0, 3, 0)], 4, cache)
    q = torch.zeros(3, 4, 64, dtype=BF16, device=cuda)
    m = torch.zeros(3, 1, dtype=torch.int32, device=cuda)
    kf = torch.zeros(2, 2, 4, 4, 64, 8, dtype=BF16, device=cuda)
    vf = torch.zeros(2, 2, 4, 64, 32, dtype=BF16, device=cuda)
    pt = lsk.AttnPlan([(0, 0, 3, 0)], 4, kf)
    big = lsk.KV8.zeros(2, 2, 192, 64, cuda)
    a = torch.zeros(1, dtype=torch.int64, device=cuda)
    calls = [lambda: lsk.kv8_append(x.half(), x.half(), cache, i, i), lambda: lsk.kv8_append(x, x[:2], cache, i, i),
             lambda: lsk.kv8_append(x, x, cache, i.long(), i), lambda: lsk.kv8_append(x, x, cache, i[:2], i),
             lambda: lsk.kv8_append(x.transpose(0, 2).contiguous().transpose(0, 2), x, cache, i, i),
             lambda: lsk.kv8_append(x, x, cache._replace(ks=cache.ks[:1]), i, i),
             lambda: lsk.kv8_append(x.cpu(), x, cache, i, i), lambda: lsk.kv8_read(cache, i, i, torch.float16),
             lambda: lsk.kv8_attn(q, big, plan), lambda: lsk.kv8_attn(q[:2], cache, plan),
             lambda: lsk.kv8_attn(q.float(), cache, plan), lambda: lsk.kv8_attn(q, cache, pt),
             lambda: lsk.kv8_attn(q, cache, plan, m[:2]), lambda: lsk.kv8_attn(q, cache, plan, m.long()),
             lambda: lsk.kv8_attn(q, cache, plan, out=torch.zeros(3, 128, dtype=BF16, device=cuda)),
             lambda: lsk.tree_attn(q, kf, vf, plan, m), lambda: lsk.tree_attn(q, kf, vf[:, :1], pt, m),
             lambda: lsk.tree_attn(q, kf, vf, pt, m.cpu()),
             lambda: lsk.kv_compact(kf, vf, i[:1], i[:1], a, m[:1]),
             lambda: lsk.kv_compact(kf[None], vf[None], i[:1], i[:1], a[:0], m[:1]),
             lambda: lsk.kv8_compact(cache, i[:1], i[:1], a, m[:1]), lambda: lsk.kv8_read(cache, i, i, out=(x,)),
             lambda: lsk.kv8_attn(q, cache, plan, workspace=torch.zeros(8, 2, device=cuda)[:, 0]),
             lambda: lsk.kv8_attn(q, cache, plan, scale=-1.0),
             lambda: lsk.tree_accept(a, a, i, i[:1], i[:1], 1)]
    for f in calls:
        with pytest.raises(lsk.LskError):
            f()
    assert lsk.kv8_attn(q[:0], cache, lsk.AttnPlan([], 4, cache)).shape == (0, 256)
    k, v = lsk.kv8_read(cache, i[:0], i[:0])
    assert k.shape == v.shape == (0, 2, 64)
