"""The 4-bit KV cache (write, read, attention, compaction), the norms of queries and keys with their rotation, and the
8-bit integer projections, against plain 64-bit implementations; a layer made of them; refusals on the CPU.

Tolerances.  The cache, the integer codes and their scales: exact.  Attention: as over the 8-bit cache (test_cache_ops),
whose roundings it shares.  Norms: the sum of D squares in fp32 (D adds, at most (D + 2) 2^-24 relative, halved by the
root), the root and four products with at most 2^-22 together, the rotation's two products and their sum 3 * 2^-24 of
|y1 c| + |y2 s|; then the output's rounding.  Products: the exact integer sum is rounded to fp32 and scaled twice (3 *
2^-24 relative); the residual's sum adds 2^-24 of |y| + |r|; silu in fp32 at most 2^-20 relative (its exponential is good
to 2^-22, the sum and the quotient add 2^-23) plus the argument's own error, which its slope (below 1.1) passes on; then
the output's rounding, eps / 2 of its type."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_cache_ops import (BF16, BLOCKS, F32, _cat, _gen, _heads, _i32, _items, _lsk, accept, ancestors,
                            assert_close_bf16, attention, pack_blocks, random_tree, words_of)

HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}             # eps / 2


# ----------------------------------------------------------------------------- the 4-bit cache's definition

def exponents(x):
    """e of 32 dims x [.., 32] (64 bits): the smallest integer >= -125 with amax <= 7 * 2^e; amax = 0: 0."""
    a = x.abs().amax(-1).double()
    m, e = torch.frexp(torch.where(a > 0, a, 7.0) / 7.0)
    e = (e - (m == 0.5).int()).clamp(min=-125)
    assert (a <= 7.0 * torch.exp2(e.double())).all()
    return torch.where(a > 0, e, torch.zeros_like(e)).to(torch.int64)


def held(x):
    """What the 4-bit cache stands for (64 bits), vectors x [.., d]."""
    x = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(bad, torch.zeros_like(x), x)
    e = exponents(x)[..., None]
    y = x / torch.exp2(e.double())
    unit = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    top = torch.where(e == 126, 3.0, 6.0).double()
    r = (torch.round(y / unit) * unit).clamp(-top, top) * torch.exp2(e.double())
    return torch.where(bad, torch.full_like(r, math.nan), r).flatten(-2)


def codes_of(x):
    """(codes [.., d], biased exponents [.., d / 32]) of vectors without a sign on zeros."""
    h = held(x).unflatten(-1, (-1, 32))
    bad = torch.isnan(h).any(-1)
    e = exponents(torch.where(bad[..., None], torch.zeros_like(h), x.double().unflatten(-1, (-1, 32))))
    y = h / torch.exp2(e.double())[..., None]
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    c = torch.searchsorted(table, y.abs().nan_to_num(0).contiguous()) | ((y < 0).long() << 3)
    return c.flatten(-2).to(torch.uint8), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def dense4(cache):
    """Codes [B, H, S, D] and biased exponents [B, H, S, D / 32] of K and of V, index by index from the layout."""
    k, v, ks, vs = (t.cpu() for t in cache)
    B, H, nb, nd = vs.shape[:4]
    S, D = nb * 64, nd * 32
    p, d = np.meshgrid(np.arange(S), np.arange(D), indexing="ij")
    q, a, r, blk, b = p % 64 // 16, p % 16 // 4, p % 4, p // 64, d // 32
    lane = d // (D // 4) * 16 + 4 * q + r
    byte = d % 32 // 2 if D == 128 else a % 2 * 8 + d % 16 // 2
    frag = a if D == 128 else a // 2
    t = lambda x: torch.as_tensor(x)                  # noqa: E731
    kc = k[:, :, t(blk), t(frag), t(lane), t(byte)] >> t(4 * (d % 2)).to(torch.uint8) & 15
    lane, byte = p % 64 // 16 * 16 + d % 16, d % 32 // 16 * 8 + p % 16 // 2
    vc = v[:, :, t(blk), t(b), t(lane), t(byte)] >> t(4 * (p % 2)).to(torch.uint8) & 15
    one = (slice(None), slice(None), t(blk[:, ::32]), t(b[:, ::32]))
    ke = ks[(*one, t((4 * q + r)[:, ::32]), t(a[:, ::32]))]
    ve = vs[(*one, t(p[:, ::32] % 64))]
    return kc, ke, vc, ve


def kv4_from(lsk, cuda, k, v):
    """A 4-bit cache written by kv4_append with dense k, v [B, Hkv, S, D]."""
    B, H, S, D = k.shape
    cache = lsk.KV4.zeros(B, H, S, D, cuda)
    flat = lambda x: x.permute(0, 2, 1, 3).reshape(B * S, H, D).contiguous().to(cuda)  # noqa: E731
    lsk.kv4_append(flat(k), flat(v), cache, _i32(torch.arange(B).repeat_interleave(S), cuda),
                   _i32(torch.arange(S).repeat(B), cuda))
    return cache


def _awkward(g, n, h, d, dtype):
    """Vectors of every size: zeros, tiny, subnormal, huge, with the largest value at and next to 7 * 2^e, ties."""
    x = torch.randn(n, h, d, generator=g) * torch.exp2(torch.randint(-30, 30, (n, h, 1), generator=g).float())
    flat = x.view(-1, d)
    m = flat.shape[0]
    flat[0] = 0.0
    flat[1 % m] = torch.randn(d, generator=g) * 1e-39
    flat[2 % m] = torch.randn(d, generator=g).clamp(-1, 1) * 3e38
    flat[3 % m] = (torch.arange(d).float() % 29 - 14) / 4              # ties between e2m1 values, +-3.5: half of 7
    flat[4 % m] = (torch.arange(d).float() % 29 - 14) / 2              # the largest value is 7
    flat[5 % m] = (torch.arange(d).float() % 29 - 14) / 2
    flat[5 % m, ::32] = 7.0625                                        # and just past it: the next scale
    flat[6 % m] = 0.0
    flat[6 % m, d - 1] = -2.0 ** -133
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,h", [(1, 1), (7, 3), (16, 8), (33, 2), (200, 8), (300, 1)])
def test_kv4_append_and_read_are_exact(cuda, dtype, D, n, h):
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
    cache = lsk.KV4.zeros(B, h, S, D, cuda)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    want = dense4(cache)
    lsk.kv4_append(k.to(cuda), v.to(cuda), cache, _i32(rows, cuda), _i32(pos, cuda))
    for x, codes, exps in ((k, want[0], want[1]), (v, want[2], want[3])):
        c, e = codes_of(x)
        codes[rows[ok], :, pos[ok]] = c[ok]
        exps[rows[ok], :, pos[ok]] = e[ok]
    neg0 = lambda t: torch.where(t == 8, torch.zeros_like(t), t)      # noqa: E731  (the sign of a zero is free)
    for got, w in zip(dense4(cache), want):
        assert torch.equal(got, w) if w.shape[-1] < 32 else torch.equal(neg0(got), neg0(w))
    for out in (BF16, F32):
        kr, vr = lsk.kv4_read(cache, _i32(rows, cuda), _i32(pos, cuda), out)
        for got, x in ((kr, k), (vr, v)):
            assert torch.equal(got.cpu().double(), torch.where(ok[:, None, None], held(x), 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_runs_of_positions_from_any_start(cuda, D):
    """Prompts from any position, next to each other, across 64-position blocks and up to the cache's end, between
    single tokens: every token's values, and nothing of its neighbours, which share its bytes."""
    lsk = _lsk()
    g = _gen(31)
    B, h, S = 7, 2, 256
    runs = [(0, 1, 16), (1, 2, 33), (2, 57, 31), (2, 88, 40), (3, 240, 16), (4, 3, 1), (0, 61, 5), (5, 255, 1),
            (5, 0, 96), (4, 130, 29), (6, 5, 250)]
    rows = torch.cat([torch.full((n,), r) for (r, _, n) in runs])
    pos = torch.cat([torch.arange(p, p + n) for (_, p, n) in runs])
    for order in ("as they are", "shifted", "shuffled"):
        if order == "shifted":                        # (the workgroups hold other runs)
            rows, pos = rows.roll(3), pos.roll(3)
        elif order == "shuffled":
            perm = torch.randperm(len(rows), generator=g)
            rows, pos = rows[perm], pos[perm]
        n = len(rows)
        k, v = (torch.randn(n, h, D, generator=g).to(BF16) for _ in range(2))
        cache = lsk.KV4.zeros(B, h, S, D, cuda)
        for x in (cache.k, cache.v):
            x.fill_(0x33)                             # (1.5 everywhere else)
        lsk.kv4_append(k.to(cuda), v.to(cuda), cache, _i32(rows, cuda), _i32(pos, cuda))
        allrows, allpos = torch.arange(B).repeat_interleave(S), torch.arange(S).repeat(B)
        for got, x in zip(lsk.kv4_read(cache, _i32(allrows, cuda), _i32(allpos, cuda), F32), (k, v)):
            want = torch.full((B, S, h, D), 1.5, dtype=torch.float64)
            want[rows, pos] = held(x)
            assert torch.equal(got.cpu().double().view(B, S, h, D), want)
        for got, x in zip(lsk.kv4_read(cache, _i32(rows, cuda), _i32(pos, cuda), F32), (k, v)):
            assert torch.equal(got.cpu().double(), held(x))


@pytest.mark.gpu
def test_kv4_rounds_every_bf16_value_to_the_nearest_code(cuda):
    """All bf16 values up to 7 beside a 7: the nearest e2m1 value, ties to even, at most 6."""
    lsk = _lsk()
    vals = torch.arange(0, 0x40E1, dtype=torch.int32).to(torch.int16).view(BF16)       # 0 .. 7
    n = (len(vals) + 30) // 31
    x = torch.zeros(n, 1, 64, dtype=BF16)
    x[:, 0, 0] = 7.0
    body = torch.zeros(n * 31, dtype=BF16)
    body[:len(vals)] = vals * torch.where(torch.arange(len(vals)) % 2 == 0, 1.0, -1.0).to(BF16)
    x[:, 0, 1:32] = body.view(n, 31)
    S = (n + 63) // 64 * 64
    cache = lsk.KV4.zeros(1, 1, S, 64, cuda)
    rows, pos = _i32(np.zeros(n), cuda), _i32(np.arange(n), cuda)
    lsk.kv4_append(x.to(cuda), x.to(cuda), cache, rows, pos)
    a = x.double().abs()
    want = sum((a > b).double() * s if tie else (a >= b).double() * s
               for b, s, tie in ((.25, .5, 1), (.75, .5, 0), (1.25, .5, 1), (1.75, .5, 0), (2.5, 1., 1), (3.5, 1., 0),
                                 (5., 2., 1))) * torch.sign(x.double())
    for got in lsk.kv4_read(cache, rows, pos, F32):
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.gpu
def test_kv4_append_takes_strides_and_non_finite_values(cuda):
    """k and v as views of a fused qkv row (at any bf16 address); NaN and infinities make their 32 dims NaN."""
    lsk = _lsk()
    g = _gen(5)
    n, h, D, S = 9, 2, 64, 64
    buf = torch.randn(n * 2 * (h * D) + n + 1, generator=g).to(BF16)
    buf[1 + 5], buf[1 + 70], buf[1 + 130 + h * D] = math.nan, math.inf, -math.inf
    dev = buf.to(cuda)
    view = lambda t, o: torch.as_strided(t, (n, h, D), (2 * h * D + 1, D, 1), o)  # noqa: E731
    cache = lsk.KV4.zeros(1, h, S, D, cuda)
    rows, pos = _i32(np.zeros(n), cuda), _i32(np.arange(n), cuda)
    lsk.kv4_append(view(dev, 1), view(dev, 1 + h * D), cache, rows, pos)
    for got, x in zip(lsk.kv4_read(cache, rows, pos, F32), (view(buf, 1), view(buf, 1 + h * D))):
        want = held(x)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().double().nan_to_num(0), want.nan_to_num(0))
    assert torch.isnan(held(view(buf, 1))).sum() == 3 * 32


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_kv4_keeps_the_largest_finite_values_finite(cuda, dtype, D):
    lsk = _lsk()
    top = torch.finfo(dtype).max
    x = torch.randn(5, 2, D, generator=_gen(7)).to(dtype)
    x[0, :, :4] = torch.tensor([top, -top, top / 2, top / 300], dtype=dtype)
    x[1, :, 5], x[2, :, 5] = 3.5 * 2.0 ** 126, 3.25 * 2.0 ** 126
    x[3] = top * torch.linspace(-1, 1, D, dtype=torch.float64).to(dtype)
    cache = lsk.KV4.zeros(1, 2, 64, D, cuda)
    rows, pos = _i32(np.zeros(5), cuda), _i32(np.arange(5), cuda)
    lsk.kv4_append(x.to(cuda), x.flip(0).contiguous().to(cuda), cache, rows, pos)
    want = held(x)
    assert torch.isfinite(want.to(dtype)).all()
    for out in (F32, BF16):
        for got, w in zip(lsk.kv4_read(cache, rows, pos, out), (want, want.flip(0))):
            assert torch.equal(got.double().cpu(), w)


# ----------------------------------------------------------------------------- attention over the 4-bit cache

@pytest.mark.gpu
@pytest.mark.parametrize("split", [64, 256, 8192])
@pytest.mark.parametrize("blocks", sorted(BLOCKS))
@pytest.mark.parametrize("heads", ["gqa128", "gqa64", "mha64", "mqa128"])
def test_kv4_attention(cuda, heads, blocks, split):
    lsk = _lsk()
    Hq, Hkv, D = _heads(heads)
    tab, n = pack_blocks(BLOCKS[blocks])
    S = (max(p + t for (_, p, t) in BLOCKS[blocks]) + 63) // 64 * 64
    B = 1 + max(r for (r, _, _) in BLOCKS[blocks])
    g = _gen(split + n)
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    cache = kv4_from(lsk, cuda, k, v)
    plan = lsk.AttnPlan(tab, Hq, cache, split=split)
    got = lsk.kv4_attn(q.to(cuda), cache, plan)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)
    # a chain's mask gives the causal rule, within the same bounds
    most = max(T for (_, _, T, _) in tab)
    words = words_of([set(range(t + 1)) for (_, _, T, _) in tab for t in range(T)], most // 32 + 1)
    assert_close_bf16(lsk.kv4_attn(q.to(cuda), cache, plan, _i32(words, cuda)), ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("row_groups", [1, 2, 4])
@pytest.mark.parametrize("heads", ["gqa128", "gqa64", "mha64"])
def test_kv4_trees(cuda, heads, row_groups):
    lsk = _lsk()
    Hq, Hkv, D = _heads(heads)
    rng = np.random.default_rng(row_groups)
    blocks = [(2, 0, 33), (0, 70, 64), (1, 130, 13), (3, 64, 1), (4, 257, 100)]
    tab, n = pack_blocks(blocks)
    sets = [s for (_, _, t) in blocks for s in ancestors(random_tree(rng, t))]
    g = _gen(row_groups)
    k, v = (torch.randn(5, Hkv, 384, D, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    cache = kv4_from(lsk, cuda, k, v)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 0.25, sets)
    mask = _i32(words_of(sets, 4), cuda)
    for split in (64, 512):
        plan = lsk.AttnPlan(tab, Hq, cache, split=split, row_groups=row_groups, tree=True)
        assert_close_bf16(lsk.kv4_attn(q.to(cuda), cache, plan, mask, scale=0.25), ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("row_groups", [1, 4])
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_slots_that_are_not_read_never_matter(cuda, D, row_groups):
    """Codes and exponents of every kind, NaN among them, in slots behind a row's and beside its ancestors; a NaN that
    is read reaches the rows that read it (V: in its 32 dims); rows that read nothing are zeros."""
    lsk = _lsk()
    g = _gen(D)
    Hq, Hkv, S = 8, 2, 256
    blocks = [(0, 0, 40), (1, 100, 33), (2, 130, 3)]
    tab, n = pack_blocks(blocks)
    rng = np.random.default_rng(3)
    sets = [s for (_, _, t) in blocks for s in ancestors(random_tree(rng, t))]
    sets[0], sets[4] = frozenset(), frozenset()       # (block 0 has no prefix: these rows read nothing)
    for i in range(40):
        sets[i] = sets[i] - {7}                       # nobody of block 0 reads its node 7
    k, v = (torch.randn(3, Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    k[1, 0, 60, 3] = math.nan                         # in the prefix: every row of the block, KV head 0
    v[1, 1, 70, D - 1] = math.inf                     # the last 32 dims of KV head 1's rows
    k[2, 1, 131, 0] = -math.inf                       # node 1 of block 2
    v[2, 0, 132, 1] = math.nan                        # node 2 of it
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    cache = kv4_from(lsk, cuda, k, v)
    # what no row reads: node 7 of block 0 and everything behind the blocks
    for t, fill in ((cache.k, 0xF7), (cache.v, 0x7F)):
        t[:, :, 3:] = fill
    cache.ks[:, :, 3:], cache.vs[:, :, 3:] = 255, 255
    cache.vs[0, :, 0, :, 7], cache.vs[0, :, 0, :, 40:] = 255, 255
    cache.ks[0, :, 0, :, 3, 1] = 255                  # ([4 q + r][a] of position 7)
    cache.ks[0, :, 0, :, 8:12, 2:], cache.ks[0, :, 0, :, 12:] = 255, 255          # positions 40 .. 63
    fresh = kv4_from(lsk, cuda, k, v)
    kd, vd = held(k), held(v)
    ref, mag, _ = attention(q.double(), kd, vd, tab, 1 / math.sqrt(D), sets)
    plan = lsk.AttnPlan(tab, Hq, cache, row_groups=row_groups, tree=True)
    got = lsk.kv4_attn(q.to(cuda), cache, plan, _i32(words_of(sets, 2), cuda))
    assert_close_bf16(got, ref, mag)
    assert (got[0] == 0).all() and (got[4] == 0).all() and torch.isnan(got).any()
    causal = lsk.AttnPlan([(0, 0, 41, 0), (41, 190, 1, 1), (42, 130, 2, 2)], Hq, fresh, tree=False)
    q2 = torch.randn(44, Hq, D, generator=g).to(BF16)
    ref, mag, _ = attention(q2.double(), kd, vd, [(0, 0, 41, 0), (41, 190, 1, 1), (42, 130, 2, 2)], 1 / math.sqrt(D))
    assert_close_bf16(lsk.kv4_attn(q2.to(cuda), fresh, causal), ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_of_large_and_small_scales(cuda, D):
    """K and V whose 32-dim scales differ by far, contexts over 128 splits, prompts of several hundred tokens."""
    lsk = _lsk()
    g = _gen(11)
    S = 8192
    k = torch.randn(2, 1, S, D, generator=g) * torch.exp2(torch.randint(-3, 2, (2, 1, S, D // 32), generator=g).float()
                                                          ).repeat_interleave(32, -1)
    v = torch.randn(2, 1, S, D, generator=g) * torch.exp2(torch.randint(-40, 40, (2, 1, 1, D // 32), generator=g).float()
                                                          ).repeat_interleave(32, -1)
    k, v = k.to(BF16), v.to(BF16)
    cache = kv4_from(lsk, cuda, k, v)
    for tab, split in ([(0, 8100, 3, 0), (3, 8191, 1, 1)], 64), ([(0, 1, 300, 0), (300, 77, 201, 1)], None):
        n = tab[-1][0] + tab[-1][2]
        q = torch.randn(n, 4, D, generator=g).to(BF16)
        got = lsk.kv4_attn(q.to(cuda), cache, lsk.AttnPlan(tab, 4, cache, split=split, tree=False))
        ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
        assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens", [(20, 33, 47, 17, 2), (12, 11, 9, 10, 2)])
def test_kv4_attention_of_prompt_pieces_in_a_large_cache(cuda, tokens, D):
    """Items of 128 rows (of 33 to 48), one of them in two splits, beside a block of few rows; NaN everywhere behind the
    blocks, NaN and infinities in slots and a query that some rows read; a row's bits do not depend on the rest of the
    launch."""
    lsk = _lsk()
    g = _gen(D + 1)
    B, Hkv, Hq, S = 100, 8, 32, 4288
    real = [99, 3, 50, 51, 0]
    blocks = [(r, p0, t) for r, (p0, t) in enumerate(zip((4200, 0, 31, 60, 5), tokens))]       # 800 stripes
    tab, n = pack_blocks(blocks)
    k, v = (torch.randn(len(real), Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    k[1, 0, 20, 5], k[2, 3, 60, D - 1], v[1, 2, 32, 0], v[3, 7, 10, D - 1] = math.nan, math.inf, -math.inf, math.nan
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    q[30] *= 2.0 ** 40                                # (the scale of 32 of its dims; one position takes all)
    q[31, :, :32] *= 2.0 ** -60
    q[32, 4, 7], q[33, 5, 40] = math.inf, math.nan
    q[34] = 0
    cache = lsk.KV4.zeros(B, Hkv, S, D, cuda)
    for t, fill in zip(cache, (0xF7, 0x7F, 255, 255)):
        t.fill_(fill)
    for (r, p0, t) in blocks:
        m = p0 + t
        lsk.kv4_append(k[r, :, :m].transpose(0, 1).to(cuda), v[r, :, :m].transpose(0, 1).to(cuda), cache,
                       _i32(np.full(m, real[r]), cuda), _i32(np.arange(m), cuda))
    where = [(a, b, c, real[r]) for (a, b, c, r) in tab]
    wide = tokens[0] == 20
    split = 64 if wide else 2112
    plan = lsk.AttnPlan(where, Hq, cache, split=split, tree=False)
    if wide:                                          # (few items of 128 dims: 64 rows each)
        assert plan.causal.n_shared == (2 * 2 + 3 + 3 + 2 if D == 128 else 2 * 1 + 2 + 2 + 1) * Hkv
    assert plan.causal.n_parts == (4 if wide and D == 128 else 2)
    assert plan.causal.row_groups == (2 if D == 128 else 4 if wide else 1)
    got = lsk.kv4_attn(q.to(cuda), cache, plan)
    ref, mag, _ = attention(q.double(), held(k), held(v), tab, 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)
    for i, (qs, p0, T, row) in enumerate(where):
        alone = lsk.AttnPlan([(0, p0, T, row)], Hq, cache, split=split, tree=False)
        one = lsk.kv4_attn(q[qs:qs + T].to(cuda), cache, alone)
        assert torch.equal(one.view(torch.int16), got[qs:qs + T].view(torch.int16))


@pytest.mark.gpu
def test_kv4_attention_of_many_prompt_pieces(cuda):
    """More pieces than CUs: items of 128 rows, whose rows have the bits of those in items of 64."""
    lsk = _lsk()
    g = _gen(17)
    B, Hkv, Hq, S, D, n_blocks = 100, 8, 32, 128, 128, 40
    tab, n = pack_blocks([((7 * i) % B, (11 * i) % 60, 17 + i % 3) for i in range(n_blocks)])
    k, v = (torch.randn(B, Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    cache = kv4_from(lsk, cuda, k, v)
    plan = lsk.AttnPlan(tab, Hq, cache, tree=False)
    assert plan.causal.row_groups == 4 and plan.causal.n_shared == n_blocks * Hkv
    got = lsk.kv4_attn(q.to(cuda), cache, plan)
    few = tab[:9] + tab[-2:]
    ref, mag, _ = attention(q.double(), held(k), held(v), few, 1 / math.sqrt(D))
    rows = torch.cat([torch.arange(qs, qs + T) for (qs, _, T, _) in few])
    assert_close_bf16(got[rows.to(cuda)], ref[rows], mag[rows])
    for (qs, p0, T, row) in tab:
        alone = lsk.AttnPlan([(0, p0, T, row)], Hq, cache, tree=False)
        assert alone.causal.row_groups == 2
        assert torch.equal(lsk.kv4_attn(q[qs:qs + T].to(cuda), cache, alone), got[qs:qs + T])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("G,split", [(4, 64), (1, 512), (8, 8192), (3, 4160)])
def test_kv4_plans_cover_every_row_and_position_once(G, split, tree, D):
    lsk = _lsk()
    rng = np.random.default_rng(G)
    B, Hkv, S = 90, 3, 8192
    cache = lsk.KV4.zeros(1, 1, 64, D, "cpu")
    cache = lsk.KV4(*(t.expand(B, Hkv, S // 64, *t.shape[3:]) for t in cache))
    blocks = [(r, int(rng.integers(0, S - 400)), int(t)) for r, t in enumerate((400, 1, 64 // G, 65, 0, 200, 130))]
    tab, _ = pack_blocks(blocks)
    plan = lsk.AttnPlan(tab, G * Hkv, cache, split=split, tree=tree)
    p = plan.tree if tree else plan.causal
    items, seen = _items(p, p), []
    for (q0, p0, t, _) in tab:
        wide = not tree and t * G > (48 if D == 128 else 64) and B * Hkv * -(-t * G // 32) > (768 if D == 128 else 1280)
        two = D == 128 and not wide and -(-t * G // 48) < -(-t * G // 32) and B * Hkv * -(-t * G // 32) > 512
        covered = np.zeros((Hkv, t * G, S), dtype=np.int8)
        for (_, r0, nr, g, h, lo, hi, part) in (i for i in items if i[0] == q0 and t):
            assert tree or (g == (4 if wide else 2 if two else 1) and nr <= (128 if wide else 48))
            assert nr <= 32 * g or not tree and g < 4 and nr <= 48
            assert part < 0 or nr <= p.part_rows
            assert lo % (max(split, 4096) if wide else split) == 0
            assert (part >= 0) == (p0 + (r0 + nr - 1) // G + 1 > (max(split, 4096) if wide else split))
            covered[h, r0:r0 + nr, lo:hi] += 1
            seen += [(h, part)] if part >= 0 else []
        for r in range(t * G):
            assert (covered[:, r, :p0 + r // G + 1] == 1).all()
    assert len(set(seen)) == len(seen) == p.n_parts * Hkv


@pytest.mark.gpu
def test_kv4_attention_strides_streams_batches_and_graphs(cuda):
    """q as a view of fused rows; a row's bits do not depend on the batch; another stream; replays of a captured graph
    between eager calls."""
    lsk = _lsk()
    g = _gen(21)
    Hq, Hkv, D, S = 8, 2, 128, 1024
    blocks = [(r, int(p), int(t)) for r, (p, t) in enumerate([(0, 1), (500, 5), (1000, 9), (63, 33), (700, 1)])]
    tab, n = pack_blocks(blocks)
    k, v = (torch.randn(5, Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    cache = kv4_from(lsk, cuda, k, v)
    fused = torch.randn(n, Hq * D + 3, generator=g).to(BF16).to(cuda)
    q = torch.as_strided(fused, (n, Hq, D), (Hq * D + 3, D, 1), 1)
    plan = lsk.AttnPlan(tab, Hq, cache, split=256, tree=False)
    want = lsk.kv4_attn(q.contiguous(), cache, plan)
    assert torch.equal(lsk.kv4_attn(q, cache, plan), want)
    for (qs, p0, T, row) in tab:
        alone = lsk.kv4_attn(q[qs:qs + T], cache, lsk.AttnPlan([(0, p0, T, row)], Hq, cache, split=256, tree=False))
        assert torch.equal(alone, want[qs:qs + T])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lsk.kv4_attn(q, cache, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    out, ws = torch.empty_like(want), torch.empty(plan.causal.ws_bytes, dtype=torch.uint8, device=cuda)
    x = torch.randn(n, 2 * Hkv, D, generator=g).to(BF16).to(cuda)
    rows, pos = (_i32(np.concatenate(y), cuda) for y in zip(*[([r] * t, np.arange(p, p + t)) for (r, p, t) in blocks]))
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):  # (as the engine captures: the generator state is shared)
        lsk.kv4_append(x[:, :Hkv], x[:, Hkv:], cache, rows, pos)
        lsk.kv4_attn(q, cache, plan, out=out, workspace=ws)
    for i in range(4):
        x.normal_(generator=torch.Generator(device=cuda).manual_seed(i))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        lsk.kv4_append(x[:, :Hkv], x[:, Hkv:], cache, rows, pos)
        assert torch.equal(lsk.kv4_attn(q, cache, plan), out)


@pytest.mark.gpu
def test_kv4_caches_past_32_bits(cuda):
    """Codes and exponents of the last rows lie past 2^32 bytes."""
    lsk = _lsk()
    B, Hkv, S, D = 514, 8, 16384, 128                 # 4.3 GB of K codes
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    new = lambda *s: torch.empty(B, Hkv, S // 64, D // 32, *s, dtype=torch.uint8, device=cuda)  # noqa: E731
    cache = lsk.KV4(new(64, 16), new(64, 16), new(16, 4), new(64))
    assert cache.k.numel() > 1 << 32
    g = _gen(2)
    n, p0, row = 200, S - 203, B - 1
    k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
    rows, pos = _i32(np.full(n, row), cuda), _i32(np.arange(n), cuda)
    for start in (p0, 0):
        lsk.kv4_append(k.to(cuda), v.to(cuda), cache, rows, pos + start)
        for got, x in zip(lsk.kv4_read(cache, rows, pos + start, F32), (k, v)):
            assert torch.equal(got.cpu().double(), held(x))
    q = torch.randn(3, 32, D, generator=g).to(BF16)
    tab = [(0, 190, 3, row)]
    got = lsk.kv4_attn(q.to(cuda), cache, lsk.AttnPlan(tab, 32, cache))
    kd, vd = (held(x).permute(1, 0, 2)[None] for x in (k, v))
    ref, mag, _ = attention(q.double(), kd, vd, [(0, 190, 3, 0)], 1 / math.sqrt(D))
    assert_close_bf16(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_trees_are_verified_accepted_and_compacted(cuda, D):
    """Steps of a server with drafted trees over the 4-bit cache: append, attention, acceptance, compaction, rollback;
    the cache of every layer is the definition's after each."""
    lsk = _lsk()
    rng, g = np.random.default_rng(D), _gen(D)
    L, B, Hq, Hkv, S = 2, 3, 4, 2, 256
    cache = lsk.KV4.zeros(B, Hkv, S, D, cuda, layers=L)
    kd, vd = (torch.zeros(L, B, Hkv, S, D, dtype=torch.float64) for _ in range(2))
    length = [0, 17, 63]
    kv_len = torch.tensor(length, device=cuda)
    for r, n in enumerate(length):
        for i in range(L if n else 0):
            k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
            lsk.kv4_append(k.to(cuda), v.to(cuda), cache.layer(i), _i32(np.full(n, r), cuda), _i32(np.arange(n), cuda))
            kd[i, r, :, :n], vd[i, r, :, :n] = held(k).transpose(0, 1), held(v).transpose(0, 1)
    for step in range(3):
        sizes = [40, 20, 33] if step == 0 else [int(rng.integers(1, 30)) for _ in range(B)]
        parents = [random_tree(rng, t) for t in sizes]
        tokens = [rng.integers(0, 2, t) for t in sizes]
        y = [rng.integers(0, 2, t) for t in sizes]
        order = rng.permutation(B)
        tab, n = pack_blocks([(int(r), length[r], sizes[r]) for r in order])
        rows = np.concatenate([[r] * sizes[r] for r in order])
        pos = np.concatenate([length[r] + np.arange(sizes[r]) for r in order])
        starts, lens = _i32([b[0] for b in tab], cuda), _i32([b[2] for b in tab], cuda)
        par = _cat([parents[r] for r in order], torch.int32, cuda)
        mask, _ = lsk.tree_masks(par, starts, lens, max(sizes))
        plan = lsk.AttnPlan(tab, Hq, cache.layer(0), split=None if step % 2 else 64, tree=True)
        sets = [s for r in order for s in ancestors(parents[r])]
        for i in range(L):
            k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
            q = torch.randn(n, Hq, D, generator=g).to(BF16)
            lsk.kv4_append(k.to(cuda), v.to(cuda), cache.layer(i), _i32(rows, cuda), _i32(pos, cuda))
            kd[i, rows, :, pos], vd[i, rows, :, pos] = held(k), held(v)
            got = lsk.kv4_attn(q.to(cuda), cache.layer(i), plan, mask)
            ref, mag, _ = attention(q.double(), kd[i], vd[i], tab, 1 / math.sqrt(D), sets)
            assert_close_bf16(got, ref, mag)
        acc, path, _ = lsk.tree_accept(_cat([y[r] for r in order], torch.int64, cuda),
                                       _cat([tokens[r] for r in order], torch.int64, cuda), par, starts, lens, max(sizes))
        r_t, p_t = _i32(order, cuda), _i32([length[r] for r in order], cuda)
        lsk.kv4_compact(cache, r_t, p_t, acc, path)
        lsk.kv_rollback(kv_len, r_t, acc, B)
        for i, r in enumerate(order):
            p = accept(parents[r], tokens[r], y[r])
            assert int(acc[i]) == len(p) - 1
            src = [length[r] + j for j in p]
            for x in (kd, vd):
                x[:, r, :, length[r]:length[r] + len(p)] = x[:, r][:, :, src].clone()
            length[r] += len(p)
        assert kv_len.cpu().tolist() == length
        for i in range(L):
            for r in range(B):
                at = (_i32(np.full(S, r), cuda), _i32(np.arange(S), cuda))
                for got, x in zip(lsk.kv4_read(cache.layer(i), *at, F32), (kd, vd)):
                    assert torch.equal(got.cpu().double(), x[i, r].transpose(0, 1))


# ----------------------------------------------------------------------------- query and key norms with rotation

def norm_rope(x, w, eps, cos, sin):
    """(value, magnitude of its two products) of heads x [n, h, d] at rows cos, sin [n, d], in 64 bits."""
    x, half = x.double(), x.shape[-1] // 2
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    turned = torch.cat([-y[..., half:], y[..., :half]], -1)
    return y * c + turned * s, (y * c).abs() + (turned * s).abs()


def assert_norms(got, ref, mag, dtype, d):
    tol = HALF[dtype] * ref.abs() * 1.01 + ((d + 2) / 2 * 2.0 ** -24 + 2.0 ** -22 + 3 * 2.0 ** -24) * 1.01 * mag + 1e-37
    assert ((got.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,Hq,Hkv,D", [(1, 1, 1, 64), (5, 8, 2, 128), (33, 4, 4, 32), (70, 6, 2, 64), (3, 40, 8, 128),
                                        (129, 2, 1, 256), (300, 8, 8, 128)])
def test_qk_norm_rope(cuda, dtype, n, Hq, Hkv, D):
    """Queries and keys, to tensors and to a cache: values, storage, untouched neighbours, tokens outside, rows with a
    pitch of their own; heads of zeros, of large and of small values."""
    lsk = _lsk()
    g = _gen(n + D)
    B, S, eps = 3, 128, 1e-5
    W = (Hq + 2 * Hkv) * D
    x = torch.randn(n, W, generator=g) * torch.exp2(torch.randint(-12, 12, (n, 1), generator=g).float())
    x[0, :D] = 0.0
    x = x.to(dtype)
    wq, wk = ((1 + torch.randn(D, generator=g) / 4).to(dtype) for _ in range(2))
    a = torch.arange(S).double()[:, None] * (10000.0 ** (-torch.arange(0, D, 2).double() / D)).repeat(2)
    cos, sin = a.cos().float(), a.sin().float()
    slot = torch.randperm(B * S, generator=g)[:n]
    rows, pos = slot // S, slot % S
    if n > 4:
        rows[1], pos[2], pos[3], rows[4] = -1, S, -1, B
    ok = (rows >= 0) & (rows < B) & (pos >= 0) & (pos < S)
    dev = torch.zeros(n, W + 5, dtype=dtype, device=cuda)[:, 2:W + 2]
    dev.copy_(x)
    tabs = (wq.to(cuda), wk.to(cuda), eps, cos.to(cuda), sin.to(cuda))
    q = torch.full((n, Hq, D), 7.0, dtype=dtype, device=cuda)
    k0, v0 = (torch.randn(B, Hkv, S, D, generator=g).to(dtype) for _ in range(2))
    kc = (lsk.k_to_frag(k0) if dtype == BF16 else k0).to(cuda).contiguous()
    vc = lsk.v_to_blocked(v0).to(cuda)
    lsk.qk_norm_rope_append(dev, q, kc, vc, *tabs, _i32(rows, cuda), _i32(pos, cuda), Hq, Hkv, D)
    heads = x.view(n, Hq + 2 * Hkv, D)
    p = pos.clamp(0, S - 1)
    ref_q, mag_q = norm_rope(heads[:, :Hq], wq, eps, cos[p], sin[p])
    ref_k, mag_k = norm_rope(heads[:, Hq:Hq + Hkv], wk, eps, cos[p], sin[p])
    assert_norms(q[ok], ref_q[ok], mag_q[ok], dtype, D)
    assert (q.cpu()[~ok] == 7.0).all()
    kd = lsk.k_from_frag(kc.cpu()) if dtype == BF16 else kc.cpu()
    vd = lsk.v_from_blocked(vc.cpu())
    assert_norms(kd[rows[ok], :, pos[ok]], ref_k[ok], mag_k[ok], dtype, D)
    assert torch.equal(vd[rows[ok], :, pos[ok]], heads[ok, Hq + Hkv:])
    rest = torch.ones(B, S, dtype=torch.bool)
    rest[rows[ok], pos[ok]] = False
    for got, was in ((kd, k0), (vd, v0)):
        assert torch.equal(got.transpose(1, 2)[rest], was.transpose(1, 2)[rest])
    inside = (pos >= 0) & (pos < S)
    q2, k2 = lsk.qk_norm_rope(dev, *tabs, _i32(pos, cuda), Hq, Hkv, D)
    assert torch.equal(q2.cpu()[ok], q.cpu()[ok])
    assert torch.equal(k2.cpu()[ok], kd[rows[ok], :, pos[ok]])
    assert_norms(k2[inside], ref_k[inside], mag_k[inside], dtype, D)


@pytest.mark.gpu
def test_qk_norm_rope_of_prompts_and_in_graphs(cuda):
    """Runs of positions from any start in several rows; replays between eager calls; a captured call."""
    lsk = _lsk()
    g = _gen(9)
    Hq, Hkv, D, B, S = 4, 2, 128, 4, 512
    runs = [(0, 1, 130), (1, 31, 33), (2, 0, 64), (3, 479, 33), (1, 64, 7)]
    rows = torch.cat([torch.full((n,), r) for (r, _, n) in runs])
    pos = torch.cat([torch.arange(p, p + n) for (_, p, n) in runs])
    n = len(rows)
    a = torch.arange(S).double()[:, None] * (10000.0 ** (-torch.arange(0, D, 2).double() / D)).repeat(2)
    w = torch.ones(D, dtype=BF16, device=cuda)
    tabs = (w, w, 1e-6, a.cos().float().to(cuda), a.sin().float().to(cuda))
    x = torch.randn(n, (Hq + 2 * Hkv) * D, generator=g).to(BF16).to(cuda)
    r_t, p_t = _i32(rows, cuda), _i32(pos, cuda)
    fresh = lambda: (torch.zeros(n, Hq, D, dtype=BF16, device=cuda), torch.zeros(B, Hkv, S // 32, D // 16, 64, 8, dtype=BF16, device=cuda),  # noqa: E731,E501
                     torch.zeros(B, Hkv, S // 32, D, 32, dtype=BF16, device=cuda))
    q, kc, vc = fresh()
    graph = torch.cuda.CUDAGraph()
    lsk.qk_norm_rope_append(x, q, kc, vc, *tabs, r_t, p_t, Hq, Hkv, D)
    with torch.inference_mode(), torch.cuda.graph(graph):  # (as the engine captures: the generator state is shared)
        lsk.qk_norm_rope_append(x, q, kc, vc, *tabs, r_t, p_t, Hq, Hkv, D)
    for i in range(3):
        x.normal_(generator=torch.Generator(device=cuda).manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        eager = fresh()
        lsk.qk_norm_rope_append(x, *eager, *tabs, r_t, p_t, Hq, Hkv, D)
        assert all(torch.equal(s, t) for s, t in zip(eager, (q, kc, vc)))
    heads = x.cpu().view(n, -1, D)
    assert torch.equal(lsk.v_from_blocked(vc.cpu())[rows, :, pos], heads[:, Hq + Hkv:])
    ref, mag = norm_rope(heads[:, Hq:Hq + Hkv], w.cpu(), 1e-6, tabs[3].cpu()[pos], tabs[4].cpu()[pos])
    assert_norms(lsk.k_from_frag(kc.cpu())[rows, :, pos], ref, mag, BF16, D)


# ----------------------------------------------------------------------------- 8-bit integer projections

def rows8(x):
    """(codes, scales) of the definition, 64 bits with its three fp32 roundings."""
    amax = x.float().abs().amax(1)
    ok = torch.isfinite(amax) & (amax >= 2.0 ** -100)
    safe = torch.where(ok, amax, torch.ones_like(amax))
    r, s = (torch.ones_like(safe) / safe) * 127.0, safe / 127.0       # fp32
    codes = torch.where(ok[:, None], torch.round(x.double().nan_to_num(0, 0, 0) * r.double()[:, None]), 0.0)
    s = torch.where(ok, s, torch.where(torch.isfinite(amax), 0.0, math.nan))
    return codes, s


def unpacked(data, rows, k):
    """Codes [rows, k] of packed fragments, index by index."""
    nks = (k + 63) // 64
    f = data.cpu().view(-1, nks, 64, 16)
    r, c = np.meshgrid(np.arange(rows), np.arange(k), indexing="ij")
    t = torch.as_tensor
    return f[t(r // 16), t(c // 64), t(c % 64 // 16 * 16 + r % 16), t(c % 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 64), (3, 63), (17, 100), (33, 1000), (5, 4096), (2, 20000), (40, 14336)])
def test_quant_rows_i8_is_exact(cuda, dtype, M, K):
    lsk = _lsk()
    g = _gen(M * K)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-20, 20, (M, 1), generator=g).float())
    x = x.to(dtype)
    if M > 2:
        x[0], x[1], x[2, 0] = 0.0, 2.0 ** -101, math.inf if K % 2 else math.nan
    if M > 4:
        x[3] = torch.finfo(dtype).max
        x[4] = (torch.arange(K) % 255 - 127).to(dtype) / 2             # half of the largest value: next to a tie
    view = torch.zeros(M, K + 3, dtype=dtype, device=cuda)[:, 1:K + 1]
    view.copy_(x)
    codes, scales = rows8(x)
    a = lsk.quant_rows_i8(view)
    assert torch.equal(a.scales.cpu().nan_to_num(-1), scales.nan_to_num(-1))
    live = torch.isfinite(scales)
    assert torch.equal(unpacked(a.codes, M, K)[live].double(), codes[live])
    nks = (K + 63) // 64
    pad = a.codes.cpu().view(-1, nks, 64, 16)[:, -1]                   # zeros past K in the rows that are there
    for r in range(M):
        tail = pad[r // 16].view(4, 16, 16)[:, r % 16].reshape(-1)[K - 64 * (nks - 1):]
        assert (tail == 0).all()
    again = lsk.quant_rows_i8(view, out=a)
    assert again is a
    w = lsk.PackedWeightI8(view)                                       # a weight is quantised by the same rule
    assert torch.equal(w.unpack().cpu()[live].double(), codes[live])
    w2 = lsk.PackedWeightI8(codes.nan_to_num(0).to(torch.int8).to(cuda), scales.to(cuda))
    assert torch.equal(w2.unpack().cpu().double(), codes.nan_to_num(0))
    assert torch.equal(unpacked(w2.data, M, K).double(), codes.nan_to_num(0))


def project(ca, sa, cw, sw, dtype, epilogue, res):
    """(exact value, what the kernel's fp32 steps may be off by) from integer codes and scales."""
    y = (ca @ cw.T) * sa.double()[:, None] * sw.double()
    err = 3 * 2.0 ** -24 * y.abs()
    if epilogue == 1:
        return y + res.double(), err + 2.0 ** -24 * (y.abs() + res.double().abs())
    if epilogue == 2:
        n = y.shape[1] // 2
        g, u, eg, eu = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
        s = g / (1 + torch.exp(-g))
        return s * u, (1.1 * eg + 2.0 ** -20 * s.abs()) * u.abs() * 1.01 + s.abs() * (eu + 2.0 ** -24 * u.abs())
    return y, err


def assert_project(got, want, dtype):
    ref, err = want
    got, nan = got.double().cpu(), torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    tol = HALF[dtype] * 1.01 * ref.abs() + 1.01 * err + 1e-37
    assert ((got - ref).abs() <= tol)[~nan].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("M,N,K", [(1, 16, 1), (1, 48, 64), (2, 33, 70), (15, 20, 256), (16, 100, 128), (17, 64, 1000),
                                   (33, 31, 520), (48, 256, 512), (64, 96, 2048), (65, 130, 300), (200, 272, 640),
                                   (257, 512, 1024), (513, 300, 192), (1025, 520, 1100)])
def test_gemm_i8(cuda, dtype, epilogue, M, N, K):
    lsk = _lsk()
    g = _gen(M + N + K)
    if epilogue == 2:
        N = (N + 15) // 16 * 16
    x = (torch.randn(M, K, generator=g) * 2).to(dtype)
    if M > 3:
        x[2, K // 2] = math.nan
        x[3] = 0.0
    w = torch.randn(2 * N if epilogue == 2 else N, K, generator=g) / math.sqrt(K)
    res = torch.randn(M, N + 1, generator=g).to(dtype)[:, :N] if epilogue == 1 else None
    ca, sa = rows8(x)
    cw, sw = rows8(w)
    want = project(ca, sa, cw, sw, dtype, epilogue, res)
    wp = lsk.PackedWeightI8(w.to(cuda))
    res_d = None
    if res is not None:
        res_d = torch.zeros(M, N + 1, dtype=dtype, device=cuda)[:, :N]
        res_d.copy_(res)
    buf = torch.full((M + 1, N + 3), 5.0, dtype=dtype, device=cuda)
    got = lsk.gemm_i8(lsk.quant_rows_i8(x.to(cuda)), wp, out=buf[:M, 1:N + 1], residual=res_d, epilogue=epilogue)
    assert_project(got, want, dtype)
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[:M, 1:N + 1] = False
    assert (buf[rest] == 5.0).all()
    # a row's bits do not depend on the rows beside it
    for lo, hi in ((0, 1), (M // 2, M // 2 + 3), (max(M - 40, 0), M)):
        part = lsk.gemm_i8(lsk.quant_rows_i8(x[lo:hi].to(cuda)), wp, residual=res_d[lo:hi] if res is not None else None,
                           epilogue=epilogue)
        assert torch.equal(part.nan_to_num(9), got[lo:hi].nan_to_num(9))


@pytest.mark.gpu
@pytest.mark.parametrize("epilogue,M,N,K", [(1, 131, 106, 70), (0, 130, 2048, 8192), (0, 65, 10006, 70),
                                            (1, 65, 10004, 4100), (1, 1602, 20011, 70), (0, 65, 20030, 70),
                                            (0, 257, 20002, 1100), (2, 65, 10000, 2104), (2, 66, 96, 70),
                                            (2, 65, 96, 600), (2, 65, 28000, 2100)])
def test_gemm_i8_of_many_tokens(cuda, epilogue, M, N, K):
    """A shape for each tiling of the many-token kernel; every row has the bits of the few-token kernel's."""
    lsk = _lsk()
    g = _gen(M + N + K)
    x = torch.randn(M, K, generator=g).to(BF16).to(cuda)
    w = lsk.PackedWeightI8(torch.randn(2 * N if epilogue == 2 else N, K, generator=g).to(cuda))
    res = torch.randn(M, N, generator=g).to(BF16).to(cuda) if epilogue == 1 else None
    a = lsk.quant_rows_i8(x)
    got = lsk.gemm_i8(a, w, residual=res, epilogue=epilogue)
    for lo in range(0, M, 64):
        part = lsk.gemm_i8(lsk.quant_rows_i8(x[lo:lo + 64]), w, residual=None if res is None else res[lo:lo + 64],
                           epilogue=epilogue)
        assert torch.equal(part, got[lo:lo + 64])
    pick = torch.tensor([0, M // 2, M - 1])
    ca, sa = rows8(x[pick.to(cuda)].cpu())
    cw, sw = (t.cpu() for t in (w.unpack().double(), w.scales))
    assert_project(got[pick.to(cuda)], project(ca, sa, cw, sw, BF16, epilogue, None if res is None else
                                               res[pick.to(cuda)].cpu()), BF16)


@pytest.mark.gpu
def test_gemm_i8_sums_do_not_overflow(cuda):
    """The longest rows, all of the largest magnitude: 127^2 * 131072 is below 2^31, and exact in fp32's rounding."""
    lsk = _lsk()
    K = 131072
    for M in (3, 70):
        x = torch.ones(M, K, device=cuda)
        x[1] = -1
        w = torch.full((20, K), 127, dtype=torch.int8, device=cuda)
        w[3] = -127
        got = lsk.gemm_i8(lsk.quant_rows_i8(x), lsk.PackedWeightI8(w, torch.full((20,), 1 / 127, device=cuda)))
        want = torch.full((M, 20), float(K), dtype=torch.float64)
        want[1] *= -1
        want[:, 3] *= -1
        assert ((got.double().cpu() - want).abs() <= 6 * 2.0 ** -24 * K).all()


@pytest.mark.gpu
def test_gemm_i8_in_graphs_and_on_streams(cuda):
    lsk = _lsk()
    g = _gen(4)
    x = torch.randn(37, 512, generator=g).to(BF16).to(cuda)
    w = lsk.PackedWeightI8(torch.randn(192, 512, generator=g).to(BF16).to(cuda))
    a = lsk.quant_rows_i8(x)
    out = lsk.gemm_i8(a, w, epilogue=lsk.EPI_SILU_MUL)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):  # (as the engine captures: the generator state is shared)
        lsk.gemm_i8(lsk.quant_rows_i8(x, out=a), w, out=out, epilogue=lsk.EPI_SILU_MUL)
    side = torch.cuda.Stream()
    for i in range(3):
        x.normal_(generator=torch.Generator(device=cuda).manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        eager = lsk.gemm_i8(lsk.quant_rows_i8(x), w, epilogue=lsk.EPI_SILU_MUL)
        assert torch.equal(eager, out)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = lsk.gemm_i8(lsk.quant_rows_i8(x), w, epilogue=lsk.EPI_SILU_MUL)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, out)


# ----------------------------------------------------------------------------- together

@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_layer_of_low_precision(cuda, D):
    """A prompt and then decode steps through a layer with integer projections, query and key norms and a 4-bit cache:
    every step against the formulas on the values that the step before gave."""
    lsk = _lsk()
    g = _gen(D)
    Hq, Hkv, B, S, eps, ffn = 4, 2, 2, 192, 1e-5, 320
    dim = Hq * D
    shapes = {"qkv": ((Hq + 2 * Hkv) * D, dim), "o": (dim, dim), "w13": (2 * ffn, dim), "w2": (dim, ffn)}
    w = {k: torch.randn(*s, generator=g) / math.sqrt(s[1]) for k, s in shapes.items()}
    wp = {k: lsk.PackedWeightI8(t.to(BF16).to(cuda)) for k, t in w.items()}
    ws = {k: rows8(t.to(BF16)) for k, t in w.items()}
    a = torch.arange(S).double()[:, None] * (10000.0 ** (-torch.arange(0, D, 2).double() / D)).repeat(2)
    cos, sin = a.cos().float(), a.sin().float()
    wq, wk = ((1 + torch.randn(D, generator=g) / 8).to(BF16) for _ in range(2))
    cache = lsk.KV4.zeros(B, Hkv, S, D, cuda)
    kd, vd = (torch.zeros(B, Hkv, S, D, dtype=torch.float64) for _ in range(2))
    length = [0, 0]

    def linear(x, name, epilogue=0, residual=None):
        got = lsk.gemm_i8(lsk.quant_rows_i8(x), wp[name], residual=residual, epilogue=epilogue)
        assert_project(got, project(*rows8(x.cpu()), *ws[name], BF16, epilogue,
                                    residual.cpu() if residual is not None else None), BF16)
        return got

    for T in ([70, 33], [1, 1], [5, 1], [1, 2]):
        tab, n = pack_blocks([(r, length[r], t) for r, t in enumerate(T)])
        rows = np.concatenate([[r] * t for r, t in enumerate(T)])
        pos = np.concatenate([length[r] + np.arange(t) for r, t in enumerate(T)])
        r_t, p_t = _i32(rows, cuda), _i32(pos, cuda)
        x = torch.randn(n, dim, generator=g).to(BF16).to(cuda)
        qkv = linear(x, "qkv")
        q, k = lsk.qk_norm_rope(qkv, wq.to(cuda), wk.to(cuda), eps, cos.to(cuda), sin.to(cuda), p_t, Hq, Hkv, D)
        heads = qkv.cpu().view(n, -1, D)
        assert_norms(q, *norm_rope(heads[:, :Hq], wq, eps, cos[pos], sin[pos]), BF16, D)
        assert_norms(k, *norm_rope(heads[:, Hq:Hq + Hkv], wk, eps, cos[pos], sin[pos]), BF16, D)
        v = qkv.view(n, -1, D)[:, Hq + Hkv:]
        lsk.kv4_append(k, v.contiguous(), cache, r_t, p_t)
        kd[rows, :, pos], vd[rows, :, pos] = held(k.cpu()), held(v.cpu())
        att = lsk.kv4_attn(q, cache, lsk.AttnPlan(tab, Hq, cache, tree=False))
        ref, mag, _ = attention(q.cpu().double(), kd, vd, tab, 1 / math.sqrt(D))
        assert_close_bf16(att, ref, mag)
        h = linear(att, "o", lsk.EPI_RESIDUAL, x)
        y = linear(linear(h, "w13", lsk.EPI_SILU_MUL), "w2", lsk.EPI_RESIDUAL, h)
        assert torch.isfinite(y).all()
        length = [p + t for p, t in zip(length, T)]


# ----------------------------------------------------------------------------- refusals

def test_lowbit_entry_points_refuse_bad_arguments():
    lib = _lsk().load()
    P = 16
    ok = [1, P, P, 128, 64, P, P, P, P, P, P, 4, 2, 64, 3, 128, None]
    bad = lambda i, x: lib.lsk_kv4_append(*(ok[:i] + [x] + ok[i + 1:]))  # noqa: E731
    for i in (1, 2, 5, 6, 7, 8, 9, 10):
        assert bad(i, None) == -1
    assert bad(0, 7) == -3 and bad(13, 96) == -3 and bad(15, 96) == -2 and bad(11, -1) == -2 and bad(3, -1) == -2
    assert bad(5, 24) == -1 and bad(14, 0) == -2 and bad(11, 0) == 0
    r = lib.lsk_kv4_read
    assert r(1, P, P, P, P, P, P, P, None, 4, 2, 64, 3, 128, None) == -1
    assert r(1, P, P, P, P, P, P, P, P, 4, 2, 32, 3, 128, None) == -3
    assert r(1, P, P, P, P, P, P, P, P, 0, 2, 64, 3, 128, None) == 0
    ok2 = [P, 512, 64, P, P, P, P, None, 0, None, 0, 0, P, 1, 1, 0, 1, 1, 16, P, 8, 2, 64, 128, 0.125, None, 0, None]
    k4 = lambda **kw: lib.lsk_kv4_attn(*[kw.get(f"a{i}", x) for i, x in enumerate(ok2)])  # noqa: E731
    assert k4(a0=None) == -1 and k4(a5=None) == -1 and k4(a12=None) == -1 and k4(a7=P) == -1 and k4(a5=24) == -1
    assert k4(a16=4) == -1 and k4(a22=32) == -3 and k4(a23=96) == -2 and k4(a10=1, a11=3) == -4 and k4(a13=0) == 0
    assert k4(a24=-0.5) == -1 and k4(a20=7) == -2 and k4(a17=2) == -1
    c = lib.lsk_kv_compact
    assert c(4, P, P, None, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == -1
    assert c(4, P, 24, P, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == -1
    assert c(4, P, P, P, P, 1, P, P, P, P, 1, 4, 2, 64, 3, 96, None) == -2
    assert c(4, P, P, P, P, 1, P, P, P, P, 1, 4, 2, 96, 3, 128, None) == -3
    assert c(4, P, P, P, P, 0, P, P, P, P, 1, 4, 2, 64, 3, 128, None) == 0
    # dtype, qkv, ld, weights, eps, tables, tab_len, rows, pos, n, Hq, Hkv, D, q, k, caches, B, S, stream
    ok3 = [1, P, 768, P, P, 1e-5, P, P, 64, P, P, 3, 4, 4, 64, P, None, P, P, 2, 64, None]
    nr = lambda **kw: lib.lsk_qk_norm_rope(*[kw.get(f"a{i}", x) for i, x in enumerate(ok3)])  # noqa: E731
    for i in (1, 3, 4, 6, 7, 9, 10, 15, 17, 18):
        assert nr(**{f"a{i}": None}) == -1
    assert nr(a16=P) == -1 and nr(a0=2) == -3 and nr(a14=96) == -3 and nr(a2=767) == -2 and nr(a13=3) == -2
    assert nr(a20=48) == -2 and nr(a5=-1.0) == -1 and nr(a5=math.nan) == -1 and nr(a11=0) == 0 and nr(a11=-1) == -2
    assert nr(a16=P, a17=None, a18=None, a9=None, a11=0) == 0
    qr = lib.lsk_quant_rows_i8
    assert qr(1, None, 64, P, P, 1, 64, None) == -1 and qr(5, P, 64, P, P, 1, 64, None) == -3
    assert qr(1, P, 63, P, P, 2, 64, None) == -2 and qr(1, P, 64, 24, P, 1, 64, None) == -1
    assert qr(1, P, 1 << 18, P, P, 1, 131073, None) == -2 and qr(1, P, 64, P, P, 0, 64, None) == 0
    assert lib.lsk_pack_i8(P, 64, 24, 16, 64, None) == -1 and lib.lsk_pack_i8(P, 60, P, 16, 64, None) == -2
    assert lib.lsk_unpack_i8(None, P, 64, 16, 64, None) == -1 and lib.lsk_unpack_i8(P, P, 64, 0, 64, None) == -2
    ok4 = [1, P, P, P, P, P, 64, None, 0, 2, 64, 64, 0, 0, None]
    gm = lambda **kw: lib.lsk_gemm_i8(*[kw.get(f"a{i}", x) for i, x in enumerate(ok4)])  # noqa: E731
    for i in (1, 2, 3, 4, 5):
        assert gm(**{f"a{i}": None}) == -1
    assert gm(a0=4) == -3 and gm(a12=3) == -3 and gm(a12=1) == -1 and gm(a6=63) == -2 and gm(a11=131073) == -2
    assert gm(a12=2, a13=32) == -2 and gm(a12=2, a10=24, a13=24) == -2 and gm(a1=24) == -1 and gm(a9=0) == 0


def test_calls_with_packed_arguments_are_the_same_calls():
    lsk = _lsk()
    lib = lsk.load()
    P = 16
    calls = {"lsk_kv4_append": (1, P, P, 128, 64, P, P, P, P, P, P, 0, 2, 64, 3, 128, 0),
             "lsk_kv4_read": (1, P, P, P, P, P, P, P, P, 0, 2, 64, 3, 128, 0),
             "lsk_kv4_attn": (P, 512, 64, P, P, P, P, 0, 0, 0, 0, 0, P, 0, 1, 0, 1, 1, 16, P, 8, 2, 64, 128, 0.125, 0, 0, 0),
             "lsk_qk_norm_rope": (1, P, 768, P, P, 1e-5, P, P, 64, P, P, 0, 4, 4, 64, P, 0, P, P, 2, 64, 0),
             "lsk_quant_rows_i8": (1, P, 64, P, P, 0, 64, 0),
             "lsk_gemm_i8": (1, P, P, P, P, P, 64, 0, 0, 0, 64, 64, 0, 0, 0)}
    assert set(calls) == set(lsk._CALLS)
    for name, args in calls.items():
        number, n, pack = lsk._CALLS[name]
        assert n == len(args) and lib.lsk_call(number, n, pack(*args)) == getattr(lib, name)(*args) == 0
        for i, x in enumerate(args):
            bad = args[:i] + (-1.0 if isinstance(x, float) else -7,) + args[i + 1:]
            got, text = lib.lsk_call(number, n, pack(*bad)), lib.lsk_last_error()
            assert got == getattr(lib, name)(*bad)
            assert got == 0 or text == lib.lsk_last_error() and text.startswith(name.encode())
        assert lib.lsk_call(number, n - 1, pack(*args)) == -1
    assert lib.lsk_call(len(calls), 1, bytes(8)) == lib.lsk_call(-1, 1, bytes(8)) == lib.lsk_call(0, 17, None) == -1


def test_kv4_plans_and_caches_refuse_what_does_not_fit():
    lsk = _lsk()
    cache = lsk.KV4.zeros(2, 2, 128, 64, "cpu")
    assert cache.dims == (2, 2, 128, 64) == cache.check("x") and cache.k.numel() == 2 * 2 * 128 * 32
    plan = lsk.AttnPlan([(0, 3, 2, 1), (2, 0, 0, 0), (2, 127, 1, 0)], 4, cache)
    assert plan.n_tokens == 3 and plan.causal.n_items > 0 and plan.tree.n_items > 0
    with pytest.raises(ValueError):
        lsk.AttnPlan([(0, 127, 2, 0)], 4, cache)
    for shape in ((2, 2, 100, 64), (2, 2, 128, 96), (2, 2, 0, 64)):
        with pytest.raises(ValueError):
            lsk.KV4.zeros(*shape, "cpu")
    for bad in (cache._replace(k=cache.k[:1]), cache._replace(vs=cache.vs[..., :32]), cache._replace(ks=cache.vs),
                cache._replace(v=cache.v.to(torch.int8))):
        with pytest.raises(lsk.LskError):
            bad.check("x")
    with pytest.raises(lsk.LskError):
        cache.check("x", layers=True)
    x, i = torch.zeros(1, 2, 64, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: lsk.kv4_append(x, x, cache, i, i), lambda: lsk.kv4_read(cache, i, i),
              lambda: lsk.kv4_attn(torch.zeros(3, 4, 64, dtype=BF16), cache, plan),
              lambda: lsk.quant_rows_i8(torch.zeros(2, 8)), lambda: lsk.PackedWeightI8(torch.zeros(2, 8))):
        with pytest.raises(lsk.LskError):                             # tensors off the GPU
            f()


@pytest.mark.gpu
def test_lowbit_wrappers_refuse_what_does_not_fit(cuda):
    lsk = _lsk()
    new = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=cuda)  # noqa: E731
    cache = lsk.KV4.zeros(2, 2, 128, 64, cuda)
    x, i, q, m = new(3, 2, 64), new(3, dtype=torch.int32), new(3, 4, 64), new(3, 1, dtype=torch.int32)
    plan = lsk.AttnPlan([(0, 0, 3, 0)], 4, cache)
    k8 = lsk.KV8.zeros(2, 2, 128, 64, cuda)
    p8 = lsk.AttnPlan([(0, 0, 3, 0)], 4, k8)
    qkv, w, t = new(3, 512), new(64), new(128, 64, dtype=F32)
    kf, vf = new(2, 2, 4, 4, 64, 8), new(2, 2, 4, 64, 32)
    norm = lambda **k: lsk.qk_norm_rope_append(*[k.get(f"a{j}", y) for j, y in enumerate(  # noqa: E731
        [qkv, q, kf, vf, w, w, 1e-5, t, t, i, i, 4, 2, 64])])
    norm()
    a, wt = lsk.quant_rows_i8(new(3, 64)), lsk.PackedWeightI8(torch.ones(32, 64, device=cuda))
    acc = new(1, dtype=torch.int64)
    calls = [lambda: lsk.kv4_append(x.half(), x.half(), cache, i, i), lambda: lsk.kv4_append(x, x[:2], cache, i, i),
             lambda: lsk.kv4_append(x, x, k8, i, i), lambda: lsk.kv4_read(cache, i, i, torch.float16),
             lambda: lsk.kv4_attn(q, cache, p8), lambda: lsk.kv8_attn(q, k8, plan), lambda: lsk.kv4_attn(q, k8, p8),
             lambda: lsk.kv4_attn(q.float(), cache, plan), lambda: lsk.kv4_attn(q, cache, plan, m[:2]),
             lambda: lsk.kv4_attn(q, cache, plan, scale=-1.0), lambda: lsk.kv4_attn(q[:2], cache, plan),
             lambda: lsk.kv4_compact(cache, i[:1], i[:1], acc, m[:1]),
             lambda: norm(a0=qkv[:, :500]), lambda: norm(a0=qkv.half()), lambda: norm(a1=q[:2]), lambda: norm(a2=kf[:, :1]),
             lambda: norm(a3=vf[:1]), lambda: norm(a4=w[:32]), lambda: norm(a5=w.float()), lambda: norm(a7=t[:, :32]),
             lambda: norm(a8=t[:64]), lambda: norm(a9=i.long()), lambda: norm(a10=i[:2]), lambda: norm(a13=32),
             lambda: norm(a11=3), lambda: norm(a10=i.cpu()),
             lambda: lsk.qk_norm_rope(qkv, w, w, 1e-5, t, t, i, 4, 2, 64, out=(q, x[:2])),
             lambda: lsk.qk_norm_rope(qkv, w, w, -1.0, t, t, i, 4, 2, 64),
             lambda: lsk.quant_rows_i8(new(3, 64).half()), lambda: lsk.quant_rows_i8(new(64, 3).T),
             lambda: lsk.quant_rows_i8(new(4, 64), out=a), lambda: lsk.quant_rows_i8(new(3, 131073)),
             lambda: lsk.PackedWeightI8(new(4, 64, dtype=torch.int8)), lambda: lsk.PackedWeightI8(new(4, 64), new(4, dtype=F32)),
             lambda: lsk.PackedWeightI8(new(4, 64, dtype=torch.int8), new(3, dtype=F32)), lambda: lsk.PackedWeightI8(new(0, 64)),
             lambda: lsk.gemm_i8(lsk.quant_rows_i8(new(3, 32)), wt), lambda: lsk.gemm_i8(a, wt, epilogue=1),
             lambda: lsk.gemm_i8(a, wt, residual=new(3, 32)), lambda: lsk.gemm_i8(a, wt, residual=new(3, 31), epilogue=1),
             lambda: lsk.gemm_i8(a, wt, out=new(3, 32, dtype=F32)), lambda: lsk.gemm_i8(a, wt, out=new(32, 3).T),
             lambda: lsk.gemm_i8(a, lsk.PackedWeightI8(torch.ones(48, 64, device=cuda)), epilogue=2)]
    for j, f in enumerate(calls):
        with pytest.raises(lsk.LskError):
            f()
            print("not refused:", j)
    assert lsk.kv4_attn(q[:0], cache, lsk.AttnPlan([], 4, cache)).shape == (0, 256)
    assert lsk.gemm_i8(lsk.quant_rows_i8(new(0, 64)), wt).shape == (0, 32)
    assert lsk.qk_norm_rope(qkv[:0], w, w, 1e-5, t, t, i[:0], 4, 2, 64)[1].shape == (0, 2, 64)
    lsk.kv4_append(x[:0], x[:0], cache, i[:0], i[:0])
