"""The low-precision operators at the edges of what a caller may hand them: rows closer together than their length,
buffers that do not fit, plans of another kind.  Refusals run on the CPU: the wrappers' launches are caught there."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import test_lowbit_ops as ops
from test_cache_ops import BF16, F32, _gen, _i32, _lsk
from test_lowbit_ops import assert_project, project, rows8


@pytest.fixture
def launches(monkeypatch):
    """The wrappers on CPU tensors: the launches [(entry point, its arguments)] that they would make."""
    lsk, made = _lsk(), []
    monkeypatch.setattr(lsk, "_dev", lambda *ts: None)
    monkeypatch.setattr(lsk, "_one_device", lambda *ts: 0)
    monkeypatch.setattr(lsk, "_launch", lambda dev, what, *args: made.append((what, args)))
    return made


def _refused(launches, f):
    lsk = _lsk()
    launches.clear()
    with pytest.raises(lsk.LskError):
        f()
    assert not [what for what, _ in launches if what != "lsk_pack_i8"]


def _overlapping(m, n, pitch, dtype=BF16):
    """[m, n] with rows `pitch` < n elements apart."""
    return torch.zeros((m - 1) * pitch + n, dtype=dtype).as_strided((m, n), (pitch, 1))


# ----------------------------------------------------------------------------- rows closer together than their length

@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gemm_i8_takes_the_pitch_of_out_and_residual_as_it_is(launches, dtype):
    lsk = _lsk()
    M, N, K = 5, 32, 64
    w = lsk.PackedWeightI8(torch.zeros(N, K, dtype=torch.int8), torch.ones(N))
    a = lsk.quant_rows_i8(torch.zeros(M, K, dtype=dtype))
    bias = torch.zeros(N, dtype=dtype)
    for r in (bias.expand(M, N), _overlapping(M, N, 8, dtype), _overlapping(M, N, N - 1, dtype)):
        _refused(launches, lambda: lsk.gemm_i8(a, w, residual=r, epilogue=lsk.EPI_RESIDUAL))
        _refused(launches, lambda: lsk.gemm_i8(a, w, out=r))
    launches.clear()
    out, res = torch.zeros(M, N + 3, dtype=dtype)[:, :N], torch.zeros(2 * M, N, dtype=dtype)[::2]
    lsk.gemm_i8(a, w, out=out, residual=res, epilogue=lsk.EPI_RESIDUAL)
    one = lsk.quant_rows_i8(torch.zeros(1, K, dtype=dtype))           # (the pitch of a single row means nothing)
    lsk.gemm_i8(one, w, out=bias.as_strided((1, N), (3, 1)), residual=bias.expand(1, N), epilogue=lsk.EPI_RESIDUAL)
    (_, args), (_, single) = (x for x in launches if x[0] == "lsk_gemm_i8")
    assert args[6] == N + 3 and args[8] == 2 * N                      # ldc, ldr
    assert single[6] >= N and single[8] >= N


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quant_rows_i8_takes_the_pitch_of_the_rows_as_it_is(launches, dtype):
    lsk = _lsk()
    K = 64
    row = torch.zeros(K, dtype=dtype)
    for x in (row.expand(5, K), _overlapping(5, K, 8, dtype), _overlapping(5, K, K - 1, dtype)):
        _refused(launches, lambda: lsk.quant_rows_i8(x))
        _refused(launches, lambda: lsk.PackedWeightI8(x))
    launches.clear()
    lsk.quant_rows_i8(torch.zeros(5, K + 7, dtype=dtype)[:, 3:K + 3])
    lsk.PackedWeightI8(torch.zeros(10, K, dtype=dtype)[::2])
    lsk.quant_rows_i8(row.as_strided((1, K), (1, 1)))
    assert [args[2] for _, args in launches] == [K + 7, 2 * K, K]


def test_packed_weights_take_the_pitch_of_the_codes_as_it_is(launches):
    lsk = _lsk()
    N, K = 6, 64
    for w in (torch.zeros(K, dtype=torch.int8).expand(N, K), _overlapping(N, K, 16, torch.int8)):
        launches.clear()
        with pytest.raises(lsk.LskError):
            lsk.PackedWeightI8(w, torch.ones(N))
        assert not launches
    lsk.PackedWeightI8(torch.zeros(N, K + 5, dtype=torch.int8)[:, :K], torch.ones(N))
    lsk.PackedWeightI8(torch.zeros(K, dtype=torch.int8).expand(1, K), torch.ones(1))
    assert [args[1] for _, args in launches] == [K + 5, K]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_qk_norm_rope_takes_the_pitch_of_the_rows_as_it_is(launches, dtype):
    lsk = _lsk()
    n, Hq, Hkv, D, S = 5, 4, 2, 32, 64
    W = (Hq + 2 * Hkv) * D
    w, tab = torch.ones(D, dtype=dtype), torch.zeros(S, D)
    kc = torch.zeros(1, Hkv, S // 32, D // 16, 64, 8, dtype=dtype) if dtype == BF16 else torch.zeros(1, Hkv, S, D)
    vc = torch.zeros(1, Hkv, S // 32, D, 32, dtype=dtype)

    def both(qkv):
        m = len(qkv)
        i = torch.zeros(m, dtype=torch.int32)
        return (lambda: lsk.qk_norm_rope(qkv, w, w, 1e-5, tab, tab, i, Hq, Hkv, D),
                lambda: lsk.qk_norm_rope_append(qkv, torch.zeros(m, Hq, D, dtype=dtype), kc, vc, w, w, 1e-5, tab, tab, i, i,
                                                Hq, Hkv, D))

    for qkv in (torch.zeros(W, dtype=dtype).expand(n, W), _overlapping(n, W, D, dtype), _overlapping(n, W, W - 1, dtype)):
        for f in both(qkv):
            _refused(launches, f)
    launches.clear()
    for qkv in (torch.zeros(n, W + 9, dtype=dtype)[:, :W], torch.zeros(3 * n, W, dtype=dtype)[::3],
                torch.zeros(W, dtype=dtype).expand(1, W)):
        for f in both(qkv):
            f()
    assert [args[2] for _, args in launches] == [W + 9] * 2 + [3 * W] * 2 + [W] * 2


# ----------------------------------------------------------------------------- buffers of quantised rows

def test_rows_i8_refuse_buffers_that_do_not_hold_them():
    """The kernel writes codes and scales behind them: (M + 15) / 16 * (K + 63) / 64 KiB and 4 M bytes."""
    lsk = _lsk()
    M, K = 17, 100
    need = 2 * 2 * 1024 + 4 * M
    new = lambda n, dtype=torch.int8: torch.zeros(n, dtype=dtype)     # noqa: E731
    for n in (need, need + 5):
        rows = lsk.RowsI8(new(n), (M, K), BF16)
        assert rows.codes.numel() == need - 4 * M and rows.scales.shape == (M,)
    lsk.RowsI8(new(0), (0, K), F32)
    for data, shape, dtype in ((new(need - 1), (M, K), BF16), (new(16), (1, 2097152), BF16), (new(0), (1, 1), F32),
                               (new(need, torch.float32), (M, K), BF16), (new(2 * need)[::2], (M, K), BF16),
                               (new(1).expand(need), (M, K), BF16), (new(need).view(1, need), (M, K), BF16),
                               (new(need), (M, K), torch.float16), (new(need), (M,), BF16), (new(need), (-1, K), BF16),
                               (new(need), (M, 0), BF16), (new(need + 1)[1:], (M, K), BF16)):
        with pytest.raises(lsk.LskError):
            lsk.RowsI8(data, shape, dtype)


def test_quantised_rows_given_again_have_to_be_of_the_same_shape(launches):
    lsk = _lsk()
    a = lsk.quant_rows_i8(torch.zeros(3, 64, dtype=BF16))
    assert lsk.quant_rows_i8(torch.ones(3, 64, dtype=BF16), out=a) is a
    for x in (torch.zeros(4, 64, dtype=BF16), torch.zeros(3, 65, dtype=BF16), torch.zeros(3, 64)):
        _refused(launches, lambda: lsk.quant_rows_i8(x, out=a))


# ----------------------------------------------------------------------------- plans of another kind

@pytest.mark.parametrize("D", [64, 128])
def test_a_trees_plan_over_a_4_bit_cache_needs_its_mask(D):
    """The kernels without a mask hold fewer rows of an item of two row groups than a tree's plan gives them.  The check of
    the workspace comes after that of the plan's kind: -4 says that the kind was taken."""
    lsk = _lsk()
    lib, P = lsk.load(), 16

    def attn(cnt, mask, fmt=2, rg=None):
        _, ng, parts, rounds, tiles, part_rows, _, used, shared = (int(x) for x in cnt)
        args = (P, 512, 64, P, P, P, P, P if mask else None, 4 if mask else 0, P, ng, parts, P, rounds, 512, shared, tiles,
                used if rg is None else rg, part_rows, P, 32, 8, D, 8192, 0.125, None, 0, None)
        return (lib.lsk_kv4_attn if fmt == 2 else lib.lsk_kv8_attn)(*args)

    def plan(t, tree, rows=8, groups=0, fmt=2, pos0=5000):
        blk, cnt = np.array([0, pos0, t, 0], dtype=np.int32), np.zeros(9, dtype=np.int64)
        assert lib.lsk_cache_attn_plan(blk.ctypes.data, 1, 4, 64, rows, 8, D, fmt, int(tree), groups, 512, None, 0,
                                       cnt.ctypes.data) == 0 and cnt[2] > 0
        return cnt

    for t in (9, 12, 16, 40, 100):
        for groups in (0, 1, 2, 4):
            for fmt in (1, 2):
                cnt = plan(t, True, 8, groups, fmt)
                assert cnt[7] in (1, 2, 4) and attn(cnt, True, fmt) == -4
                assert attn(cnt, False, fmt) == (-4 if cnt[7] == 1 else -1)
        for rows in (8, 40, 100, 1000):               # no groups, pairs, wide blocks
            cnt = plan(t, False, rows)
            assert attn(cnt, False) == -4
            assert cnt[7] == 1 and cnt[8] == 0 or cnt[7] in (8 + 2, 8 + 4)
            if cnt[7] > 1:                            # (a tree's of as many row groups; no 8-bit plan has them)
                assert attn(cnt, False, rg=int(cnt[7]) & 7) == -1 and attn(cnt, False, 1) == -1
    cnt = plan(40, False, 1000)
    assert cnt[8] > 0
    for rg in (0, 1, 2, 3, 4, 5, 6, 8, 9, 11, 16, -2):
        assert attn(cnt, False, rg=rg) == -1
    one = lsk.AttnPlan([(0, 3, 40, 0)], 32, lsk.KV4(*(t.expand(1000, 8, *t.shape[2:]) for t in lsk.KV4.zeros(
        1, 1, 64, D, "cpu"))), tree=False).causal
    assert one.row_groups in (2, 4) and one.args[8] == 8 + one.row_groups


# ----------------------------------------------------------------------------- a residual that takes the result

def test_gemm_i8_takes_the_residuals_pitch_where_it_is_the_output(launches):
    lsk = _lsk()
    M, N, K = 5, 32, 64
    w = lsk.PackedWeightI8(torch.zeros(N, K, dtype=torch.int8), torch.ones(N))
    h = torch.zeros(M, N + 4, dtype=BF16)[:, :N]
    lsk.gemm_i8(lsk.quant_rows_i8(torch.zeros(M, K, dtype=BF16)), w, out=h, residual=h, epilogue=lsk.EPI_RESIDUAL)
    what, args = launches[-1]
    assert what == "lsk_gemm_i8" and args[5] == args[7] == h.data_ptr() and args[6] == args[8] == N + 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 33, 100), (5, 32, 64), (64, 130, 300), (130, 272, 640), (513, 520, 192)])
def test_gemm_i8_adds_to_its_output_in_place(cuda, dtype, M, N, K):
    lsk = _lsk()
    g = _gen(M + K)
    a = lsk.quant_rows_i8(torch.randn(M, K, generator=g).to(dtype).to(cuda))
    w = lsk.PackedWeightI8(torch.randn(N, K, generator=g).to(cuda))
    buf = torch.randn(M, N + 5, generator=g).to(dtype).to(cuda)
    for h in (buf[:, 2:N + 2], buf[:, :N].contiguous()):
        want = lsk.gemm_i8(a, w, residual=h.clone(), epilogue=lsk.EPI_RESIDUAL)
        assert lsk.gemm_i8(a, w, out=h, residual=h, epilogue=lsk.EPI_RESIDUAL) is h
        assert torch.equal(h, want)


# ----------------------------------------------------------------------------- scales at the ends of fp32's range

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("M", [4, 130])
def test_gemm_i8_of_the_largest_activations_stays_finite(cuda, dtype, epilogue, M):
    """Rows up to the type's largest value against weights that bring the products back: sum * scale alone passes 2^128."""
    lsk = _lsk()
    g = _gen(M)
    N, K = 48, 256
    x = torch.randn(M, K, generator=g)
    x *= torch.exp2(torch.linspace(-60, 120, M))[:, None]             # (the last rows' scales pass 2^90)
    x[-1] = torch.finfo(dtype).max * torch.sign(x[-1])
    x = x.to(dtype)
    w = torch.randn(2 * N if epilogue == 2 else N, K, generator=g) * 2.0 ** -75
    w[0] = w[0].abs() * torch.sign(x[-1].float())                     # 256 products of one sign
    res = torch.randn(M, N, generator=g).to(dtype) if epilogue == 1 else None
    (ca, sa), (cw, sw) = rows8(x), rows8(w)
    assert ((ca @ cw.T).float().abs().amax(1) * sa).isinf().any()
    want = project(ca, sa, cw, sw, dtype, epilogue, res)
    assert torch.isfinite(want[0].to(dtype)).all()
    got = lsk.gemm_i8(lsk.quant_rows_i8(x.to(cuda)), lsk.PackedWeightI8(w.to(cuda)),
                      residual=None if res is None else res.to(cuda), epilogue=epilogue)
    assert_project(got, want, dtype)


# ----------------------------------------------------------------------------- the kernels for many tokens

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,n,h", [(64, 520, 32), (128, 520, 32), (64, 576, 17), (128, 300, 40), (128, 257, 32)])
def test_kv4_append_and_read_of_many_tokens_are_exact(cuda, dtype, D, n, h):
    """From 8192 tokens times heads on, positions in any order: the same checks as for few (test_lowbit_ops)."""
    assert n * h >= 8192
    ops.test_kv4_append_and_read_are_exact(cuda, dtype, D, n, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,h", [(64, 32), (128, 32), (128, 17)])
def test_kv4_runs_of_many_tokens_from_any_start(cuda, dtype, D, h):
    """Runs that start and end inside 16 positions, beside each other and across the workgroups' tokens, with stray tokens
    and NaN between them, as views of fused rows: every token's values, and nothing of its neighbours."""
    lsk = _lsk()
    g = _gen(D + h)
    B, S = 7, 256
    runs = [(0, 1, 16), (1, 2, 33), (2, 57, 31), (2, 88, 40), (3, 240, 16), (4, 3, 1), (0, 61, 5), (5, 255, 1),
            (5, 0, 96), (4, 130, 29), (6, 5, 250)]
    rows = torch.cat([torch.full((n,), r) for (r, _, n) in runs])
    pos = torch.cat([torch.arange(p, p + n) for (_, p, n) in runs])
    for order in ("as they are", "shifted", "shuffled"):
        if order == "shifted":
            rows, pos = rows.roll(3), pos.roll(3)
        elif order == "shuffled":
            perm = torch.randperm(len(rows), generator=g)
            rows, pos = rows[perm], pos[perm]
        r, p = rows.clone(), pos.clone()
        r[20], p[40], r[60], p[300] = -1, -3, B, S    # (in the middle of runs)
        ok = (r >= 0) & (r < B) & (p >= 0) & (p < S)
        n = len(rows)
        assert n * h >= 8192
        x = torch.randn(n, 3 * h * D + 1, generator=g).to(dtype)
        x[7, 5], x[100, h * D + 70], x[200, 2 * h * D - 1] = math.nan, math.inf, -math.inf
        k, v = (t[:, o:o + h * D].unflatten(1, (h, D)) for t, o in ((x, 1), (x, 1 + h * D)))
        dev = x.to(cuda)
        cache = lsk.KV4.zeros(B, h, S, D, cuda)
        for t in (cache.k, cache.v):
            t.fill_(0x33)                             # (1.5 everywhere else)
        lsk.kv4_append(*(dev[:, o:o + h * D].unflatten(1, (h, D)) for o in (1, 1 + h * D)), cache, _i32(r, cuda),
                       _i32(p, cuda))
        every = (_i32(torch.arange(B).repeat_interleave(S), cuda), _i32(torch.arange(S).repeat(B), cuda))
        for got, some, t in zip(lsk.kv4_read(cache, *every, F32), lsk.kv4_read(cache, _i32(r, cuda), _i32(p, cuda), dtype),
                                (k, v)):
            want = torch.full((B, S, h, D), 1.5, dtype=torch.float64)
            want[r[ok], p[ok]] = ops.held(t[ok])
            for a, b in ((got.view(B, S, h, D), want), (some[ok.to(cuda)], ops.held(t[ok]))):
                assert torch.equal(torch.isnan(a.cpu()), torch.isnan(b))
                assert torch.equal(a.cpu().double().nan_to_num(0), b.nan_to_num(0))
            assert (some[~ok.to(cuda)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,Hkv,D", [(40, 10, 128), (6, 2, 64), (32, 8, 128), (52, 4, 32), (3, 1, 256)])
def test_qk_norm_rope_of_many_tokens(cuda, dtype, Hq, Hkv, D):
    """From 512 tokens on: prompts from any start and single tokens, some outside the cache or the tables, head counts that
    leave part of a workgroup's last pass empty."""
    lsk = _lsk()
    g = _gen(Hq + D)
    B, S, eps = 6, 320, 1e-5
    runs = [(0, 1, 130), (1, 31, 33), (2, 0, 64), (3, 287, 33), (1, 64, 7), (4, 5, 255), (5, 300, 1), (5, 100, 1), (0, 200, 3)]
    rows = torch.cat([torch.full((n,), r) for (r, _, n) in runs])
    pos = torch.cat([torch.arange(p, p + n) for (_, p, n) in runs])
    n, W = len(rows), (Hq + 2 * Hkv) * D
    assert n >= 512
    rows[11], pos[70], rows[200], pos[333] = -1, S, B, -1
    limit = S - 2                                     # (the last positions lie outside the tables)
    a = torch.arange(limit).double()[:, None] * (10000.0 ** (-torch.arange(0, D, 2).double() / D)).repeat(2)
    cos, sin = a.cos().float(), a.sin().float()
    ok = (rows >= 0) & (rows < B) & (pos >= 0) & (pos < limit)
    assert int((~ok).sum()) > 4
    x = (torch.randn(n, W + 3, generator=g) * torch.exp2(torch.randint(-12, 12, (n, 1), generator=g).float())).to(dtype)
    x[5, 1:1 + D] = 0.0
    wq, wk = ((1 + torch.randn(D, generator=g) / 4).to(dtype) for _ in range(2))
    tabs = (wq.to(cuda), wk.to(cuda), eps, cos.to(cuda), sin.to(cuda))
    dev = x.to(cuda)[:, 1:W + 1]
    q = torch.full((n, Hq, D), 7.0, dtype=dtype, device=cuda)
    k0, v0 = (torch.randn(B, Hkv, S, D, generator=g).to(dtype) for _ in range(2))
    kc = (lsk.k_to_frag(k0) if dtype == BF16 else k0).to(cuda).contiguous()
    vc = lsk.v_to_blocked(v0).to(cuda)
    lsk.qk_norm_rope_append(dev, q, kc, vc, *tabs, _i32(rows, cuda), _i32(pos, cuda), Hq, Hkv, D)
    heads, p = x[:, 1:W + 1].unflatten(1, (-1, D)), pos.clamp(0, limit - 1)
    ref_q, mag_q = ops.norm_rope(heads[:, :Hq], wq, eps, cos[p], sin[p])
    ref_k, mag_k = ops.norm_rope(heads[:, Hq:Hq + Hkv], wk, eps, cos[p], sin[p])
    ops.assert_norms(q[ok.to(cuda)], ref_q[ok], mag_q[ok], dtype, D)
    assert (q.cpu()[~ok] == 7.0).all()
    kd = lsk.k_from_frag(kc.cpu()) if dtype == BF16 else kc.cpu()
    vd = lsk.v_from_blocked(vc.cpu())
    ops.assert_norms(kd[rows[ok], :, pos[ok]], ref_k[ok], mag_k[ok], dtype, D)
    assert torch.equal(vd[rows[ok], :, pos[ok]], heads[ok, Hq + Hkv:])
    rest = torch.ones(B, S, dtype=torch.bool)
    rest[rows[ok], pos[ok]] = False
    for got, was in ((kd, k0), (vd, v0)):
        assert torch.equal(got.transpose(1, 2)[rest], was.transpose(1, 2)[rest])
    k2 = torch.full((n, Hkv, D), 7.0, dtype=dtype, device=cuda)
    q2 = torch.full_like(q, 7.0)
    lsk.qk_norm_rope(dev, *tabs, _i32(pos, cuda), Hq, Hkv, D, out=(q2, k2))
    inside = (pos >= 0) & (pos < limit)
    assert torch.equal(q2.cpu()[ok], q.cpu()[ok]) and torch.equal(k2.cpu()[ok], kd[rows[ok], :, pos[ok]])
    ops.assert_norms(k2[inside.to(cuda)], ref_k[inside], mag_k[inside], dtype, D)
    assert (q2.cpu()[~inside] == 7.0).all() and (k2.cpu()[~inside] == 7.0).all()


# ----------------------------------------------------------------------------- items of 128 rows over 128 dims

def _cache_of_blocks(lsk, cuda, B, Hkv, S, D, tab, g):
    """A 4-bit cache whose rows hold the blocks' contexts, NaN behind them; K and V [blocks, Hkv, S, D] on the CPU."""
    k, v = (torch.randn(len(tab), Hkv, S, D, generator=g).to(BF16) for _ in range(2))
    cache = lsk.KV4.zeros(B, Hkv, S, D, cuda)
    for t, fill in zip(cache, (0xF7, 0x7F, 255, 255)):
        t.fill_(fill)
    ends = [p0 + T for (_, p0, T, _) in tab]
    rows = _i32(np.concatenate([np.full(m, row) for (_, _, _, row), m in zip(tab, ends)]), cuda)
    pos = _i32(np.concatenate([np.arange(m) for m in ends]), cuda)
    flat = lambda x: torch.cat([x[i, :, :m].transpose(0, 1) for i, m in enumerate(ends)]).to(cuda)  # noqa: E731
    lsk.kv4_append(flat(k), flat(v), cache, rows, pos)
    return cache, k, v


def _check_blocks(lsk, cuda, got, q, cache, k, v, tab, Hq, D, split, few, sets=None, words=None):
    """`few` blocks against 64 bits; every block's bits against the block planned alone, in items of 64 rows."""
    for i in few:
        qs, p0, T, _ = tab[i]
        ref, mag, _ = ops.attention(q[qs:qs + T].double(), ops.held(k[i:i + 1]), ops.held(v[i:i + 1]), [(0, p0, T, 0)],
                                    1 / math.sqrt(D), None if sets is None else sets[qs:qs + T])
        ops.assert_close_bf16(got[qs:qs + T], ref, mag)
    for (qs, p0, T, row) in tab:
        alone = lsk.AttnPlan([(0, p0, T, row)], Hq, cache, split=split, tree=sets is not None)
        launch = alone.causal if sets is None else alone.tree
        assert launch.row_groups < 4
        one = lsk.kv4_attn(q[qs:qs + T].to(cuda), cache, alone, None if sets is None else words[qs:qs + T])
        assert torch.equal(one.view(torch.int16), got[qs:qs + T].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("split", [256, 1024])
@pytest.mark.parametrize("small", [False, True])
def test_kv4_large_trees_in_items_of_128_rows(cuda, small, split):
    """More trees of 64 nodes than CUs, alone and beside small ones in one launch; contexts in splits; nodes that read
    nothing; NaN behind every block."""
    lsk = _lsk()
    g, rng = _gen(split), np.random.default_rng(split + small)
    B, Hkv, Hq, S, D = 48, 8, 32, 640, 128
    blocks = [(int(r), 0 if j == 1 else int(rng.integers(0, 570)), 64 - j % 3) for j, r in enumerate(rng.permutation(B)[:34])]
    blocks += [(r, 90 * i, 1 + 2 * i) for i, r in enumerate(sorted(set(range(B)) - {b[0] for b in blocks})[:4])] if small else []
    tab, n = ops.pack_blocks(blocks)
    sets = [s for (_, _, t) in blocks for s in ops.ancestors(ops.random_tree(rng, t))]
    first = tab[1][0]                                 # (block 1 has no prefix)
    sets[first], sets[first + 40] = frozenset(), frozenset()
    cache, k, v = _cache_of_blocks(lsk, cuda, B, Hkv, S, D, tab, g)
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    words = _i32(ops.words_of(sets, 2), cuda)
    plan = lsk.AttnPlan(tab, Hq, cache, split=split, tree=True)
    assert plan.tree.row_groups == 4 and plan.tree.n_shared > 256 and (plan.tree.n_rounds > 0) == small
    assert (plan.tree.n_parts > 0) == (split < 640)
    got = lsk.kv4_attn(q.to(cuda), cache, plan, words)
    assert (got[first] == 0).all() and (got[first + 40] == 0).all() and torch.isfinite(got).all()
    _check_blocks(lsk, cuda, got, q, cache, k, v, tab, Hq, D, split, [0, 1, 2, len(tab) - 1], sets, words)


@pytest.mark.gpu
def test_kv4_prompt_pieces_in_items_of_128_rows_beside_single_tokens(cuda):
    """More large pieces than CUs, blocks of two row groups and single tokens in one launch."""
    lsk = _lsk()
    g, rng = _gen(23), np.random.default_rng(23)
    B, Hkv, Hq, S, D = 100, 8, 32, 192, 128
    tokens = [17 + i % 3 for i in range(38)] + [1] * 20 + [9] * 6 + [40, 5]
    tab, n = ops.pack_blocks([(int(r), int(rng.integers(0, 150)), t) for r, t in zip(rng.permutation(B), tokens)])
    cache, k, v = _cache_of_blocks(lsk, cuda, B, Hkv, S, D, tab, g)
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    plan = lsk.AttnPlan(tab, Hq, cache, tree=False)
    assert plan.causal.row_groups == 4 and plan.causal.n_shared > 256 and plan.causal.n_rounds > 0
    got = lsk.kv4_attn(q.to(cuda), cache, plan)
    assert torch.isfinite(got).all()
    _check_blocks(lsk, cuda, got, q, cache, k, v, tab, Hq, D, None, [0, 1, 37, 38, 60, 64, 65])
