"""ctypes binding of liblsk.so, the C ABI of the gfx950 kernels (include/lsk.h).

Only device pointers, sizes and the current HIP stream cross the boundary.  Tensors stay owned by
PyTorch (device memory + streams are plumbing; every FLOP of the packed forward runs in liblsk).
There is no fallback: a missing or stale library raises at the first call.
"""

from __future__ import annotations

import ctypes
import math
import os
from pathlib import Path
from typing import NamedTuple

import numpy as np
import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "liblsk.so"

DTYPE_F32 = 0
DTYPE_BF16 = 1
DTYPE_KV8 = 2             # an 8-bit KV cache, where an entry point takes one
EPI_NONE, EPI_RESIDUAL, EPI_SILU_MUL = 0, 1, 2
EPI_PARTIAL, EPI_ARGMAX, EPI_QKV_ROPE = 3, 4, 5   # launch kinds known to lsk_gemm_wide_config
ATTN_SPLIT = 8192         # LSK_ATTN_SPLIT
ATTN_ROWS = 48            # query rows per attention work item (csrc/lsk_attention.hip ATTN_ROWS)
ABI_VERSION = 14

# name -> (restype, argtypes)
_P, _I, _L, _F, _Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float, ctypes.c_size_t
_SIGS = {
    "lsk_last_error": (ctypes.c_char_p, []),
    "lsk_abi_version": (_I, []),
    "lsk_rmsnorm": (_I, [_I, _P, _P, _P, _I, _I, _F, _L, _L, _P]),
    "lsk_rope_append": (_I, [_I, _P, _P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _P]),
    "lsk_kv_append": (_I, [_I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P]),
    "lsk_attn_plan": (_I, [_P, _I, _I, _I, _I, _P, _I, _P, _I, _P, _P, _P]),
    "lsk_attn_rows_cap": (_I, [_P, _I, _I, _I, _I, _I, _I]),
    "lsk_attn_schedule": (_I, [_P, _I, _I, _I, _P, _I, _P]),
    "lsk_pack_segment": (_I, [_P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _L, _P]),
    "lsk_attn_workspace_bytes": (_Z, [_I, _I, _I]),
    "lsk_ragged_attn": (_I, [_I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _P, _I, _I, _I, _P, _I, _I, _I, _I, _F, _P,
                             _Z, _P]),
    "lsk_ragged_attn_static_scratch_bytes": (_Z, []),
    "lsk_ragged_attn_static": (_I, [_I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _P, _I, _I, _I, _P, _I, _I, _I, _I, _F,
                                    _P]),
    "lsk_pack_weight": (_I, [_P, _L, _P, _I, _I, _P]),
    "lsk_unpack_weight": (_I, [_P, _P, _L, _I, _I, _P]),
    "lsk_pack_weight_qkv": (_I, [_P, _L, _P, _I, _I, _I, _I, _P]),
    "lsk_unpack_weight_qkv": (_I, [_P, _P, _L, _I, _I, _I, _I, _P]),
    "lsk_gemm_qkv_rope": (_I, [_P, _P, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _P]),
    "lsk_gemm": (_I, [_I, _P, _L, _P, _L, _P, _L, _P, _L, _I, _I, _I, _I, _I, _P]),
    "lsk_gemm_plan": (_I, [_I, _I, _P, _P]),
    "lsk_gemm_wide_config": (_I, [_I, _I, _I, _I, _I, _I, _P]),
    "lsk_gemm_deep_config": (_I, [_I, _I, _I, _I, _I, _L, _P]),
    "lsk_gemm_partial": (_I, [_P, _L, _P, _L, _P, _I, _I, _I, _I, _P]),
    "lsk_head_workspace_bytes": (_Z, [_I, _I]),
    "lsk_head_argmax": (_I, [_I, _P, _L, _P, _L, _I, _I, _I, _P, _L, _P, _P, _P, _Z, _P]),
    "lsk_head_norm_workspace_bytes": (_Z, [_I, _I, _I]),
    "lsk_head_norm_argmax": (_I, [_I, _P, _L, _P, _F, _P, _L, _I, _I, _I, _P, _L, _P, _P, _P, _Z, _P]),
    "lsk_add_rmsnorm": (_I, [_I, _P, _L, _P, _I, _P, _F, _P, _L, _P, _L, _I, _I, _P]),
    "lsk_rope_append_partial": (_I, [_I, _P, _I, _P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _P]),
    "lsk_embed": (_I, [_P, _L, _L, _P, _L, _P, _P, _P, _I, _P]),
    "lsk_copy_rows": (_I, [_P, _P, _L, _P, _P, _L, _L, _I, _P]),
    "lsk_argmax": (_I, [_I, _P, _L, _I, _I, _P, _P, _P]),
    "lsk_greedy_accept": (_I, [_P, _P, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P]),
    "lsk_kv_rollback": (_I, [_P, _P, _P, _I, _P]),
    "lsk_shift_segment_positions": (_I, [_P, _I, _I, _I, _I, _I, _I, _P, _P, _P, _I, _P]),
    "lsk_probe_matches": (_I, [_P, _P, _P, _P, _P, _I, _I, _P, _P]),
    "lsk_model_create": (_L, [_I, _I, _I, _I, _I, _I, _I, _I, _F] + [_P] * 8 + [_I, _I, _P, _P, _I]),
    "lsk_model_destroy": (_I, [_L]),
    "lsk_segment_workspace_bytes": (_Z, [_L, _I, _I]),
    "lsk_gemm_partial_frag": (_I, [_P, _P, _P, _I, _I, _I, _I, _P]),
    "lsk_gemm_silu_frag": (_I, [_P, _P, _P, _I, _I, _I, _I, _P]),
    "lsk_gemm_residual_frag": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "lsk_forward_layers": (_I, [_L, _P, _P, _I, _I, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P, _Z, _P,
                                ctypes.c_double, ctypes.c_double, _P]),
    "lsk_kv8_append": (_I, [_I, _P, _P, _L, _L] + [_P] * 6 + [_I] * 5 + [_P]),
    "lsk_kv8_read": (_I, [_I] + [_P] * 8 + [_I] * 5 + [_P]),
    "lsk_cache_attn_plan": (_I, [_P] + [_I] * 10 + [_P, _L, _P]),
    "lsk_cache_attn_workspace_bytes": (_Z, [_I, _I, _I, _I]),
    "lsk_kv8_attn": (_I, [_P, _L, _L] + [_P] * 5 + [_I, _P, _I, _I, _P] + [_I] * 6 + [_P] + [_I] * 4 + [_F, _P, _Z,
                          _P]),
    "lsk_tree_attn": (_I, [_I, _P, _L, _L, _P, _P, _P, _I, _P, _I, _I, _P, _I, _I, _P] + [_I] * 6 + [_P] + [_I] * 4 +
                      [_F, _P, _Z, _P]),
    "lsk_tree_masks": (_I, [_P, _P, _P, _I, _I, _I, _P, _I, _P, _P]),
    "lsk_tree_accept": (_I, [_P] * 5 + [_I, _I, _I] + [_P] * 4),
    "lsk_kv_compact": (_I, [_I] + [_P] * 4 + [_I] + [_P] * 4 + [_I] * 6 + [_P]),
    "lsk_prof_enable": (_I, [_I]),
    "lsk_prof_start": (_I, [_I, ctypes.c_double, ctypes.c_double, _P]),
    "lsk_prof_stop": (_I, [_P]),
    "lsk_prof_collect": (_I, [_I, _P, _P, _P, _P]),
}
PROF_CLASSES = ("rmsnorm", "gemm_qkv", "rope_append", "attention", "gemm_o", "gemm_w13", "gemm_w2", "gemm_lm_head",
                "argmax", "glue")
EXPORTS = tuple(_SIGS)

_lib = None


class LskError(RuntimeError):
    pass


def load(path: str | os.PathLike | None = None):
    """Load liblsk.so (once).  Raises if it is missing: there is no CPU fallback."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path is not None else LIB_PATH
    if not p.exists():
        raise LskError(f"{p} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in _SIGS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.lsk_abi_version() != ABI_VERSION:
        raise LskError(f"liblsk ABI {lib.lsk_abi_version()} != {ABI_VERSION}; rebuild")
    if path is None:
        _lib = lib
    return lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = load().lsk_last_error().decode(errors="replace")
        raise LskError(f"{what} failed ({rc}): {msg}")


def _ptr(t) -> int | None:
    if t is None:
        return None
    return t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: int | None = None) -> int:
    """The current HIP stream of device dev, or of the current device (raw handle; the cheap query when torch has it).
    """
    if _raw_stream is not None:
        return _raw_stream(torch._C._cuda_getDevice() if dev is None else dev)
    return torch.cuda.current_stream(dev).cuda_stream


def k_to_frag(k: torch.Tensor) -> torch.Tensor:
    """[..., S, D] -> the bf16 K cache storage [..., S/32, D/16, 64, 8]: per 32-position block, 2 D/32 MFMA
    fragments (a, j) of 1 KiB; lane 16 lg + 4 q + r of fragment (a, j) holds position 8 q + 4 a + r of the
    block and d = 32 j + 8 lg .. +7."""
    *lead, S, D = k.shape
    n = len(lead)
    x = k.reshape(*lead, S // 32, 4, 2, 4, D // 32, 4, 8)          # blk, q, a, r, j, lg, e
    perm = list(range(n)) + [n + i for i in (0, 2, 4, 5, 1, 3, 6)]  # blk, a, j, lg, q, r, e
    return x.permute(*perm).reshape(*lead, S // 32, D // 16, 64, 8).contiguous()


def k_from_frag(kf: torch.Tensor) -> torch.Tensor:
    """bf16 K cache storage [..., S/32, D/16, 64, 8] -> [..., S, D] (a copy)."""
    *lead, nb, nf, _, _ = kf.shape
    n = len(lead)
    D = nf * 16
    x = kf.reshape(*lead, nb, 2, D // 32, 4, 4, 4, 8)               # blk, a, j, lg, q, r, e
    perm = list(range(n)) + [n + i for i in (0, 4, 1, 5, 2, 3, 6)]  # blk, q, a, r, j, lg, e
    return x.permute(*perm).reshape(*lead, nb * 32, D)


def k_dims(kcache: torch.Tensor) -> tuple:
    """(B, Hkv, S, D) of a K cache: fragment-major bf16 storage [B, Hkv, S/32, D/16, 64, 8] or row-major
    [B, Hkv, S, D] (fp32)."""
    if kcache.dim() == 6:
        B, Hkv, nb, nf = kcache.shape[:4]
        return B, Hkv, nb * 32, nf * 16
    return tuple(kcache.shape)


def _check_kcache(dtype: torch.dtype, kcache: torch.Tensor) -> None:
    if dtype == torch.bfloat16 and kcache.dim() != 6:
        raise LskError("bf16 K caches use the fragment-major storage [B, Hkv, S/32, D/16, 64, 8] (k_to_frag)")
    if dtype != torch.bfloat16 and kcache.dim() != 4:
        raise LskError("fp32 K caches are row-major [B, Hkv, S, D]")


def v_to_blocked(v: torch.Tensor) -> torch.Tensor:
    """[..., S, D] -> the V cache storage [..., S/32, D, 32] (32-position blocks, each transposed)."""
    *lead, S, D = v.shape
    return v.reshape(*lead, S // 32, 32, D).transpose(-1, -2).contiguous()


def v_from_blocked(vb: torch.Tensor) -> torch.Tensor:
    """V cache storage [..., S/32, D, 32] -> [..., S, D] (a copy)."""
    *lead, nb, D, b = vb.shape
    return vb.transpose(-1, -2).reshape(*lead, nb * b, D)


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return DTYPE_BF16
    if dtype == torch.float32:
        return DTYPE_F32
    raise LskError(f"unsupported dtype {dtype} (bf16 and fp32 only)")


def _dev(*ts):
    for t in ts:
        if t is not None and t.device.type != "cuda":
            raise LskError(f"liblsk kernels need CUDA (HIP) tensors, got {t.device}")


# ----------------------------------------------------------------------------- weights

class PackedWeight:
    """A bf16 weight matrix [N, K] (F.linear's [out, in]) in the GEMM kernels' fragment-major storage
    (lsk_pack_weight): every 16-row x 32-column MFMA fragment is 1 KiB contiguous in lane order, so each
    wave's weight load is one contiguous 1 KiB stream.  `unpack()` returns the [N, K] tensor (a copy).
    qkv_heads=(n_heads, n_kv_heads, head_dim): a fused [q; k; v] weight stored for the fused qkv + RoPE GEMM
    (lsk_pack_weight_qkv, q and k row groups RoPE-paired); only `gemm_qkv_rope` reads it."""

    def __init__(self, w: torch.Tensor, qkv_heads: tuple | None = None):
        _dev(w)
        if w.dtype != torch.bfloat16 or w.dim() != 2 or w.stride(1) != 1:
            raise LskError("PackedWeight: a 2-D bf16 tensor with unit column stride is needed")
        N, K = w.shape
        self.shape = (N, K)
        self.dtype = w.dtype
        self.device = w.device
        self.qkv_heads = tuple(qkv_heads) if qkv_heads is not None else None
        self.data = torch.empty(N * K, dtype=w.dtype, device=w.device)
        if self.qkv_heads is None:
            _check(load().lsk_pack_weight(_ptr(w), w.stride(0), _ptr(self.data), N, K, _stream()), "lsk_pack_weight")
        else:
            hq, hkv, d = self.qkv_heads
            if N != (hq + 2 * hkv) * d:
                raise LskError(f"PackedWeight: {N} rows do not match qkv heads {self.qkv_heads}")
            _check(load().lsk_pack_weight_qkv(_ptr(w), w.stride(0), _ptr(self.data), hq, hkv, d, K, _stream()),
                   "lsk_pack_weight_qkv")

    def data_ptr(self) -> int:
        return self.data.data_ptr()

    def stride(self, dim: int) -> int:
        return self.shape[1] if dim == 0 else 1

    def dim(self) -> int:
        return 2

    def numel(self) -> int:
        return self.shape[0] * self.shape[1]

    def element_size(self) -> int:
        return 2

    def unpack(self) -> torch.Tensor:
        N, K = self.shape
        out = torch.empty(N, K, dtype=self.dtype, device=self.device)
        if getattr(self, "qkv_heads", None) is None:
            _check(load().lsk_unpack_weight(_ptr(self.data), _ptr(out), K, N, K, _stream()), "lsk_unpack_weight")
        else:
            hq, hkv, d = self.qkv_heads
            _check(load().lsk_unpack_weight_qkv(_ptr(self.data), _ptr(out), K, hq, hkv, d, K, _stream()),
                   "lsk_unpack_weight_qkv")
        return out

    def __repr__(self) -> str:
        return f"PackedWeight(shape={self.shape}, dtype={self.dtype}, device={self.device})"


GEMM_TOKEN_TILE = 64       # tokens per GEMM token tile: launches of up to this many rows read each weight once


def as_gemm_weight(w: torch.Tensor):
    """The storage the GEMMs read for a weight of this dtype: PackedWeight for bf16, the tensor for fp32."""
    return PackedWeight(w) if w.dtype == torch.bfloat16 else w.contiguous()


def _check_weight(a: torch.Tensor, w) -> None:
    if a.dtype == torch.bfloat16 and not isinstance(w, PackedWeight):
        raise LskError("bf16 GEMMs read packed weights: wrap the [out, in] tensor in PackedWeight")
    if a.dtype != torch.bfloat16 and isinstance(w, PackedWeight):
        raise LskError("packed weights are bf16 only")
    if isinstance(w, PackedWeight) and getattr(w, "qkv_heads", None) is not None:
        raise LskError("a qkv weight packed for the fused qkv + RoPE GEMM is read by gemm_qkv_rope only (its rows are "
                       "RoPE-paired); PackedWeight(w.unpack()) gives the plain storage")


# ----------------------------------------------------------------------------- ops

def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    _dev(x, w)
    assert x.dim() == 2 and x.stride(1) == 1 and w.is_contiguous() and w.numel() == x.shape[1]
    if out is None:
        out = torch.empty_like(x)
    _check(load().lsk_rmsnorm(dtype_code(x.dtype), _ptr(x), _ptr(w), _ptr(out), x.shape[0], x.shape[1], float(eps),
                              x.stride(0), out.stride(0), _stream()), "lsk_rmsnorm")
    return out


def rope_append(qkv, q_out, kcache, vcache, cos_tab, sin_tab, rows_i32, pos_i32, n_heads, n_kv_heads, head_dim):
    """kcache: K cache storage (k_dims); vcache: the blocked-transposed V storage [B, Hkv, S/32, D, 32]."""
    _dev(qkv, q_out, kcache, vcache, cos_tab, sin_tab, rows_i32, pos_i32)
    _check_kcache(q_out.dtype, kcache)
    N = qkv.shape[0]
    B, Hkv, S, D = k_dims(kcache)
    assert qkv.is_contiguous() and q_out.is_contiguous() and kcache.is_contiguous() and vcache.is_contiguous()
    assert cos_tab.dtype == torch.float32 and cos_tab.is_contiguous() and cos_tab.shape[1] == head_dim
    _check(load().lsk_rope_append(dtype_code(qkv.dtype), _ptr(qkv), _ptr(q_out), _ptr(kcache), _ptr(vcache),
                                  _ptr(cos_tab), _ptr(sin_tab), cos_tab.shape[0], _ptr(rows_i32), _ptr(pos_i32), N,
                                  n_heads, n_kv_heads, head_dim, B, S, _stream()), "lsk_rope_append")


def kv_append(k, v, kcache, vcache, rows_i32, pos_i32):
    """kcache: K cache storage (k_dims); vcache: the blocked-transposed V storage [B, Hkv, S/32, D, 32]."""
    _dev(k, v, kcache, vcache, rows_i32, pos_i32)
    _check_kcache(k.dtype, kcache)
    B, Hkv, S, D = k_dims(kcache)
    assert k.is_contiguous() and v.is_contiguous() and k.shape[1:] == (Hkv, D)
    _check(load().lsk_kv_append(dtype_code(k.dtype), _ptr(k), _ptr(v), _ptr(kcache), _ptr(vcache), _ptr(rows_i32),
                                _ptr(pos_i32), k.shape[0], Hkv, D, B, S, _stream()), "lsk_kv_append")


def attn_plan(blocks: np.ndarray, group: int, split: int, rows_cap: int = ATTN_ROWS):
    """blocks int32 [nb, 4] = (q_start, pos0, T, row) -> (works [n,8], groups [n,8], n_parts); work items of at
    most rows_cap (16, 32 or 48) query rows."""
    blocks = np.ascontiguousarray(blocks, dtype=np.int32)
    nb = blocks.shape[0]
    rows = int(((blocks[:, 2].astype(np.int64) * group + rows_cap - 1) // max(rows_cap, 1)).sum()) if nb else 0
    max_ctx = int((blocks[:, 1].astype(np.int64) + blocks[:, 2]).max()) if nb else 0
    max_works = 8 * max(1, rows * max(1, (max_ctx + split - 1) // split)) + 64   # XCD-order padding
    max_groups = max(1, rows)
    works = np.zeros((max_works, 8), dtype=np.int32)
    groups = np.zeros((max_groups, 8), dtype=np.int32)
    nw, ng, npart = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    _check(load().lsk_attn_plan(blocks.ctypes.data, nb, group, split, rows_cap, works.ctypes.data, max_works,
                                groups.ctypes.data, max_groups, ctypes.byref(nw), ctypes.byref(ng),
                                ctypes.byref(npart)), "lsk_attn_plan")
    return works[:nw.value], groups[:ng.value], npart.value


def attn_rows_cap(blocks: np.ndarray, group: int, split: int, n_kv_heads: int, head_dim: int, n_slots: int) -> int:
    """Rows per attention work item (16, 32 or 48) for a launch of these blocks over n_slots workgroups."""
    blocks = np.ascontiguousarray(blocks, dtype=np.int32)
    rc = load().lsk_attn_rows_cap(blocks.ctypes.data if len(blocks) else None, len(blocks), group, split,
                                  n_kv_heads, head_dim, n_slots)
    if rc < 0:
        _check(rc, "lsk_attn_rows_cap")
    return rc


_CU_COUNT: dict = {}


def cu_count(device) -> int:
    """Compute units of the device (the persistent attention kernel runs one workgroup per CU); 256 (MI355X)
    for a non-CUDA device, where plans are only built, never run."""
    device = torch.device(device)
    if device.type != "cuda":
        return 256
    idx = device.index if device.index is not None else torch.cuda.current_device()
    n = _CU_COUNT.get(idx)
    if n is None:
        n = _CU_COUNT[idx] = int(torch.cuda.get_device_properties(idx).multi_processor_count)
    return n


def attn_schedule(works: np.ndarray, n_kv_heads: int, n_slots: int):
    """Static longest-first schedule of (work, KV head) items over n_slots persistent workgroups
    -> (recs int32 [n_slots * n_rounds * 8], n_rounds): slot s's records are recs[s * n_rounds * 8 ...]."""
    works = np.ascontiguousarray(works, dtype=np.int32)
    lib = load()
    wp = works.ctypes.data if len(works) else None
    R = ctypes.c_int(0)
    _check(lib.lsk_attn_schedule(wp, len(works), n_kv_heads, n_slots, None, 0, ctypes.byref(R)), "lsk_attn_schedule")
    recs = np.zeros(max(n_slots * R.value * 8, 8), dtype=np.int32)
    _check(lib.lsk_attn_schedule(wp, len(works), n_kv_heads, n_slots, recs.ctypes.data, n_slots * R.value,
                                 ctypes.byref(R)), "lsk_attn_schedule")
    return recs[:n_slots * R.value * 8], R.value


_PACK_BUF = [np.zeros(1 << 16, dtype=np.int32)]
_PACK_COUNTS = np.zeros(11, dtype=np.int64)


def pack_segment(rows: np.ndarray, pos0: np.ndarray, T: np.ndarray, group: int, split: int, n_kv_heads: int,
                 head_dim: int, n_slots: int, bucketing: int, max_batch: int, max_seq: int, rope_len: int):
    """lsk_pack_segment over int64 block arrays in packed order -> (meta int32 [meta_len] (a fresh array),
    counts (N, n_works, n_groups, n_parts, n_rounds, meta_len, kv_read, kv_read_padded, kv_gathered, pairs,
    rows_cap)).
    Out-of-range blocks raise ValueError (the reference's build_packed behaviour)."""
    lib = load()
    nb = len(T)
    r = rows if rows.dtype == np.int64 and rows.flags.c_contiguous else np.ascontiguousarray(rows, dtype=np.int64)
    p = pos0 if pos0.dtype == np.int64 and pos0.flags.c_contiguous else np.ascontiguousarray(pos0, dtype=np.int64)
    t = T if T.dtype == np.int64 and T.flags.c_contiguous else np.ascontiguousarray(T, dtype=np.int64)
    cnt = _PACK_COUNTS
    for _ in range(2):
        buf = _PACK_BUF[0]
        rc = lib.lsk_pack_segment(r.ctypes.data, p.ctypes.data, t.ctypes.data, nb, group, split, n_kv_heads,
                                  head_dim, n_slots, bucketing, max_batch, max_seq, rope_len, buf.ctypes.data,
                                  buf.size, cnt.ctypes.data)
        if rc == -4:                                   # LSK_EWORKSPACE: grow to the reported length and retry
            _PACK_BUF[0] = np.zeros(int(cnt[5]) * 2, dtype=np.int32)
            continue
        if rc == -2:
            raise ValueError(lib.lsk_last_error().decode())
        _check(rc, "lsk_pack_segment")
        c = cnt.tolist()
        return buf[:c[5]].copy(), tuple(c)
    raise LskError("lsk_pack_segment: metadata buffer")


def attn_workspace_bytes(n_parts: int, n_kv_heads: int, head_dim: int) -> int:
    return int(load().lsk_attn_workspace_bytes(n_parts, n_kv_heads, head_dim))


def ragged_attn(q, kcache, vcache, blocks_dev, works_dev, n_works, groups_dev, n_groups, n_parts, out, n_heads,
                scale, workspace=None, recs_dev=None, n_rounds=0, n_slots=0, rows_cap=ATTN_ROWS):
    """kcache: K cache storage (k_dims); vcache: the blocked-transposed V storage [B, Hkv, S/32, D, 32];
    rows_cap: the cap the plan was made with."""
    _dev(q, kcache, vcache, blocks_dev, works_dev, out)
    _check_kcache(q.dtype, kcache)
    B_, H_, S_, D_ = k_dims(kcache)
    assert vcache.shape == (B_, H_, S_ // 32, D_, 32) and S_ % 64 == 0
    B, Hkv, S, D = k_dims(kcache)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _check(load().lsk_ragged_attn(dtype_code(q.dtype), _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(blocks_dev),
                                  _ptr(works_dev), n_works, _ptr(groups_dev), n_groups, n_parts, _ptr(recs_dev),
                                  n_rounds, n_slots, rows_cap, _ptr(out), n_heads, Hkv, D, S, float(scale),
                                  _ptr(workspace), ws_bytes, _stream()), "lsk_ragged_attn")


def ragged_attn_static(q, kcache, vcache, blocks_dev, works_dev, n_works, groups_dev, n_groups, n_parts, out,
                       n_heads, scale, recs_dev=None, n_rounds=0, n_slots=0, rows_cap=ATTN_ROWS):
    """ragged_attn without a workspace: the split partials live in the library's static per-GPU scratch array
    (lsk_ragged_attn_static; plans needing more than lsk_ragged_attn_static_scratch_bytes() raise)."""
    _dev(q, kcache, vcache, blocks_dev, works_dev, out)
    _check_kcache(q.dtype, kcache)
    B, Hkv, S, D = k_dims(kcache)
    assert vcache.shape == (B, Hkv, S // 32, D, 32) and S % 64 == 0
    _check(load().lsk_ragged_attn_static(dtype_code(q.dtype), _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(blocks_dev),
                                         _ptr(works_dev), n_works, _ptr(groups_dev), n_groups, n_parts,
                                         _ptr(recs_dev), n_rounds, n_slots, rows_cap, _ptr(out), n_heads, Hkv, D, S,
                                         float(scale), _stream()), "lsk_ragged_attn_static")


def gemm(a: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
         epilogue: int = EPI_NONE) -> torch.Tensor:
    _dev(a, w, out, residual)
    _check_weight(a, w)
    assert a.dim() == 2 and w.dim() == 2 and a.stride(1) == 1 and w.stride(1) == 1
    M, K = a.shape
    if epilogue == EPI_SILU_MUL:
        N = w.shape[0] // 2
        ffn = N
    else:
        N = w.shape[0]
        ffn = 0
    if out is None:
        out = torch.empty(M, N, dtype=a.dtype, device=a.device)
    ldr = residual.stride(0) if residual is not None else 0
    _check(load().lsk_gemm(dtype_code(a.dtype), _ptr(a), a.stride(0), _ptr(w), w.stride(0), _ptr(out), out.stride(0),
                           _ptr(residual), ldr, M, N, K, epilogue, ffn, _stream()), "lsk_gemm")
    return out


def embed(table: torch.Tensor, alt_ids: torch.Tensor, out: torch.Tensor, seq_buf: torch.Tensor | None = None,
          sel: torch.Tensor | None = None) -> torch.Tensor:
    _dev(table, alt_ids, out, seq_buf, sel)
    n = alt_ids.numel()
    row_bytes = table.shape[1] * table.element_size()
    _check(load().lsk_embed(_ptr(table), table.shape[0], row_bytes, _ptr(seq_buf),
                            seq_buf.numel() if seq_buf is not None else 0, _ptr(sel), _ptr(alt_ids), _ptr(out), n,
                            _stream()), "lsk_embed")
    return out


def copy_rows(dst: torch.Tensor, dst_idx, src: torch.Tensor, src_idx, n: int) -> None:
    _dev(dst, src, dst_idx, src_idx)
    row_bytes = dst[0].numel() * dst.element_size()
    assert src[0].numel() * src.element_size() == row_bytes
    _check(load().lsk_copy_rows(_ptr(dst), _ptr(dst_idx), dst.shape[0], _ptr(src), _ptr(src_idx), src.shape[0],
                                row_bytes, n, _stream()), "lsk_copy_rows")


def argmax(logits: torch.Tensor, out: torch.Tensor, dst_idx: torch.Tensor | None = None, n_rows: int | None = None):
    _dev(logits, out, dst_idx)
    n = logits.shape[0] if n_rows is None else n_rows
    _check(load().lsk_argmax(dtype_code(logits.dtype), _ptr(logits), logits.stride(0), n, logits.shape[1], _ptr(out),
                             _ptr(dst_idx), _stream()), "lsk_argmax")
    return out


def greedy_accept(Yv, seq_buf, Dm1, slots, starts, Ts, forced, nv, acc_out, y_out, kv_len=None):
    _dev(Yv, seq_buf, slots, starts, Ts, forced, acc_out, y_out, kv_len)
    _check(load().lsk_greedy_accept(_ptr(Yv), _ptr(seq_buf), Dm1, _ptr(slots), _ptr(starts), _ptr(Ts), _ptr(forced),
                                    nv, _ptr(acc_out), _ptr(y_out), _ptr(kv_len), _stream()), "lsk_greedy_accept")


def probe_matches(pred, Yv, acc, blk_i32, jl_i32, nc: int, nvt: int, out) -> None:
    _dev(pred, Yv, acc, blk_i32, jl_i32, out)
    _check(load().lsk_probe_matches(_ptr(pred), _ptr(Yv), _ptr(acc), _ptr(blk_i32), _ptr(jl_i32), nc, nvt, _ptr(out),
                                    _stream()), "lsk_probe_matches")


def kv_rollback(kv_len, slots, accepted, nv):
    _dev(kv_len, slots, accepted)
    _check(load().lsk_kv_rollback(_ptr(kv_len), _ptr(slots), _ptr(accepted), nv, _stream()), "lsk_kv_rollback")


def shift_segment_positions(meta, n_tokens: int, nb: int, n_works: int, n_groups: int, n_recs: int, group: int,
                            accepted, vslots, vdrafts, nv: int) -> None:
    """lsk_shift_segment_positions on a segment's device metadata `meta` (int32, pack_segment's layout; n_recs =
    n_slots * n_rounds of its plan): blocks in cache row vslots[j] planned vdrafts[j] - accepted[j] positions ahead
    move back to their actual positions (accepted: the device acc_out of greedy_accept)."""
    _dev(meta, accepted, vslots, vdrafts)
    _check(load().lsk_shift_segment_positions(_ptr(meta), n_tokens, nb, n_works, n_groups, n_recs, group,
                                              _ptr(accepted), _ptr(vslots), _ptr(vdrafts), nv, _stream()),
           "lsk_shift_segment_positions")


# ----------------------------------------------------------------------------- 8-bit cache and trees of drafted tokens

def _one_device(first: torch.Tensor, *ts) -> int:
    """The index of the device that all the tensors are on (None is skipped); LskError otherwise."""
    dev = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            dev = -1
            break
    if dev < 0:
        _dev(first, *ts)
        devs = {str(t.device) for t in (first, *ts) if t is not None}
        raise LskError(f"tensors on different devices: {sorted(devs)}")
    return dev


def _launch(dev: int, what: str, *args) -> None:
    """Calls `what` with args and device dev's current stream; dev is the current device for the call."""
    fn = getattr(load(), what)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, _stream())
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream())
    if rc:
        _check(rc, what)


def _want(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise LskError(f"{what}: {name} must be a contiguous {list(shape)} {dtype} tensor, got {list(t.shape)} "
                       f"{t.dtype}{'' if t.is_contiguous() else ', not contiguous'}")


_E4M3 = torch.float8_e4m3fn


class _KV8(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    ks: torch.Tensor
    vs: torch.Tensor


class KV8(_KV8):
    """An 8-bit K / V cache (lsk_kv8_append): e4m3 codes and one power-of-two scale per position and KV head, the byte
    e + 127.  A layer's tensors, or with a leading layer axis those of several:
      k [B, Hkv, S/64, 4, D/64, 64, 16] and v [B, Hkv, S/64, D, 64] float8_e4m3fn, ks and vs [B, Hkv, S] uint8.
    The tensors' types and shapes are checked by the object's first use; they have to stay as they are."""
    _checked = None                                   # (layers, dims) that the tensors were found to fit

    @classmethod
    def zeros(cls, max_batch: int, n_kv_heads: int, max_seq: int, head_dim: int, device, layers: int | None = None):
        if head_dim not in (64, 128) or max_seq % 64 or max_seq <= 0:
            raise ValueError(f"8-bit caches need head_dim 64 or 128 and max_seq a multiple of 64 (got {head_dim}, "
                             f"{max_seq})")
        lead = (max_batch, n_kv_heads) if layers is None else (layers, max_batch, n_kv_heads)
        codes = dict(dtype=torch.uint8, device=device)
        return cls(torch.zeros(*lead, max_seq // 64, 4, head_dim // 64, 64, 16, **codes).view(torch.float8_e4m3fn),
                   torch.zeros(*lead, max_seq // 64, head_dim, 64, **codes).view(torch.float8_e4m3fn),
                   torch.full((*lead, max_seq), 127, **codes), torch.full((*lead, max_seq), 127, **codes))

    def layer(self, i: int) -> "KV8":
        return KV8(self.k[i], self.v[i], self.ks[i], self.vs[i])

    @property
    def dims(self) -> tuple:
        """(B, Hkv, S, D)"""
        *_, B, Hkv, S = self.ks.shape
        return B, Hkv, S, self.v.shape[-2]

    def ptrs(self) -> tuple:
        k, v, ks, vs = self
        return k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()

    def check(self, what: str, layers: bool = False) -> tuple:
        """(B, Hkv, S, D) of a cache of the documented storage; LskError otherwise."""
        if self._checked is not None and self._checked[0] == layers:
            return self._checked[1]
        k, v, ks, vs = self
        lead, v_shape, n = ks.shape, v.shape, 4 if layers else 3
        if len(lead) != n or len(v_shape) != n + 2:
            raise LskError(f"{what}: an 8-bit cache of {'several layers' if layers else 'one layer'} is needed")
        S, D = lead[-1], v_shape[-2]
        if D not in (64, 128) or S % 64 or S == 0:
            raise LskError(f"{what}: 8-bit caches need head_dim 64 or 128 and max_seq a multiple of 64 (got {D}, {S})")
        blocks = (*lead[:-1], S // 64)
        want_k, want_v = (*blocks, 4, D // 64, 64, 16), (*blocks, D, 64)
        if not (k.shape == want_k and v_shape == want_v and vs.shape == lead and k.dtype is v.dtype is _E4M3 and
                ks.dtype is vs.dtype is torch.uint8 and k.is_contiguous() and v.is_contiguous() and
                ks.is_contiguous() and vs.is_contiguous()):
            _want(what, "k codes", k, _E4M3, want_k)
            _want(what, "v codes", v, _E4M3, want_v)
            _want(what, "k exponents", ks, torch.uint8, lead)
            _want(what, "v exponents", vs, torch.uint8, lead)
        self._checked = layers, (lead[-3], lead[-2], S, D)
        return self._checked[1]


def kv8_append(k: torch.Tensor, v: torch.Tensor, cache: KV8, rows_i32: torch.Tensor, pos_i32: torch.Tensor) -> None:
    """k, v [N, Hkv, D] (bf16 or fp32, of equal strides; dims contiguous) quantised into a layer's 8-bit cache at
    (rows, pos).  Tokens outside the cache are skipped; the (row, position) pairs of a call have to differ."""
    dev = _one_device(k, v, *cache, rows_i32, pos_i32)
    B, Hkv, S, D = cache.check("kv8_append")
    n = k.shape[0]
    if k.shape != (n, Hkv, D) or v.shape != k.shape or v.dtype != k.dtype:
        raise LskError(f"kv8_append: k and v must be [N, {Hkv}, {D}] of one dtype, got {list(k.shape)} {k.dtype} and "
                       f"{list(v.shape)} {v.dtype}")
    st_t, st_h, st_d = k.stride()
    if n and (st_d != 1 or v.stride() != (st_t, st_h, st_d)):
        raise LskError("kv8_append: k and v need contiguous dims and the same strides")
    _want("kv8_append", "rows", rows_i32, torch.int32, (n,))
    _want("kv8_append", "pos", pos_i32, torch.int32, (n,))
    code = dtype_code(k.dtype)
    if n == 0:
        return
    _launch(dev, "lsk_kv8_append", code, k.data_ptr(), v.data_ptr(), st_t, st_h, *cache.ptrs(), rows_i32.data_ptr(),
            pos_i32.data_ptr(), n, Hkv, D, B, S)


def kv8_read(cache: KV8, rows_i32: torch.Tensor, pos_i32: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             out: tuple | None = None) -> tuple:
    """The K and V that a layer's 8-bit cache holds at (rows, pos): two [N, Hkv, D] tensors (bf16: exactly); zeros for
    tokens outside the cache."""
    dev = _one_device(*cache, rows_i32, pos_i32, *(out or ()))
    B, Hkv, S, D = cache.check("kv8_read")
    n = rows_i32.numel()
    _want("kv8_read", "rows", rows_i32, torch.int32, (n,))
    _want("kv8_read", "pos", pos_i32, torch.int32, (n,))
    code = dtype_code(dtype if out is None else out[0].dtype)
    if out is None:
        out = cache.ks.new_empty(n, Hkv, D, dtype=dtype), cache.ks.new_empty(n, Hkv, D, dtype=dtype)
    else:
        if len(out) != 2:
            raise LskError("kv8_read: out is a pair of tensors")
        for t in out:
            _want("kv8_read", "out", t, out[0].dtype, (n, Hkv, D))
    if n:
        _launch(dev, "lsk_kv8_read", code, *cache.ptrs(), rows_i32.data_ptr(), pos_i32.data_ptr(), out[0].data_ptr(),
                out[1].data_ptr(), n, Hkv, D, B, S)
    return out


def cache_attn_split(max_batch: int, n_kv_heads: int, max_seq: int, tree: bool = False) -> int:
    """KV positions per attention split of a cache: fixed by the cache, so that a row's result never depends on the
    batch it is in.  The longest context in as many splits as make about one work item per CU out of the cache's
    (row, KV head) stripes, but each long enough to pay for the merge: 800 positions, 2048 from 128 stripes on (32 / 8
    heads of 64, one token, 1 request: 1000 positions 7.2 us whole, 11.0 in two; 5000 positions 15.8 whole, 10.8 in
    five).  Trees, whose partial outputs are many rows: 1280 positions, 2048 from 32 stripes on (64 nodes, 32 / 8 heads
    of 128: 4 requests of 1000 positions 14 us whole, 28 in two, of 5000 positions 37 and 42 in three; 1 request of 5000
    positions 33 whole, 21 in three).  512 to 8192 positions, at most 128 splits.  256: MI355X's CUs, as a constant, so
    that a row's bits are the same on every device.  The rule does not see a prompt, whose many rows need no splits: its
    plan is better given one (one prompt of 4001 tokens in a cache of its own, 32 / 8 heads of 128: 396 us and a
    workspace of 181 MB at 832 positions, 248 us and none at 8192)."""
    stripes = max_batch * n_kv_heads
    if tree:
        n = min(256 // stripes, max_seq // (1280 if stripes < 32 else 2048))
    else:
        n = min(256 // stripes, max_seq // (800 if stripes < 128 else 2048))
    split = min(max(-(-max_seq // max(n, 1)), 512), ATTN_SPLIT)
    return (max(split, -(-max_seq // 128)) + 63) // 64 * 64


class _Launch:
    """One lsk_cache_attn_plan on the device, and its arguments of a launch."""

    def __init__(self, groups: torch.Tensor, recs: torch.Tensor, n_groups: int, n_parts: int, n_rounds: int,
                 n_slots: int, n_shared: int, tiles: int, row_groups: int, part_rows: int, ws_bytes: int):
        self.groups, self.recs, self.n_groups, self.n_parts, self.n_rounds = groups, recs, n_groups, n_parts, n_rounds
        self.n_slots, self.n_shared, self.tiles, self.row_groups, self.part_rows, self.ws_bytes = \
            n_slots, n_shared, tiles, row_groups, part_rows, ws_bytes
        self.n_items = n_rounds + n_shared           # (0: nothing to launch)
        self.args = (_ptr(groups), n_groups, n_parts, _ptr(recs), n_rounds, n_slots, n_shared, tiles, row_groups,
                     part_rows)


class AttnPlan:
    """The plan of attention launches over packed blocks, shared by the layers of a segment.  blocks: int [nb, 4] =
    (q_start, pos0, T, row) with q_start the running sum of T; cache: a layer's KV8, or the K storage of a bf16 or fp32
    cache.  split: KV positions per split (cache_attn_split unless given; fp32 does not split); row_groups: a tree's at
    most (by the cache and the block unless given).  tree: which launches it is for, with a mask (True), without (False)
    or, over an 8-bit cache, either (None), which takes twice as long (256 requests: 333 us for 129).
    Its records go to the GPU on the current stream.  A launch on another stream waits for them, and they outlive it
    when the plan is dropped; a captured launch reads them with every replay: the plan is made before the capture and
    kept as long as the graph."""

    def __init__(self, blocks, n_heads: int, cache, split: int | None = None, row_groups: int | None = None,
                 tree: bool | None = None):
        self.kv8 = isinstance(cache, KV8)
        kcache = cache.k if self.kv8 else cache
        self.dims = B, Hkv, S, D = cache.dims if self.kv8 else k_dims(cache)
        self.dtype, self.device = kcache.dtype, kcache.device
        if n_heads <= 0 or n_heads % Hkv:
            raise ValueError(f"{n_heads} query heads over {Hkv} KV heads")
        b = np.asarray(blocks, dtype=np.int64).reshape(-1, 4)
        if len(b) and (not np.array_equal(b[:, 0], np.cumsum(b[:, 2]) - b[:, 2]) or (b[:, 1:3] < 0).any()):
            raise ValueError("blocks: q_start must be the running sum of T, pos0 and T not negative")
        if len(b) and ((b[:, 3] < 0) | (b[:, 3] >= B) | (b[:, 1] + b[:, 2] > S)).any():
            raise ValueError(f"a block lies outside the cache's {B} rows x {S} positions")
        if (split is not None and (split < 64 or split % 64)) or len(b) and int(b[:, 2].sum()) >= 1 << 30:
            raise ValueError(f"a split of {split} positions (a multiple of 64), or too many tokens")
        self.n_heads, self.n_tokens = n_heads, int(b[:, 2].sum())
        self.q_shape, self.width, self.scale = (self.n_tokens, n_heads, D), n_heads * D, 1.0 / math.sqrt(D)
        self.index = self.device.index if self.device.index is not None else -1
        b = np.ascontiguousarray(b, dtype=np.int32)
        group, n_slots = n_heads // Hkv, 2 * cu_count(self.device)    # (two workgroups fit a CU)
        self._buffers, self._uploaded, self._streams = [], None, set()
        self.works = self.causal = self.tree = None
        self.rows_cap = self.n_works = 0
        if self.dtype == torch.float32:
            self.split, self.rows_cap = 1 << 30, 16
            works, _, _ = attn_plan(b, group, self.split, self.rows_cap)
            self.works, self.n_works = self._upload(works.ravel()), len(works)
            self._mark_uploaded()
            return
        self.split, self.tree_split = (split if split is not None else cache_attn_split(B, Hkv, S, t)
                                       for t in (False, True))
        rg = 0 if row_groups is None else row_groups
        if self.kv8 and not tree:
            self.causal = self._plan(b, group, self.split, False, 1, n_slots)
        if tree or tree is None:
            self.tree = self._plan(b, group, self.tree_split, True, rg, n_slots)
        self._mark_uploaded()

    def _upload(self, words: np.ndarray) -> torch.Tensor:
        t = torch.from_numpy(words)
        if self.device.type != "cuda":
            return t
        if torch.cuda.is_current_stream_capturing():
            raise LskError("a plan is made before a capture begins (its upload would be replayed from freed memory)")
        self._buffers.append(t.pin_memory().to(self.device, non_blocking=True))
        return self._buffers[-1]

    def _mark_uploaded(self) -> None:
        if self.device.type == "cuda":
            stream = torch.cuda.current_stream(self.device)
            self._uploaded = stream.record_event()
            self._streams.add(stream.cuda_stream)

    def _join(self, dev: int) -> None:
        """Before a first launch on device dev's current stream: that stream waits for the records, and they outlive it.
        """
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                if not self._uploaded.query():       # (a capture cannot wait for work outside it)
                    raise LskError("the plan's upload has not ended: synchronize before the capture begins")
                return
            stream = torch.cuda.current_stream()
            stream.wait_event(self._uploaded)
            for t in self._buffers:
                t.record_stream(stream)
            self._streams.add(stream.cuda_stream)

    def _plan(self, b: np.ndarray, group: int, split: int, tree: bool, row_groups: int, n_slots: int) -> _Launch:
        lib, cnt = load(), np.zeros(9, dtype=np.int64)
        B, Hkv, _, D = self.dims
        args = (b.ctypes.data if len(b) else None, len(b), group, split, B, Hkv, D, int(self.kv8), int(tree),
                row_groups, n_slots)
        _check(lib.lsk_cache_attn_plan(*args, None, 0, cnt.ctypes.data), "lsk_cache_attn_plan")
        meta = np.zeros(max(int(cnt[6]), 1), dtype=np.int32)
        _check(lib.lsk_cache_attn_plan(*args, meta.ctypes.data, meta.size, cnt.ctypes.data), "lsk_cache_attn_plan")
        _, ng, parts, rounds, tiles, part_rows, _, used, shared = (int(x) for x in cnt)
        dev = self._upload(meta)
        ws = int(lib.lsk_cache_attn_workspace_bytes(parts, Hkv, part_rows, D)) if parts else 0
        return _Launch(dev[:ng * 8], dev[ng * 8:], ng, parts, rounds, n_slots, shared, tiles, used, part_rows,
                       ws)


def _plan_call(what: str, dev: int, q: torch.Tensor, plan: AttnPlan, launch, dims: tuple, kv8: bool,
               dtype: torch.dtype, mask, scale, out, workspace):
    """Checks shared by kv8_attn and tree_attn, and the plan joined; returns (scale, out, workspace, its bytes)."""
    if dev != plan.index:
        raise LskError(f"{what}: the plan is on {plan.device}, the tensors on cuda:{dev}")
    if plan.dims != dims or plan.kv8 != kv8 or plan.dtype is not dtype:
        raise LskError(f"{what}: the plan was made for another cache ({plan.dims} {plan.dtype})")
    if launch is None and dtype != torch.float32:
        raise LskError(f"{what}: the plan was made for launches {'without' if mask is not None else 'with'} a mask")
    want = torch.bfloat16 if kv8 else dtype
    n, width = plan.n_tokens, plan.width
    if q.shape != plan.q_shape or q.dtype is not want or (n and q.stride(2) != 1):
        raise LskError(f"{what}: q must be {list(plan.q_shape)} {want} with contiguous dims, got {list(q.shape)} "
                       f"{q.dtype}")
    if mask is not None:
        if mask.dim() != 2 or mask.shape[1] < 1:
            raise LskError(f"{what}: mask must be [{n}, words]")
        _want(what, "mask", mask, torch.int32, (n, mask.shape[1]))
    if out is None:
        out = q.new_empty(n, width)
    else:
        _want(what, "out", out, want, (n, width))
    if workspace is None:
        if launch is not None and launch.ws_bytes:
            workspace = q.new_empty(launch.ws_bytes, dtype=torch.uint8)
    elif not workspace.is_contiguous():
        raise LskError(f"{what}: the workspace must be contiguous")
    ws_bytes = workspace.nbytes if workspace is not None else 0
    if _stream(dev) not in plan._streams:
        plan._join(dev)
    return plan.scale if scale is None else float(scale), out, workspace, ws_bytes


def kv8_attn(q: torch.Tensor, cache: KV8, plan: AttnPlan, mask: torch.Tensor | None = None, scale: float | None = None,
             out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Ragged verify / decode attention over a layer's 8-bit cache (lsk_kv8_attn): q [N, Hq, D] bf16 -> [N, Hq * D].
    mask (int32 [N, words], tree_masks): blocks are trees of drafted tokens.  scale: 1 / sqrt(D) unless given.  Without
    a workspace one is taken from torch's allocator for the call."""
    p = plan.causal if mask is None else plan.tree
    dev = _one_device(q, *cache, mask, out, workspace)
    dims = _, Hkv, S, D = cache.check("kv8_attn")
    scale, out, workspace, ws = _plan_call("kv8_attn", dev, q, plan, p, dims, True, _E4M3, mask, scale, out, workspace)
    if p.n_items:
        st_t, st_h, _ = q.stride()
        masked = (None, 0) if mask is None else (mask.data_ptr(), mask.shape[1])
        _launch(dev, "lsk_kv8_attn", q.data_ptr(), st_t, st_h, *cache.ptrs(), *masked, *p.args, out.data_ptr(),
                plan.n_heads, Hkv, D, S, scale, _ptr(workspace), ws)
    return out


def tree_attn(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, plan: AttnPlan, mask: torch.Tensor,
              scale: float | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of trees of drafted tokens over a layer's bf16 or fp32 cache (lsk_tree_attn): q [N, Hq, D] ->
    [N, Hq * D].  kcache: K cache storage (k_dims); vcache: the blocked-transposed V storage; mask: int32 [N, words]
    (tree_masks).  scale: 1 / sqrt(D) unless given."""
    p = plan.tree
    dev = _one_device(q, kcache, vcache, mask, out, workspace)
    _check_kcache(kcache.dtype, kcache)
    code = dtype_code(kcache.dtype)
    dims = B, Hkv, S, D = k_dims(kcache)
    if not kcache.is_contiguous():
        raise LskError("tree_attn: the K cache must be contiguous")
    _want("tree_attn", "V cache", vcache, kcache.dtype, (B, Hkv, S // 32, D, 32))
    scale, out, workspace, ws = _plan_call("tree_attn", dev, q, plan, p, dims, False, kcache.dtype, mask, scale, out,
                                           workspace)
    if p.n_items if p is not None else plan.n_works:
        args = p.args if p is not None else (None, 0, 0, None, 0, 0, 0, 0, 0, 0)
        st_t, st_h, _ = q.stride()
        _launch(dev, "lsk_tree_attn", code, q.data_ptr(), st_t, st_h, kcache.data_ptr(), vcache.data_ptr(),
                mask.data_ptr(), mask.shape[1], _ptr(plan.works), plan.n_works, plan.rows_cap, *args, out.data_ptr(),
                plan.n_heads, Hkv, D, S, scale, _ptr(workspace), ws)
    return out


def tree_masks(parents: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, max_nodes: int) -> tuple:
    """Trees of drafted tokens -> (mask int32 [N, words], depth int32 [N]) (lsk_tree_masks): the bits of each node's
    ancestors and its own, and its depth.  parents [N], starts and lens [nb] int32 on the device; max_nodes >= every
    len."""
    dev = _one_device(parents, starts, lens)
    n, nb = parents.numel(), starts.numel()
    for name, t, k in (("parents", parents, n), ("starts", starts, nb), ("lens", lens, nb)):
        _want("tree_masks", name, t, torch.int32, (k,))
    words = max(1, (max_nodes + 31) // 32)
    mask, depth = parents.new_zeros((n, words)), parents.new_zeros((n,))
    if n and nb:
        _launch(dev, "lsk_tree_masks", _ptr(parents), _ptr(starts), _ptr(lens), nb, n, max_nodes, _ptr(mask), words,
                _ptr(depth))
    return mask, depth


def tree_accept(Yv: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, starts: torch.Tensor,
                lens: torch.Tensor, max_nodes: int) -> tuple:
    """Greedy acceptance of verified trees (lsk_tree_accept) -> (accepted int64 [nb], path int32 [nb, max_nodes],
    tokens int64 [nb, max_nodes]): the accepted nodes and the tokens to commit, -1 past the end.  Yv (the verifier's
    greedy token of every node) and tokens int64 [N], parents int32 [N], starts and lens int32 [nb]."""
    dev = _one_device(Yv, tokens, parents, starts, lens)
    n, nb = parents.numel(), starts.numel()
    for name, t, dt, k in (("Yv", Yv, torch.int64, n), ("tokens", tokens, torch.int64, n),
                           ("parents", parents, torch.int32, n), ("starts", starts, torch.int32, nb),
                           ("lens", lens, torch.int32, nb)):
        _want("tree_accept", name, t, dt, (k,))
    if max_nodes < 1:
        raise LskError(f"tree_accept: max_nodes {max_nodes}")
    acc, path, out = Yv.new_empty(nb), parents.new_empty(nb, max_nodes), Yv.new_empty(nb, max_nodes)
    if nb and n == 0:
        acc.fill_(-1), path.fill_(-1), out.fill_(-1)
    elif nb:
        _launch(dev, "lsk_tree_accept", Yv.data_ptr(), tokens.data_ptr(), parents.data_ptr(), starts.data_ptr(),
                lens.data_ptr(), nb, n, max_nodes, acc.data_ptr(), path.data_ptr(), out.data_ptr())
    return acc, path, out


def _compact(what, code, k, v, ks, vs, layers, dims, rows_i32, pos0_i32, accepted, path) -> None:
    dev = _one_device(k, v, ks, vs, rows_i32, pos0_i32, accepted, path)
    nb, (B, Hkv, S, D) = rows_i32.numel(), dims
    _want(what, "rows", rows_i32, torch.int32, (nb,))
    _want(what, "pos0", pos0_i32, torch.int32, (nb,))
    _want(what, "accepted", accepted, torch.int64, (nb,))
    most = path.shape[1] if path.dim() == 2 else 0
    if most < 1:
        raise LskError(f"{what}: path must be [{nb}, max_nodes]")
    _want(what, "path", path, torch.int32, (nb, most))
    if nb and layers:
        _launch(dev, "lsk_kv_compact", code, k.data_ptr(), v.data_ptr(), _ptr(ks), _ptr(vs), layers,
                rows_i32.data_ptr(), pos0_i32.data_ptr(), accepted.data_ptr(), path.data_ptr(), nb, most, Hkv, D, B, S)


def kv_compact(k: torch.Tensor, v: torch.Tensor, rows_i32, pos0_i32, accepted, path) -> None:
    """The accepted paths' K / V move to consecutive slots in every layer (lsk_kv_compact): slot pos0 + j of a cache row
    takes slot pos0 + path[j], j = 1 .. accepted.  k, v: the layers' storage (KVCache.kf_all or fp32 rows, and vb_all;
    or a run of their layers); path and accepted: tree_accept's; rows, pos0 int32 [nb], the rows different."""
    shape, code = tuple(k.shape), dtype_code(k.dtype)
    if len(shape) != (7 if code == DTYPE_BF16 else 5) or not k.is_contiguous():
        raise LskError("kv_compact: the K storage of several layers is needed, contiguous: fragment-major bf16 or "
                       "row-major fp32")
    L, B, Hkv = shape[:3]
    S, D = (shape[3] * 32, shape[4] * 16) if code == DTYPE_BF16 else shape[3:]
    _want("kv_compact", "V storage", v, k.dtype, (L, B, Hkv, S // 32, D, 32))
    _compact("kv_compact", code, k, v, None, None, L, (B, Hkv, S, D), rows_i32, pos0_i32, accepted, path)


def kv8_compact(cache: KV8, rows_i32, pos0_i32, accepted, path) -> None:
    """kv_compact for the layers of an 8-bit cache (tensors with a leading layer axis)."""
    dims = cache.check("kv8_compact", layers=True)
    _compact("kv8_compact", DTYPE_KV8, *cache, cache.k.shape[0], dims, rows_i32, pos0_i32, accepted, path)


# ----------------------------------------------------------------------------- layer-range runner

def _ptr_array(ptrs):
    arr = (ctypes.c_void_p * len(ptrs))()
    for i, p in enumerate(ptrs):
        arr[i] = p
    return arr


class NativeModel:
    """Handle of the native layer-range runner for one (weights, KV cache, RoPE table) set."""

    def __init__(self, dtype, n_layers, dim, n_heads, n_kv_heads, head_dim, ffn, vocab, eps, layers, kcache, vcache,
                 cos_tab, sin_tab):
        if dtype == torch.bfloat16:
            # the bf16 runner's fused qkv + RoPE launch reads wqkv in the RoPE-paired packing
            for i, lw in enumerate(layers):
                if not (isinstance(lw.wqkv, PackedWeight) and lw.wqkv.qkv_heads == (n_heads, n_kv_heads, head_dim)):
                    raise LskError(f"layer {i}: bf16 wqkv must be a PackedWeight packed with qkv_heads="
                                   f"{(n_heads, n_kv_heads, head_dim)} (got "
                                   f"{getattr(lw.wqkv, 'qkv_heads', type(lw.wqkv).__name__)})")
        lib = load()
        _dev(cos_tab, sin_tab)
        _check_kcache(dtype, kcache[0])
        B, Hkv, S, D = k_dims(kcache[0])
        assert vcache[0].shape == (B, Hkv, S // 32, D, 32) and vcache[0].is_contiguous(), \
            "V cache must be the blocked-transposed [B, Hkv, S/32, D, 32] storage"
        self._keep = (layers, kcache, vcache, cos_tab, sin_tab)
        h = lib.lsk_model_create(
            dtype_code(dtype), n_layers, dim, n_heads, n_kv_heads, head_dim, ffn, vocab, float(eps),
            _ptr_array([lw.wqkv.data_ptr() for lw in layers]), _ptr_array([lw.wo.data_ptr() for lw in layers]),
            _ptr_array([lw.w13.data_ptr() for lw in layers]), _ptr_array([lw.w2.data_ptr() for lw in layers]),
            _ptr_array([lw.attn_norm.data_ptr() for lw in layers]),
            _ptr_array([lw.ffn_norm.data_ptr() for lw in layers]),
            _ptr_array([t.data_ptr() for t in kcache]), _ptr_array([t.data_ptr() for t in vcache]),
            B, S, cos_tab.data_ptr(), sin_tab.data_ptr(), cos_tab.shape[0])
        if h <= 0:
            _check(int(h), "lsk_model_create")
        self.handle = h
        self.n_layers = n_layers

    def workspace_bytes(self, n_tokens: int, n_parts: int) -> int:
        return int(load().lsk_segment_workspace_bytes(self.handle, n_tokens, n_parts))

    def forward_layers(self, x_in, x_out, n_tokens, start, end, meta_dev, nb, n_works, n_groups, n_parts, n_rounds,
                       n_slots, rows_cap, workspace, capture_ptrs=None, attn_bytes=0.0, attn_flops=0.0):
        _dev(x_in, x_out, meta_dev, workspace)
        cap = _ptr_array(capture_ptrs) if capture_ptrs is not None else None
        ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
        _check(load().lsk_forward_layers(self.handle, _ptr(x_in), _ptr(x_out), n_tokens, start, end, _ptr(meta_dev),
                                         nb, n_works, n_groups, n_parts, n_rounds, n_slots, rows_cap, _ptr(workspace),
                                         ws_bytes,
                                         cap,
                                         float(attn_bytes), float(attn_flops), _stream()),
               "lsk_forward_layers")

    def __del__(self):
        try:
            if getattr(self, "handle", 0) > 0 and _lib is not None:
                _lib.lsk_model_destroy(self.handle)
        except Exception:
            pass


# ----------------------------------------------------------------------------- profiling

class Profiler:
    """Per-class HIP-event timing of liblsk launches (algorithmic bytes / flops per launch)."""

    enabled = False

    @classmethod
    def enable(cls, on: bool = True) -> None:
        load().lsk_prof_enable(1 if on else 0)
        cls.enabled = on

    @staticmethod
    def start(cls_idx: int, nbytes: float, flops: float) -> None:
        if Profiler.enabled:
            load().lsk_prof_start(cls_idx, float(nbytes), float(flops), _stream())

    @staticmethod
    def stop() -> None:
        if Profiler.enabled:
            load().lsk_prof_stop(_stream())

    @staticmethod
    def collect() -> dict:
        n = len(PROF_CLASSES)
        ms, by, fl, ct = (np.zeros(n), np.zeros(n), np.zeros(n), np.zeros(n, dtype=np.int64))
        _check(load().lsk_prof_collect(n, ms.ctypes.data, by.ctypes.data, fl.ctypes.data, ct.ctypes.data),
               "lsk_prof_collect")
        return {PROF_CLASSES[i]: {"ms": float(ms[i]), "bytes": float(by[i]), "flops": float(fl[i]),
                                  "launches": int(ct[i])} for i in range(n) if ct[i]}


def gemm_plan(N: int, K: int) -> tuple:
    ns, ks = ctypes.c_int(0), ctypes.c_int(0)
    _check(load().lsk_gemm_plan(N, K, ctypes.byref(ns), ctypes.byref(ks)), "lsk_gemm_plan")
    return ns.value, ks.value


def gemm_wide_config(epilogue: int, M: int, N: int, K: int, ks: int = 1, af: bool = True) -> tuple:
    """(ns, blocks, groups per block, groups per wave) the wide-M tier picks; ns == 0: the tier does not apply."""
    cfg = (ctypes.c_int * 4)()
    _check(load().lsk_gemm_wide_config(epilogue, M, N, K, ks, int(af), cfg), "lsk_gemm_wide_config")
    return tuple(cfg)


def gemm_deep_config(epilogue: int, M: int, N: int, K: int, ks: int = 1, ldc: int | None = None) -> tuple:
    """(groups, token blocks, split) of a fragment-major launch in the many-token tier; groups 0: another tier.
    ldc: row stride of the output (None: contiguous)."""
    cfg = (ctypes.c_int * 3)()
    _check(load().lsk_gemm_deep_config(epilogue, M, N, K, ks, N if ldc is None else ldc, cfg), "lsk_gemm_deep_config")
    return tuple(cfg)


def frag_rows(m: int) -> int:
    """Rows a fragment-major activation buffer of m tokens holds (whole 16-token groups)."""
    return (m + 15) // 16 * 16


def gemm_partial_frag(a_frag: torch.Tensor, m: int, w: torch.Tensor, ks: int,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """gemm_partial with A fragment-major (lsk_gemm_partial_frag): a_frag holds frag_rows(m) x K elements in
    lsk_pack_weight's layout; fp32 K-slice partials [ks, m, N]."""
    _dev(a_frag, w, out)
    _check_weight(a_frag, w)
    N, K = w.shape
    if a_frag.dtype != torch.bfloat16 or a_frag.numel() < frag_rows(m) * K or not a_frag.is_contiguous():
        raise LskError("gemm_partial_frag: a contiguous bf16 buffer of frag_rows(m) x K elements is needed")
    if out is None:
        out = torch.empty(ks, m, N, dtype=torch.float32, device=a_frag.device)
    _check(load().lsk_gemm_partial_frag(_ptr(a_frag), _ptr(w), _ptr(out), m, N, K, ks, _stream()),
           "lsk_gemm_partial_frag")
    return out


def gemm_residual_frag(a_frag: torch.Tensor, m: int, w: torch.Tensor, ks: int, residual: torch.Tensor,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """residual + the product of a many-token segment (lsk_gemm_residual_frag): a_frag as gemm_partial_frag's, residual
    and out [m, N] bf16 rows (out may be residual); the K slices are summed in slice order in the launch."""
    _dev(a_frag, w, residual, out)
    _check_weight(a_frag, w)
    N, K = w.shape
    if a_frag.dtype != torch.bfloat16 or a_frag.numel() < frag_rows(m) * K or not a_frag.is_contiguous():
        raise LskError("gemm_residual_frag: a contiguous bf16 buffer of frag_rows(m) x K elements is needed")
    if out is None:
        out = torch.empty(m, N, dtype=torch.bfloat16, device=a_frag.device)
    for t in (residual, out):
        if t.shape != (m, N) or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise LskError("gemm_residual_frag: residual and out must be contiguous [m, N] bf16 tensors")
    _check(load().lsk_gemm_residual_frag(_ptr(a_frag), _ptr(w), _ptr(residual), _ptr(out), m, N, K, ks, _stream()),
           "lsk_gemm_residual_frag")
    return out


def gemm_silu_frag(a_frag: torch.Tensor, m: int, w: torch.Tensor, h: torch.Tensor, h_frag: bool) -> torch.Tensor:
    """w13 + silu-mul with A fragment-major (lsk_gemm_silu_frag); h row-major [m, ffn] or, with h_frag,
    fragment-major (frag_rows(m) x ffn elements)."""
    _dev(a_frag, w, h)
    _check_weight(a_frag, w)
    ffn, K = w.shape[0] // 2, w.shape[1]
    if a_frag.dtype != torch.bfloat16 or a_frag.numel() < frag_rows(m) * K or not a_frag.is_contiguous():
        raise LskError("gemm_silu_frag: a contiguous bf16 buffer of frag_rows(m) x K elements is needed")
    if h.numel() < (frag_rows(m) if h_frag else m) * ffn or not h.is_contiguous():
        raise LskError("gemm_silu_frag: output too small")
    _check(load().lsk_gemm_silu_frag(_ptr(a_frag), _ptr(w), _ptr(h), 1 if h_frag else 0, m, ffn, K, _stream()),
           "lsk_gemm_silu_frag")
    return h


def gemm_partial(a: torch.Tensor, w: torch.Tensor, ks: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 K-slice partials [ks, M, N] of a @ w.T (bf16, w packed)."""
    _dev(a, w, out)
    _check_weight(a, w)
    M, K = a.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(ks, M, N, dtype=torch.float32, device=a.device)
    _check(load().lsk_gemm_partial(_ptr(a), a.stride(0), _ptr(w), w.stride(0), _ptr(out), M, N, K, ks, _stream()),
           "lsk_gemm_partial")
    return out


def head_argmax(a: torch.Tensor, w: torch.Tensor, out: torch.Tensor, dst_idx: torch.Tensor | None = None,
                logits: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    _dev(a, w, out, dst_idx, logits, workspace)
    _check_weight(a, w)
    M, K = a.shape
    N = w.shape[0]
    need = int(load().lsk_head_workspace_bytes(M, N))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=a.device)
    _check(load().lsk_head_argmax(dtype_code(a.dtype), _ptr(a), a.stride(0), _ptr(w), w.stride(0), M, N, K,
                                  _ptr(logits), logits.stride(0) if logits is not None else 0, _ptr(out),
                                  _ptr(dst_idx), _ptr(workspace), workspace.numel() * workspace.element_size(),
                                  _stream()), "lsk_head_argmax")
    return out


def head_norm_argmax(h: torch.Tensor, norm_w: torch.Tensor, eps: float, w, out: torch.Tensor,
                     dst_idx: torch.Tensor | None = None, logits: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """argmax(lm_head(rmsnorm(h))) per row in one native call (bf16), bitwise equal to rmsnorm + head_argmax."""
    _dev(h, norm_w, out, dst_idx, logits, workspace)
    _check_weight(h, w)
    M, K = h.shape
    N = w.shape[0]
    need = int(load().lsk_head_norm_workspace_bytes(M, N, K))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=h.device)
    _check(load().lsk_head_norm_argmax(dtype_code(h.dtype), _ptr(h), h.stride(0), _ptr(norm_w), float(eps), _ptr(w),
                                       w.stride(0), M, N, K, _ptr(logits), logits.stride(0) if logits is not None else 0,
                                       _ptr(out), _ptr(dst_idx), _ptr(workspace),
                                       workspace.numel() * workspace.element_size(), _stream()),
           "lsk_head_norm_argmax")
    return out


def add_rmsnorm(x: torch.Tensor, partials: torch.Tensor | None, w: torch.Tensor | None, eps: float,
                x_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> None:
    _dev(x, partials, w, x_out, out)
    n, dim = x.shape
    ks = partials.shape[0] if partials is not None else 0
    _check(load().lsk_add_rmsnorm(dtype_code(x.dtype), _ptr(x), x.stride(0), _ptr(partials), ks, _ptr(w), float(eps),
                                  _ptr(x_out), x_out.stride(0) if x_out is not None else 0, _ptr(out),
                                  out.stride(0) if out is not None else 0, n, dim, _stream()), "lsk_add_rmsnorm")


def gemm_qkv_rope(a_frag: torch.Tensor, w: "PackedWeight", M: int, q_out, kcache, vcache, cos_tab, sin_tab,
                  rows_i32, pos_i32) -> None:
    """Fused qkv projection + RoPE + KV append (lsk_gemm_qkv_rope): a_frag holds the normalised rows fragment-major
    (frag_rows(M) * K elements), w a PackedWeight packed with qkv_heads; writes q_out [M, Hq, D] and the caches."""
    _dev(a_frag, q_out, kcache, vcache, cos_tab, sin_tab, rows_i32, pos_i32)
    if not isinstance(w, PackedWeight) or w.qkv_heads is None:
        raise LskError("gemm_qkv_rope reads a PackedWeight packed with qkv_heads (lsk_pack_weight_qkv)")
    _check_kcache(q_out.dtype, kcache)
    hq, hkv, d = w.qkv_heads
    B, _, S, _ = k_dims(kcache)
    _check(load().lsk_gemm_qkv_rope(_ptr(a_frag), _ptr(w), M, hq, hkv, d, w.shape[1], _ptr(q_out), _ptr(kcache),
                                    _ptr(vcache), _ptr(cos_tab), _ptr(sin_tab), cos_tab.shape[0], _ptr(rows_i32),
                                    _ptr(pos_i32), B, S, _stream()), "lsk_gemm_qkv_rope")


def rope_append_partial(partials, q_out, kcache, vcache, cos_tab, sin_tab, rows_i32, pos_i32, n_heads, n_kv_heads,
                        head_dim):
    _dev(partials, q_out, kcache, vcache, cos_tab, sin_tab, rows_i32, pos_i32)
    _check_kcache(q_out.dtype, kcache)
    ks, N, _ = partials.shape
    B, Hkv, S, D = k_dims(kcache)
    _check(load().lsk_rope_append_partial(dtype_code(q_out.dtype), _ptr(partials), ks, _ptr(q_out), _ptr(kcache),
                                          _ptr(vcache), _ptr(cos_tab), _ptr(sin_tab), cos_tab.shape[0],
                                          _ptr(rows_i32), _ptr(pos_i32), N, n_heads, n_kv_heads, head_dim, B, S,
                                          _stream()), "lsk_rope_append_partial")
