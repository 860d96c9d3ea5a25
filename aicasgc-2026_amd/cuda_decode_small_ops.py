#!/usr/bin/env python3
"""Small fused decode ops backed by gfx950 kernels.

Same names, arguments, checks (RuntimeError on a bad dtype/shape) and return
conventions as the reference's cuda_decode_small_ops.py.

The ``*_fp8`` entry points have no counterpart there.  They are the 8-bit serving
path's: e4m3 values (``torch.float8_e4m3fn``) with a power-of-two scale per block
(``torch.float8_e8m0fnu``).  A block's scale is the least power of two with
amax <= 448 * scale over its finite values; NaN and infinities are stored as NaN.
Activations have a scale per row and 128 columns, weights per 128 x 128 block (the
product is ``cuda_decode_gemv.block_matmul_fp8``), the KV cache per 64 tokens and
head (its attention is ``cuda_decode_attention.attn_fp8_kv_cache``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from qwen3vl_hip import _lib


def _load_ext():
    return _lib.lib()


def _all_cuda_half(*ts) -> bool:
    return all(t.device.type == "cuda" and t.dtype == torch.float16 for t in ts)


def fused_qk_rms_norm_rope(q, k, q_weight, k_weight, eps: float, cos, sin):
    """Per-head RMSNorm + rotate-half RoPE of q [B,S,Hq,128] and k [B,S,Hkv,128]
    with cos/sin [B,S,128] (reference cuda_decode_small_ops.py:70-133)."""
    if not _all_cuda_half(q, k, q_weight, k_weight, cos, sin):
        raise RuntimeError("fused_qk_rms_norm_rope: every tensor must be fp16 on the GPU")
    if q.ndim != 4 or k.ndim != 4:
        raise RuntimeError("fused_qk_rms_norm_rope: q and k must be 4-D [batch, seq, heads, 128]")
    if q.shape[:2] != k.shape[:2]:
        raise RuntimeError("fused_qk_rms_norm_rope: q and k disagree on batch or sequence length")
    if q.shape[-1] != 128 or k.shape[-1] != 128:
        raise RuntimeError("fused_qk_rms_norm_rope: head size must be 128")
    if q.shape[2] != k.shape[2] * 2:
        raise RuntimeError("fused_qk_rms_norm_rope: need twice as many q heads as k heads")
    if q_weight.numel() != 128 or k_weight.numel() != 128:
        raise RuntimeError("fused_qk_rms_norm_rope: q/k norm weights must hold 128 values")
    q_in, k_in = q.contiguous(), k.contiguous()
    cos_in, sin_in = cos.contiguous(), sin.contiguous()
    if cos_in.shape != q_in.shape[:2] + (128,) or sin_in.shape != q_in.shape[:2] + (128,):
        raise RuntimeError("fused_qk_rms_norm_rope: cos/sin must be [batch, seq, 128]")
    m = q_in.shape[0] * q_in.shape[1]
    q_out, k_out = torch.empty_like(q_in), torch.empty_like(k_in)
    qw, kw = q_weight.contiguous(), k_weight.contiguous()   # held until the launch is enqueued
    _lib.check(_load_ext().qd_qk_norm_rope_f16(
        _lib.ptr(q_in), _lib.ptr(k_in), _lib.ptr(qw), _lib.ptr(kw),
        _lib.ptr(cos_in), _lib.ptr(sin_in), _lib.ptr(q_out), _lib.ptr(k_out), m, q_in.shape[2], k_in.shape[2],
        float(eps), _lib.stream(q.device)), "fused_qk_rms_norm_rope")
    return q_out, k_out


def fused_q_rope_kv_cache_update(q, k, v, q_weight, k_weight, eps: float, cos, sin, k_cache, v_cache,
                                 cache_position):
    """q/k per-head RMSNorm + RoPE; K_rot and V written at cache_position;
    returns the rotated q [1,1,Hq,128] (reference cuda_decode_small_ops.py:136-225)."""
    if not (_all_cuda_half(q, k, v, q_weight, k_weight, cos, sin, k_cache, v_cache)
            and cache_position.device.type == "cuda" and cache_position.dtype == torch.long):
        raise RuntimeError("fused_q_rope_kv_cache_update: tensors must be fp16 on the GPU, cache_position int64 on the GPU")
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise RuntimeError("fused_q_rope_kv_cache_update: q, k and v must be 4-D [batch, seq, heads, 128]")
    if q.shape[:2] != k.shape[:2] or k.shape != v.shape:
        raise RuntimeError("fused_q_rope_kv_cache_update: k and v shapes differ, or q disagrees with them")
    if q.shape[0] != 1 or q.shape[1] != 1 or k.shape[0] != 1 or k.shape[1] != 1:
        raise RuntimeError("fused_q_rope_kv_cache_update: one token per call (batch 1, seq 1)")
    if q.shape[-1] != 128 or k.shape[-1] != 128 or v.shape[-1] != 128:
        raise RuntimeError("fused_q_rope_kv_cache_update: head size must be 128")
    if q.shape[2] != k.shape[2] * 2:
        raise RuntimeError("fused_q_rope_kv_cache_update: need twice as many q heads as kv heads")
    if q_weight.numel() != 128 or k_weight.numel() != 128:
        raise RuntimeError("fused_q_rope_kv_cache_update: q/k norm weights must hold 128 values")
    if cos.shape != q.shape[:2] + (128,) or sin.shape != q.shape[:2] + (128,):
        raise RuntimeError("fused_q_rope_kv_cache_update: cos/sin must be [batch, seq, 128]")
    if k_cache.ndim != 4 or v_cache.ndim != 4:
        raise RuntimeError("fused_q_rope_kv_cache_update: caches must be 4-D [batch, kv heads, rows, 128]")
    if k_cache.shape[0] != 1 or v_cache.shape[0] != 1:
        raise RuntimeError("fused_q_rope_kv_cache_update: caches must have batch 1")
    if k_cache.shape[1] != k.shape[2] or v_cache.shape[1] != v.shape[2]:
        raise RuntimeError("fused_q_rope_kv_cache_update: cache and k have different kv head counts")
    if k_cache.shape[-1] != 128 or v_cache.shape[-1] != 128:
        raise RuntimeError("fused_q_rope_kv_cache_update: cache rows are not 128 wide")
    if cache_position.ndim != 1 or cache_position.numel() != 1:
        raise RuntimeError("fused_q_rope_kv_cache_update: cache_position must hold exactly one position")
    if (k_cache.stride(-1) != 1 or v_cache.stride(-1) != 1 or k_cache.stride(1) != v_cache.stride(1)
            or k_cache.stride(2) != v_cache.stride(2) or k_cache.shape != v_cache.shape):
        raise RuntimeError("fused_q_rope_kv_cache_update: k_cache and v_cache need the same strides and contiguous rows")
    # contiguous copies are bound to locals so they outlive the asynchronous launch's enqueue
    q_in, k_in, v_in = q.contiguous(), k.contiguous(), v.contiguous()
    qw, kw = q_weight.contiguous(), k_weight.contiguous()
    cos_in, sin_in, cp = cos.contiguous(), sin.contiguous(), cache_position.contiguous()
    q_out = torch.empty((1, 1, q.shape[2], 128), dtype=q.dtype, device=q.device)
    _lib.check(_load_ext().qd_q_rope_kv_update(
        _lib.ptr(q_in), _lib.ptr(k_in), _lib.ptr(v_in), _lib.QD_F16, 128, 128, 128,
        _lib.ptr(qw), _lib.ptr(kw), float(eps), _lib.ptr(cos_in), _lib.ptr(sin_in), None, None, 24, 20, 20,
        _lib.ptr(q_out), _lib.QD_F16, _lib.ptr(k_cache), _lib.ptr(v_cache), k_cache.stride(1), k_cache.stride(2),
        k_cache.shape[2], _lib.ptr(cp), q.shape[2], k.shape[2], _lib.stream(q.device)),
        "fused_q_rope_kv_cache_update")
    return q_out


def fused_silu_mul(gate, up):
    """silu(gate) * up (reference cuda_decode_small_ops.py:228-247)."""
    if not _all_cuda_half(gate, up):
        raise RuntimeError("fused_silu_mul: gate and up must be fp16 on the GPU")
    if gate.shape != up.shape:
        raise RuntimeError("fused_silu_mul: gate and up shapes differ")
    g, u = gate.contiguous(), up.contiguous()
    out = torch.empty_like(g)
    _lib.check(_load_ext().qd_silu_mul_f16(_lib.ptr(g), _lib.ptr(u), _lib.ptr(out), g.numel(),
                                           _lib.stream(g.device)), "fused_silu_mul")
    return out


def fused_add_rms_norm(residual, x, weight, eps: float):
    """(residual + x, rmsnorm(residual + x) * weight) (reference cuda_decode_small_ops.py:250-287)."""
    if not _all_cuda_half(residual, x, weight):
        raise RuntimeError("fused_add_rms_norm: every tensor must be fp16 on the GPU")
    if residual.shape != x.shape:
        raise RuntimeError("fused_add_rms_norm: residual and x shapes differ")
    if residual.shape[-1] != weight.numel():
        raise RuntimeError("fused_add_rms_norm: weight length differs from the last dimension")
    r, xi = residual.contiguous(), x.contiguous()
    cols = r.shape[-1]
    rows = r.numel() // cols
    out_sum, out_norm = torch.empty_like(r), torch.empty_like(r)
    wc = weight.contiguous()
    _lib.check(_load_ext().qd_add_rmsnorm_f16(_lib.ptr(r), _lib.ptr(xi), _lib.ptr(wc),
                                              _lib.ptr(out_sum), _lib.ptr(out_norm), rows, cols, float(eps),
                                              _lib.stream(r.device)), "fused_add_rms_norm")
    return out_sum, out_norm


def rms_norm(x, weight, eps: float):
    """rmsnorm(x) * weight over the last dim (reference cuda_decode_small_ops.py:290-317)."""
    if not _all_cuda_half(x, weight):
        raise RuntimeError("rms_norm: x and weight must be fp16 on the GPU")
    if x.shape[-1] != weight.numel():
        raise RuntimeError("rms_norm: weight length differs from the last dimension")
    xi = x.contiguous()
    cols = xi.shape[-1]
    out = torch.empty_like(xi)
    wc = weight.contiguous()
    _lib.check(_load_ext().qd_rmsnorm_f16(_lib.ptr(xi), _lib.ptr(wc), _lib.ptr(out),
                                          xi.numel() // cols, cols, float(eps), _lib.stream(xi.device)), "rms_norm")
    return out


def add(a, b):
    """a + b (reference cuda_decode_small_ops.py:320-339)."""
    if not _all_cuda_half(a, b):
        raise RuntimeError("add: both operands must be fp16 on the GPU")
    if a.shape != b.shape:
        raise RuntimeError("add: operand shapes differ")
    ai, bi = a.contiguous(), b.contiguous()
    out = torch.empty_like(ai)
    _lib.check(_load_ext().qd_add_f16(_lib.ptr(ai), _lib.ptr(bi), _lib.ptr(out), ai.numel(),
                                      _lib.stream(ai.device)), "add")
    return out


# ---------------------------------------------------------------- 8-bit operators

_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_EMPTY_LIKE = torch.empty_like
FP8_COLS = 128       # columns (and, of a weight, rows) per scale
KV_FP8_BLOCK = 64    # cache rows per scale


def _half_gpu(name: str, *ts) -> int:
    """The GPU that holds the fp16 tensors ``ts``, all of them."""
    dev = ts[0].get_device()
    for t in ts:
        if t.dtype is not torch.float16 or t.get_device() != dev or dev < 0:
            raise RuntimeError(f"{name}: every tensor must be fp16 on the GPU, on one device")
    return dev


def _as_rows(t: torch.Tensor):
    """``t`` as rows of its last dimension: (tensor to keep, row stride).  A view
    whose rows follow one another at one stride is used in place."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.ndim == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    if t.ndim > 2 and t.stride(-1) == 1:
        step, rows = t.shape[-1], 1
        for size, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
            if size == 1:
                continue
            if rows == 1:
                step = stride
            elif stride != step * rows:
                return t.contiguous(), t.shape[-1]
            rows *= size
        return t, step
    return t.contiguous(), t.shape[-1]


def _quantized_like(name: str, x: torch.Tensor):
    """Empty e4m3 values of x's shape, their scales, and (rows, cols)."""
    shape = x.shape
    cols = shape[-1] if shape else 0
    if cols < 1:
        raise RuntimeError(f"{name}: rows must have at least one column")
    blocks, rows = (cols + FP8_COLS - 1) // FP8_COLS, x.numel() // cols
    # (of the ways to get an empty tensor the two quickest; a decode call's time is its host side's)
    q = _EMPTY_LIKE(x, dtype=_F8) if x.is_contiguous() else x.new_empty(shape, dtype=_F8)
    if len(shape) == 2:
        scale = torch.empty_strided((rows, blocks), (blocks, 1), dtype=_E8, device=x.device)
    else:
        scale = x.new_empty((*shape[:-1], blocks), dtype=_E8)
    return q, scale, rows, cols


def quantize_fp8(x, block_rows: int = 1):
    """e4m3 values and scales of x [..., cols]: a scale per row and 128 columns, or,
    with ``block_rows=128``, per 128 x 128 block of a matrix [rows, cols] (a weight)."""
    dev = _half_gpu("quantize_fp8", x)
    if block_rows not in (1, FP8_COLS):
        raise RuntimeError("quantize_fp8: block_rows must be 1 or 128")
    if block_rows != 1 and x.ndim != 2:
        raise RuntimeError("quantize_fp8: blocks of 128 rows need a matrix [rows, cols]")
    q, scale, rows, cols = _quantized_like("quantize_fp8", x)
    if block_rows != 1:
        scale = x.new_empty(((rows + FP8_COLS - 1) // FP8_COLS, scale.shape[1]), dtype=_E8)
    xi, ld = _as_rows(x)
    _lib.call_on(dev, _lib.entry("qd_quantize_fp8"), xi.data_ptr(), ld, q.data_ptr(), scale.data_ptr(), rows, cols,
                 block_rows)
    return q, scale


def fused_silu_mul_fp8(gate, up):
    """silu(gate) * up in 8 bits: (values, scales).  gate and up [..., cols] may be the
    two halves of one product's output (rows at any stride)."""
    dev = _half_gpu("fused_silu_mul_fp8", gate, up)
    if gate.shape != up.shape:
        raise RuntimeError("fused_silu_mul_fp8: gate and up shapes differ")
    q, scale, rows, cols = _quantized_like("fused_silu_mul_fp8", gate)
    g, ldg = _as_rows(gate)
    u, ldu = _as_rows(up)
    _lib.call_on(dev, _lib.entry("qd_silu_mul_fp8"), g.data_ptr(), ldg, u.data_ptr(), ldu, q.data_ptr(), scale.data_ptr(),
                 rows, cols)
    return q, scale


def _norm_fp8(name, dev, residual, x, weight, eps):
    q, scale, rows, cols = _quantized_like(name, x)
    if weight.numel() != cols:
        raise RuntimeError(f"{name}: weight length differs from the last dimension")
    xi, ld = _as_rows(x)
    wc = weight.contiguous()
    ri, ldr, total, r_ptr, t_ptr = None, 0, None, None, None
    if residual is not None:
        ri, ldr = _as_rows(residual)
        total = _EMPTY_LIKE(x, memory_format=torch.contiguous_format)
        r_ptr, t_ptr = ri.data_ptr(), total.data_ptr()
    _lib.call_on(dev, _lib.entry("qd_add_rmsnorm_fp8"), r_ptr, ldr, xi.data_ptr(), ld, wc.data_ptr(), t_ptr, q.data_ptr(),
                 scale.data_ptr(), rows, cols, eps)
    return total, q, scale


def fused_add_rms_norm_fp8(residual, x, weight, eps: float):
    """(residual + x in fp16, rmsnorm(residual + x) * weight in 8 bits: values, scales).
    The norm is taken of the unrounded sum, as ``fused_add_rms_norm`` does."""
    dev = _half_gpu("fused_add_rms_norm_fp8", residual, x, weight)
    if residual.shape != x.shape:
        raise RuntimeError("fused_add_rms_norm_fp8: residual and x shapes differ")
    return _norm_fp8("fused_add_rms_norm_fp8", dev, residual, x, weight, eps)


def rms_norm_fp8(x, weight, eps: float):
    """rmsnorm(x) * weight over the last dim in 8 bits: (values, scales)."""
    dev = _half_gpu("rms_norm_fp8", x, weight)
    return _norm_fp8("rms_norm_fp8", dev, None, x, weight, eps)[1:]


class KVCacheFP8(NamedTuple):
    """The 8-bit KV cache of one layer: rows in blocks of 64 tokens, one scale per
    (sequence, kv head, block) for K and one for V.  V is transposed inside its
    block.  Views of some sequences or heads are caches too (one sequence expanded
    to several can be read, not written)."""

    k: torch.Tensor          # e4m3 [B, Hkv, T, 128], T a multiple of 64
    v: torch.Tensor          # e4m3 [B, Hkv, T / 64, 128, 64]
    k_scale: torch.Tensor    # e8m0 [B, Hkv, T / 64]
    v_scale: torch.Tensor    # e8m0 [B, Hkv, T / 64]


def new_kv_cache_fp8(batch: int, kv_heads: int, capacity: int, device="cuda") -> KVCacheFP8:
    """An empty cache of ``capacity`` rows (rounded up to a multiple of 64) per sequence."""
    if batch < 1 or kv_heads < 1 or capacity < 1:
        raise RuntimeError("new_kv_cache_fp8: batch, kv_heads and capacity must be positive")
    nb = (capacity + KV_FP8_BLOCK - 1) // KV_FP8_BLOCK

    def full(byte, dtype, *shape):
        return torch.full(shape, byte, dtype=torch.uint8, device=device).view(dtype)

    # values 0, scales the smallest that a cache has, 2^-32
    return KVCacheFP8(full(0, _F8, batch, kv_heads, nb * KV_FP8_BLOCK, 128),
                      full(0, _F8, batch, kv_heads, nb, 128, KV_FP8_BLOCK),
                      full(127 - 32, _E8, batch, kv_heads, nb), full(127 - 32, _E8, batch, kv_heads, nb))


def _kv_fp8_args(name: str, cache, dev: int):
    """(B, Hkv, T, the C entries' cache arguments) of a valid cache on GPU ``dev``."""
    k, v, ks, vs = cache
    if (k.dtype is not _F8 or v.dtype is not _F8 or ks.dtype is not _E8 or vs.dtype is not _E8 or k.ndim != 4
            or k.get_device() != dev or v.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev):
        raise RuntimeError(f"{name}: cache must be a KVCacheFP8 on the inputs' device")
    b, h, t, d = k.shape
    nb = t // KV_FP8_BLOCK
    shape = ks.shape
    if (d != 128 or t != nb * KV_FP8_BLOCK or shape != (b, h, nb) or vs.shape != shape
            or v.shape != (b, h, nb, 128, KV_FP8_BLOCK)):
        raise RuntimeError(f"{name}: cache shapes must be k [B, Hkv, T, 128], v [B, Hkv, T / 64, 128, 64] and scales "
                           "[B, Hkv, T / 64]")
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3, v4 = v.stride()
    s0, s1, s2 = ks.stride()
    if (k2 != 128 or k3 != 1 or v3 != KV_FP8_BLOCK or v4 != 1
            or (nb > 1 and (v2 != 128 * KV_FP8_BLOCK or s2 != 1)) or (b > 1 and k0 != v0) or (h > 1 and k1 != v1)
            or vs.stride() != (s0, s1, s2)):
        raise RuntimeError(f"{name}: a head of the cache must be contiguous, k and v (and their scales) at the same strides")
    return b, h, t, (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k0, k1, s0, s1, t)


def _positions(name: str, cache_position, b: int, dev: int) -> torch.Tensor:
    if cache_position.dtype is not torch.int64 or cache_position.get_device() != dev or cache_position.shape != (b,):
        raise RuntimeError(f"{name}: cache_position must be int64 [{b}] on the inputs' device")
    return cache_position if cache_position.is_contiguous() else cache_position.contiguous()


def _strided_heads(t: torch.Tensor, multiple: int):
    """t [.., .., .., 128] (any order of the first three) itself where its heads can be
    read in place, contiguous, at strides and an address of whole ``multiple``s, or a
    copy of it: (tensor to keep, address, the first three strides)."""
    s0, s1, s2, s3 = t.stride()
    ptr = t.data_ptr()
    if s3 == 1 and not (s0 | s1 | s2) % multiple and not ptr % (2 * multiple):
        return t, ptr, s0, s1, s2
    t = t.contiguous()
    if t.data_ptr() % (2 * multiple):
        t = t.clone()
    return t, t.data_ptr(), *t.stride()[:3]


def _aligned8(t: torch.Tensor):
    """t, or a copy of it, contiguous at an 8-byte aligned address: (tensor to keep, address)."""
    ptr = t.data_ptr()
    if t.is_contiguous() and not ptr % 8:
        return t, ptr
    t = t.contiguous() if not t.is_contiguous() else t.clone()
    return t, t.data_ptr()


def fused_q_rope_kv_cache_update_fp8(q, k, v, q_weight, k_weight, eps: float, cos, sin, cache: KVCacheFP8,
                                     cache_position):
    """q/k per-head RMSNorm + RoPE of S new tokens of each sequence, their K_rot and V
    written to the 8-bit cache from row ``cache_position[b]`` on; returns the
    rotated q [B, S, Hq, 128] in fp16.

    q [B, S, Hq, 128], k and v [B, S, Hkv, 128], cos and sin [B, S, 128], all fp16;
    cache_position int64 [B].  Rows outside [0, T) are not written.  The rows
    before cache_position stay (a block's earlier rows are rescaled, within e4m3,
    when the new ones need a larger scale); rows from cache_position on that are
    not written here are no longer the sequence's: a block's scale follows the
    rows up to the last one written."""
    name = "fused_q_rope_kv_cache_update_fp8"
    dev = _half_gpu(name, q, k, v, q_weight, k_weight, cos, sin)
    if q.ndim != 4 or k.ndim != 4:
        raise RuntimeError(f"{name}: q must be [B, S, Hq, 128], k and v [B, S, Hkv, 128]")
    bs, s, hq, d = q.shape
    b, h, t, where = _kv_fp8_args(name, cache, dev)
    if (b > 1 and 0 in where[4:7:2]) or (h > 1 and 0 in where[5:8:2]):
        raise RuntimeError(f"{name}: sequences (or heads) that share their rows or scales cannot be written")
    if d != 128 or k.shape != (bs, s, h, 128) or v.shape != (bs, s, h, 128) or bs != b:
        raise RuntimeError(f"{name}: q must be [B, S, Hq, 128], k and v [B, S, Hkv, 128], with the cache's B and Hkv")
    if hq % h or not h <= hq <= 64 * h:
        raise RuntimeError(f"{name}: q heads must be 1 to 64 times the kv heads")
    if q_weight.numel() != 128 or k_weight.numel() != 128:
        raise RuntimeError(f"{name}: q/k norm weights must hold 128 values")
    if cos.shape != (b, s, 128) or sin.shape != (b, s, 128):
        raise RuntimeError(f"{name}: cos/sin must be [B, S, 128]")
    cp = _positions(name, cache_position, b, dev)
    # (the copies, where there are any, live until the launch)
    qi, *q_at = _strided_heads(q, 4)
    ki, *k_at = _strided_heads(k, 4)
    vi, *v_at = _strided_heads(v, 4)
    qw, qw_at = _aligned8(q_weight)
    kw, kw_at = _aligned8(k_weight)
    cs, cs_at = _aligned8(cos)
    sn, sn_at = _aligned8(sin)
    out = _EMPTY_LIKE(q, memory_format=torch.contiguous_format)
    _lib.call_on(dev, _lib.entry("qd_q_rope_kv_update_fp8"), *q_at, *k_at, *v_at, qw_at, kw_at, eps, cs_at, sn_at,
                 out.data_ptr(), *where, cp.data_ptr(), b, s, hq, h)
    return out


def read_kv_cache_fp8(cache: KVCacheFP8, rows: int):
    """The first ``rows`` rows of every sequence in fp16: (k, v), each [B, Hkv, rows, 128]."""
    dev = cache[0].get_device()
    if dev < 0:
        raise RuntimeError("read_kv_cache_fp8: the cache must be on the GPU")
    b, h, t, where = _kv_fp8_args("read_kv_cache_fp8", cache, dev)
    if not 0 <= rows <= t:
        raise RuntimeError(f"read_kv_cache_fp8: rows must lie in [0, {t}]")
    k = torch.empty((b, h, rows, 128), dtype=torch.float16, device=cache[0].device)
    v = torch.empty_like(k)
    _lib.call_on(dev, _lib.entry("qd_kv_read_fp8"), *where, k.data_ptr(), v.data_ptr(), b, h, rows)
    return k, v
