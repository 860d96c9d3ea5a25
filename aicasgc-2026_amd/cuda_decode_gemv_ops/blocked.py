"""Block-scaled 8-bit product backed by the gfx950 MFMA kernels (no counterpart in the
reference, whose weights are fp16)."""

from __future__ import annotations

import torch

from qwen3vl_hip import _lib

_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_OUT = {torch.float16: _lib.QD_F16, torch.float32: _lib.QD_F32}


def block_matmul_fp8(x, x_scale, weight, weight_scale, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """y = x W^T of e4m3 operands with power-of-two scales, fp32 sums, y in fp16 or fp32.

    x [..., K] with x_scale [..., ceil(K / 128)] (``cuda_decode_small_ops.quantize_fp8``
    and the ``fused_*_fp8`` entry points), weight [N, K] with weight_scale
    [ceil(N / 128), ceil(K / 128)] (``quantize_fp8(w, block_rows=128)``); K a
    multiple of 16.  From one row (a decode token) to 2^20 (thousands: a prompt)."""
    name = "block_matmul_fp8"
    dev = x.get_device()
    if (x.dtype is not _F8 or weight.dtype is not _F8 or x_scale.dtype is not _E8 or weight_scale.dtype is not _E8
            or dev < 0 or weight.get_device() != dev or x_scale.get_device() != dev or weight_scale.get_device() != dev):
        raise RuntimeError(f"{name}: x and weight must be float8_e4m3fn and the scales float8_e8m0fnu, all on one GPU")
    lead = x.shape[:-1]
    if weight.ndim != 2 or x.ndim < 1:
        raise RuntimeError(f"{name}: weight must be [N, K] and x [..., K]")
    n, k = weight.shape
    kb = (k + 127) // 128
    if x.shape[-1] != k or x_scale.shape != (*lead, kb) or weight_scale.shape != ((n + 127) // 128, kb):
        raise RuntimeError(f"{name}: need x [..., {k}] with scales [..., {kb}] and weight scales [{(n + 127) // 128}, {kb}]")
    if n < 1 or k < 16 or k % 16 or x.numel() // k > 1 << 20:
        raise RuntimeError(f"{name}: K must be a positive multiple of 16, N positive and x of at most 2^20 rows")
    code = _OUT.get(out_dtype)
    if code is None:
        raise RuntimeError(f"{name}: out_dtype must be float16 or float32")
    xi, xs, w, ws = _aligned(x), x_scale.contiguous(), _aligned(weight), weight_scale.contiguous()
    y = torch.empty((*lead, n), dtype=out_dtype, device=x.device)
    _lib.call_on(dev, _lib.entry("qd_block_matmul_fp8"), xi.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(),
                 y.data_ptr(), code, x.numel() // k, n, k)
    return y


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy of it at a 16-byte aligned address."""
    if t.is_contiguous() and not t.data_ptr() % 16:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()
