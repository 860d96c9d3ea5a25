"""Refusals of the 8-bit operators, without a GPU: the Python entry points reject CPU
tensors and wrong shapes before any launch, the C entries reject bad arguments
with a status and a message (the addresses below are never dereferenced)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp8_oracle as O

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
A16 = 0x10000


@pytest.fixture()
def lib():
    from qwen3vl_hip import _lib

    return _lib.lib()


def _refused(lib, status, code, word):
    assert status == code, (status, lib.qd_last_error())
    assert word in lib.qd_last_error(), lib.qd_last_error()


def test_oracle_exponents():
    """Borders of the scale rule, against its definition."""
    for e in (-40, -9, 0, 5):
        assert O.exponent(448 * 2.0 ** e, -126) == e
        assert O.exponent(math.nextafter(448 * 2.0 ** e, math.inf), -126) == e + 1
        assert O.exponent(math.nextafter(224 * 2.0 ** e, math.inf), -126) == e
    assert O.exponent(0.0, -32) == -32 and O.exponent(1e-30, -32) == -32


def test_cpu_tensors_are_refused():
    import cuda_decode_attention as A
    import cuda_decode_gemv as G
    import cuda_decode_small_ops as S

    x = torch.randn(2, 256).half()
    w = torch.ones(256).half()
    cache = S.new_kv_cache_fp8(1, 2, 100, "cpu")
    assert cache.k.shape == (1, 2, 128, 128) and cache.v.shape == (1, 2, 2, 128, 64) and cache.k_scale.shape == (1, 2, 2)
    pos = torch.zeros(1, dtype=torch.int64)
    q, kv, cs = torch.zeros(1, 1, 4, 128).half(), torch.zeros(1, 1, 2, 128).half(), torch.zeros(1, 1, 128).half()
    n = torch.ones(128).half()
    for call in (lambda: S.quantize_fp8(x), lambda: S.quantize_fp8(x, block_rows=128), lambda: S.fused_silu_mul_fp8(x, x),
                 lambda: S.fused_add_rms_norm_fp8(x, x, w, 1e-6), lambda: S.rms_norm_fp8(x, w, 1e-6),
                 lambda: G.block_matmul_fp8(x.to(F8), torch.zeros(2, 2, dtype=torch.uint8).view(E8), x.to(F8),
                                            torch.zeros(1, 2, dtype=torch.uint8).view(E8)),
                 lambda: S.fused_q_rope_kv_cache_update_fp8(q, kv, kv, n, n, 1e-6, cs, cs, cache, pos),
                 lambda: S.read_kv_cache_fp8(cache, 3), lambda: A.attn_fp8_kv_cache(q.transpose(1, 2), cache, 0.1, pos)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    for bad in ((0, 1, 64), (1, 0, 64), (1, 1, 0)):
        with pytest.raises(RuntimeError):
            S.new_kv_cache_fp8(*bad, "cpu")


def test_cache_arguments_are_checked():
    import cuda_decode_small_ops as S

    cpu = -1   # get_device() of a CPU tensor
    c = S.new_kv_cache_fp8(2, 3, 128, "cpu")
    assert S._kv_fp8_args("t", c, cpu)[:3] == (2, 3, 128)
    assert S._kv_fp8_args("t", [t[1:, ::2] for t in c], cpu)[:3] == (1, 2, 128)
    bad = [c._replace(k=c.k.view(torch.uint8)), c._replace(k_scale=c.k_scale[:, :, :1]), c._replace(v=c.v[:, :2]),
           c._replace(k=c.k[:, :, :64]), c._replace(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)),
           c._replace(v=c.v.transpose(-1, -2).contiguous().transpose(-1, -2)), c._replace(k=c.k[..., :64])]
    for cache in bad:
        with pytest.raises(RuntimeError):
            S._kv_fp8_args("t", cache, cpu)
    for pos in (torch.zeros(2), torch.zeros(1, dtype=torch.int64), torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(RuntimeError):
            S._positions("t", pos, 2, cpu)


def test_rows_of_views():
    """Views whose rows lie at one stride are used in place, others are copied."""
    import cuda_decode_small_ops as S

    big = torch.arange(4 * 6 * 300).half().view(4, 6, 300)
    for view, own in ((big, True), (big[..., 8:264], True), (big[:, ::2, :256], True), (big[:, :3], False),
                      (big.transpose(0, 1), False), (big[0], True), (big[1, 2], True), (big[..., ::2], False), (big[:, :1], True)):
        t, ld = S._as_rows(view)
        cols = view.shape[-1]
        rows = torch.as_strided(t, (view.numel() // cols, cols), (ld, 1))
        assert torch.equal(rows, view.reshape(-1, cols))
        assert (t.data_ptr() == view.data_ptr()) == own


def test_c_row_entries_refuse(lib):
    _refused(lib, lib.qd_quantize_fp8(None, 128, A16, A16, 4, 128, 1, None), -1, b"null")
    _refused(lib, lib.qd_quantize_fp8(A16, 128, A16, A16, 4, 128, 64, None), -1, b"block_rows")
    _refused(lib, lib.qd_quantize_fp8(A16, 128, A16, A16, -1, 128, 1, None), -2, b"rows")
    _refused(lib, lib.qd_quantize_fp8(A16, 128, A16, A16, (1 << 23) + 1, 128, 1, None), -2, b"rows")
    _refused(lib, lib.qd_quantize_fp8(A16, 128, A16, A16, 4, 0, 1, None), -2, b"cols")
    _refused(lib, lib.qd_quantize_fp8(A16 + 1, 128, A16, A16, 4, 128, 1, None), -1, b"aligned")
    _refused(lib, lib.qd_silu_mul_fp8(A16, 128, None, 128, A16, A16, 4, 128, None), -1, b"up")
    _refused(lib, lib.qd_add_rmsnorm_fp8(A16, 128, A16, 128, None, A16, A16, A16, 4, 128, 1e-6, None), -1, b"null")
    _refused(lib, lib.qd_add_rmsnorm_fp8(A16 + 1, 128, A16, 128, A16, A16, A16, A16, 4, 128, 1e-6, None), -1, b"aligned")
    # nothing to do
    assert lib.qd_quantize_fp8(None, 128, None, None, 0, 128, 1, None) == 0
    assert lib.qd_silu_mul_fp8(None, 128, None, 128, None, None, 0, 128, None) == 0
    assert lib.qd_add_rmsnorm_fp8(None, 0, None, 128, None, None, None, None, 0, 128, 1e-6, None) == 0


def test_c_matmul_refuses(lib):
    def call(x=A16, y=A16, dtype=0, m=2, n=64, k=128):
        return lib.qd_block_matmul_fp8(x, A16, A16, A16, y, dtype, m, n, k, None)

    _refused(lib, call(dtype=7), -1, b"y_dtype")
    for over in (dict(k=0), dict(k=24), dict(n=0), dict(m=-1), dict(m=(1 << 20) + 1), dict(n=(1 << 24) + 1)):
        assert call(**over) == -2, over
    _refused(lib, call(x=None), -1, b"null")
    _refused(lib, call(x=A16 + 8), -1, b"aligned")
    _refused(lib, call(y=A16 + 4), -1, b"aligned")
    assert call(x=None, m=0) == 0


def test_c_cache_entries_refuse(lib):
    def update(q=A16, kc=A16, cos=A16, sb=8192, T=64, pos=A16, b=1, s=1, hq=4, hkv=2, qs=512):
        return lib.qd_q_rope_kv_update_fp8(q, qs, qs, 128, A16, 256, 256, 128, A16, 256, 256, 128, A16, A16, 1e-6, cos, A16,
                                           A16, kc, A16, A16, A16, sb, 8192, 1, 1, T, pos, b, s, hq, hkv, None)

    _refused(lib, update(T=100), -2, b"multiple of 64")
    _refused(lib, update(kc=None), -1, b"null")
    _refused(lib, update(kc=A16 + 8), -1, b"aligned")
    _refused(lib, update(sb=8200), -1, b"aligned")
    _refused(lib, update(q=None), -1, b"null")
    _refused(lib, update(q=A16 + 4), -1, b"aligned")
    _refused(lib, update(cos=A16 + 2), -1, b"aligned")
    _refused(lib, update(qs=510), -1, b"strides")
    _refused(lib, update(pos=A16 + 4), -1, b"aligned")
    for over in (dict(hq=3), dict(hq=130), dict(hkv=0), dict(s=-1), dict(b=40000)):
        assert update(**over) == -2, over
    assert update(q=None, s=0) == 0 and update(q=None, kc=None, b=0) == 0

    def read(rows, out=A16):
        return lib.qd_kv_read_fp8(A16, A16, A16, A16, 8192, 8192, 1, 1, 64, out, out, 1, 1, rows, None)

    _refused(lib, read(65), -2, b"rows")
    _refused(lib, read(-1), -2, b"rows")
    _refused(lib, read(3, None), -1, b"k_out")
    assert read(0, None) == 0


def test_c_attention_refuses(lib):
    def call(q=A16, T=64, scale=0.1, window=0, sinks=0, sq=1, hq=4, hkv=2, ws=None, n=0, stride=128, b=1):
        return lib.qd_attention_fp8(q, 512, stride, 512, A16, A16, A16, A16, 8192, 8192, 1, 1, T, A16, scale, window, sinks, A16,
                                    b, sq, hq, hkv, ws, n, None)

    _refused(lib, call(T=65), -2, b"multiple of 64")
    _refused(lib, call(q=None), -1, b"null")
    _refused(lib, call(q=A16 + 8), -1, b"aligned")
    _refused(lib, call(stride=132), -1, b"aligned")
    for scale in (0.0, -1.0, math.inf, math.nan):
        _refused(lib, call(scale=scale), -1, b"scale")
    _refused(lib, call(window=-1), -1, b"window")
    _refused(lib, call(sinks=-1), -1, b"window")
    for over in (dict(hq=5), dict(sq=-1), dict(sq=1 << 22, hq=4), dict(sq=20000, b=32767), dict(b=40000)):
        assert call(**over) == -2, over
    assert call(q=None, sq=0) == 0
    need = lib.qd_attention_fp8_workspace_bytes(1, 1, 16, 8, 32768, 0, 0)
    assert need > 0
    _refused(lib, call(T=32768, hq=16, hkv=8, ws=A16, n=need - 1), -3, b"workspace")
    _refused(lib, call(T=32768, hq=16, hkv=8, ws=None, n=need), -3, b"workspace")
    assert lib.qd_attention_fp8_workspace_bytes(0, 1, 16, 8, 64, 0, 0) == 0
    assert lib.qd_attention_fp8_workspace_bytes(1, 1, 16, 8, 32768, 64, 0) < need
