"""The 8-bit operators on the GPU against their 64-bit restatement
(oracle/fp8_oracle.py).

Bars.  Bytes and scales are equal where the value before rounding is exact (plain
rows, weights, V rows, rescaled rows).  Elsewhere a value is within half an e4m3
step of the 64-bit one (2^-4 relative, 2^-10 of the block's scale for subnormals)
plus the fp32 arithmetic's part, and a scale may differ only where the block's
largest value lies within that part of a power-of-two border.  Products and the
attention: see _product_bound and fp8_oracle.attention_bound."""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

EPS = 1e-6
FP32 = 2.0 ** -18   # relative part of the fp32 arithmetic before a rounding to e4m3: RMSNorm's sum of squares
                    # is at most 50 additions deep (8 per 2048 columns, 8 lane and wave steps), SiLU 4 steps


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu()


def _randn(g, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).half()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _check_quantized(q, scale, y, rows=1, low=O.ROW_LOW, what=""):
    """q, scale (2-D) against the 64-bit y, within the bars above."""
    q, scale, y = q.cpu(), scale.cpu(), y.cpu()
    e, ref = O.exponents(scale), O.block_exponents(y, rows, low)
    up, down = O.block_exponents(y * (1 + FP32), rows, low), O.block_exponents(y * (1 - FP32), rows, low)
    assert ((e == ref) | (e == up) | (e == down)).all(), f"{what}: scales differ"
    got = O.widen(q, scale, rows)
    finite = y.isfinite()
    assert torch.equal(finite, got.isfinite()), f"{what}: NaN in other places"
    bound = (O.HALF_STEP + FP32) * y.abs() + torch.ldexp(torch.tensor(O.TINY_STEP, dtype=torch.float64), O.spread(e, rows, y.shape))
    off = ((got - y).abs() - bound)[finite]
    print(f"[parity] {what}: worst off by {off.max().item() if off.numel() else 0:.3e} over its bound", flush=True)
    assert (off <= 0).all(), what


# ---------------------------------------------------------------- row quantisers

@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 128), (5, 129), (2, 2048), (37, 2056), (3, 6144), (2, 8200),
                                       (300, 200)])
def test_plain_rows_are_exact(cuda, rows, cols):
    import cuda_decode_small_ops as S

    x = _randn(_gen(rows * 1000 + cols), rows, cols) * torch.exp2(torch.randint(-12, 9, (rows, 1))).half()
    q, s = S.quantize_fp8(x.to(cuda))
    e = O.block_exponents(x, 1)
    assert q.shape == x.shape and s.shape == (rows, -(-cols // 128))
    assert torch.equal(_bytes(s), O.scale_bytes(e))
    assert torch.equal(_bytes(q), _bytes(O.round_f8(x, O.spread(e, 1, x.shape))))


@pytest.mark.parametrize("rows,cols", [(1, 16), (128, 128), (129, 2048), (300, 200), (17, 1001)])
def test_weight_blocks_are_exact(cuda, rows, cols):
    import cuda_decode_small_ops as S

    x = _randn(_gen(rows + cols), rows, cols, std=0.02)
    q, s = S.quantize_fp8(x.to(cuda), block_rows=128)
    e = O.block_exponents(x, 128)
    assert torch.equal(_bytes(s), O.scale_bytes(e))
    assert torch.equal(_bytes(q), _bytes(O.round_f8(x, O.spread(e, 128, x.shape))))


def test_special_values_and_borders(cuda):
    """Zeros, subnormals, 448 * 2^e itself and the value after it, infinities and NaN."""
    import cuda_decode_small_ops as S

    x = torch.zeros(7, 128, dtype=torch.float16)
    x[1, 5] = 2.0 ** -24
    x[2] = 448.0 * 2.0 ** -10
    x[3, 0] = float(torch.nextafter(torch.tensor(448.0 * 2.0 ** -10).half(), torch.tensor(1.0).half()))
    x[4] = torch.arange(128).half()
    x[4, 3], x[4, 9], x[4, 100] = float("inf"), float("nan"), float("-inf")
    x[5] = float("nan")
    x[6] = torch.linspace(-65504, 65504, 128).half()
    q, s = S.quantize_fp8(x.to(cuda))
    e = O.block_exponents(x, 1)
    assert e.flatten().tolist() == [-126, -32, -10, -9, -1, -126, 8]
    assert torch.equal(_bytes(s), O.scale_bytes(e))
    want = torch.where(x.isfinite(), O.round_f8(x, O.spread(e, 1, x.shape)).float(), torch.tensor(float("nan")))
    assert torch.equal(q.float().cpu().nan_to_num(nan=999.0), want.nan_to_num(nan=999.0))


@pytest.mark.parametrize("rows,cols", [(1, 2048), (37, 2048), (2, 6144), (3, 100), (5, 4104), (2, 9000), (4, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_rms_norm_rows(cuda, rows, cols, residual):
    import cuda_decode_small_ops as S

    g = _gen(cols + rows)
    x, r = _randn(g, rows, cols), _randn(g, rows, cols, std=3.0)
    w = _randn(g, cols, std=0.1, mean=1.0)
    if residual:
        total, q, s = S.fused_add_rms_norm_fp8(r.to(cuda), x.to(cuda), w.to(cuda), EPS)
        assert torch.equal(total.cpu(), (r.float() + x.float()).half())
        y = O.rms_norm(r.double() + x.double(), w, EPS)
    else:
        q, s = S.rms_norm_fp8(x.to(cuda), w.to(cuda), EPS)
        y = O.rms_norm(x, w, EPS)
    _check_quantized(q, s, y, what=f"norm {rows}x{cols}")


@pytest.mark.parametrize("rows,cols", [(1, 6144), (37, 6144), (3, 100), (9, 2052)])
def test_silu_mul_rows_of_a_fused_product(cuda, rows, cols):
    import cuda_decode_small_ops as S

    gu = _randn(_gen(cols), rows, 2 * cols, std=4.0)
    gate, up = gu.to(cuda).chunk(2, -1)
    q, s = S.fused_silu_mul_fp8(gate, up)
    t = gu.double()
    _check_quantized(q, s, t[:, :cols] / (1 + torch.exp(-t[:, :cols])) * t[:, cols:], what=f"silu {rows}x{cols}")


def test_silu_keeps_its_precision_far_out(cuda):
    """Gates of one size per block, from -80 to 80: e^-v has |v| times the rounding of its
    exponent unless that is made up for."""
    import cuda_decode_small_ops as S

    g = _gen(4)
    gate = torch.tensor([-80.0, -60, -30, -5, -1e-3, 0, 1e-3, 5, 30, 80]).half()[:, None] + _randn(g, 10, 128, std=0.05)
    up = _randn(g, 10, 128)
    q, s = S.fused_silu_mul_fp8(gate.to(cuda), up.to(cuda))
    t = gate.double()
    _check_quantized(q, s, t / (1 + torch.exp(-t)) * up.double(), what="silu far out")


def test_silu_of_every_finite_gate(cuda):
    """All 63488 finite fp16 gates in order, 128 neighbours to a block."""
    import cuda_decode_small_ops as S

    g = torch.arange(0x7C00, dtype=torch.int16).view(torch.float16)
    g = torch.cat([-g.flip(0), g]).view(-1, 128)
    q, s = S.fused_silu_mul_fp8(g.to(cuda), torch.ones_like(g).to(cuda))
    assert not torch.isnan(q.float()).any()
    t = g.double()
    _check_quantized(q, s, t / (1 + torch.exp(-t)), what="silu of every gate")


def test_rows_at_odd_strides_and_ranks(cuda):
    import cuda_decode_small_ops as S

    g = _gen(3)
    big = _randn(g, 4, 6, 300).to(cuda)
    for view in (big[:, ::2, 3:259], big.transpose(0, 1)[..., :256], big[1:2, :, 1:2], big[..., 5:5 + 130], big[0, 0],
                 big[:, :1].expand(4, 5, 300)):
        q, s = S.quantize_fp8(view)
        q2, s2 = S.quantize_fp8(view.contiguous())
        assert q.shape == view.shape and torch.equal(_bytes(q), _bytes(q2)) and torch.equal(_bytes(s), _bytes(s2))
    q, s = S.quantize_fp8(big[:0])
    assert q.shape == (0, 6, 300) and s.shape == (0, 6, 3)


# ---------------------------------------------------------------- block-scaled product

def _operands(g, m, n, k, cuda):
    import cuda_decode_small_ops as S

    x = _randn(g, m, k) * torch.exp2(torch.randint(-6, 7, (m, 1))).half()
    w = _randn(g, n, k, std=0.02) * torch.exp2(torch.randint(-3, 4, (n, 1))).half()
    return S.quantize_fp8(x.to(cuda)), S.quantize_fp8(w.to(cuda), block_rows=128)


def _product_bound(xd, wd, out, dtype):
    """fp32 sums of exact products: K additions, each within 2^-23 of the running
    |sum| <= sum |x w| (to nearest 2^-24; a matrix unit may truncate); then the result's
    type.  fp16 results of more than 16 rows: of each 8 neighbouring products up to 7
    lose what is below 2^-13 of the largest, so at most 7 * 2^-13 of sum |x w|."""
    k, half = xd.shape[1], dtype == torch.float16
    part = k * 2.0 ** -23 + (7 * 2.0 ** -13 if half and xd.shape[0] > 16 else 0.0)
    return part * (xd.abs() @ wd.abs().T) + (2.0 ** -11 * out.abs() + 2.0 ** -25 if half else 2.0 ** -24 * out.abs())


SHAPES = [(1, 16, 16), (1, 4096, 2048), (3, 100, 144), (8, 1000, 2048), (16, 129, 6144), (17, 130, 2048), (33, 2048, 400),
          (64, 257, 1040), (65, 300, 2048), (128, 128, 128), (200, 1111, 272), (257, 600, 2048), (300, 128, 6144),
          (513, 2048, 1008), (1029, 4096, 2048), (5, 60000, 2048), (16, 33000, 1152), (2000, 1500, 1024), (1300, 12288, 576),
          (2111, 8200, 2048), (700, 1004, 7424), (130, 12288, 144), (770, 500, 144), (1029, 6000, 7296), (1029, 1004, 1152),
          (1029, 500, 144), (500, 8200, 576), (1029, 8200, 1152), (1029, 8199, 576), (16, 33001, 1040)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_block_matmul(cuda, m, n, k, dtype):
    import cuda_decode_gemv as G

    (x, xs), (w, ws) = _operands(_gen(m + n + k), m, n, k, cuda)
    y = G.block_matmul_fp8(x, xs, w, ws, out_dtype=dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    xd, wd = O.widen(x, xs, 1), O.widen(w, ws, 128)
    ref = xd @ wd.T
    off = (y.double() - ref).abs() - _product_bound(xd, wd, ref, dtype)
    print(f"[parity] matmul {m}x{n}x{k}: rel {((y.double() - ref).norm() / ref.norm()).item():.2e}", flush=True)
    assert (off <= 0).all()


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_block_matmul_of_small_integers_is_exact(cuda, m, n, k, dtype):
    """Integers whose sums fit fp32 with any power-of-two scales: nothing is rounded
    but the result, so every term counts once, at its own scale."""
    import cuda_decode_gemv as G

    g = _gen(n)
    kb = -(-k // 128)
    x = torch.randint(-4, 5, (m, k), generator=g).float().to(O.F8)
    w = torch.randint(-4, 5, (n, k), generator=g).float().to(O.F8)
    xs = torch.randint(125, 128, (m, kb), generator=g).to(torch.uint8).view(O.E8)
    ws = torch.randint(126, 129, (-(-n // 128), kb), generator=g).to(torch.uint8).view(O.E8)
    y = G.block_matmul_fp8(x.to(cuda), xs.to(cuda), w.to(cuda), ws.to(cuda), out_dtype=dtype)
    ref = O.widen(x.to(cuda), xs.to(cuda), 1) @ O.widen(w.to(cuda), ws.to(cuda), 128).T
    assert torch.equal(y, ref.to(dtype))


def test_block_matmul_far_scales_nan_rows_and_ranks(cuda):
    """Block scales at both ends; a NaN stays in its row (or column); zero rows; ranks."""
    import cuda_decode_gemv as G

    (x, xs), (w, ws) = _operands(_gen(5), 70, 200, 384, cuda)
    base = G.block_matmul_fp8(x, xs, w, ws, out_dtype=torch.float32)
    x2, w2 = x.clone(), w.clone()
    x2.view(torch.uint8)[7, 200] = 0x7F
    w2.view(torch.uint8)[31, 3] = 0xFF
    y = G.block_matmul_fp8(x2, xs, w2, ws, out_dtype=torch.float32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7], bad[:, 31] = True, True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], base[~bad])
    # 2^100 * 2^-100: the operands' scales meet before anything is rounded
    up, down = xs.view(torch.uint8) + 100, ws.view(torch.uint8) - 100
    assert torch.equal(G.block_matmul_fp8(x, up.view(O.E8), w, down.view(O.E8), out_dtype=torch.float32), base)
    assert G.block_matmul_fp8(x[:0], xs[:0], w, ws).shape == (0, 200)
    y3 = G.block_matmul_fp8(x.view(2, 35, 384), xs.view(2, 35, 3), w, ws, out_dtype=torch.float32)
    assert torch.equal(y3.view(70, 200), base)
    one = G.block_matmul_fp8(x[3], xs[3], w, ws, out_dtype=torch.float32)
    assert one.shape == (200,)
    # strided operands are copied
    assert torch.equal(G.block_matmul_fp8(x[::2], xs[::2], w, ws, out_dtype=torch.float32),
                       G.block_matmul_fp8(x[::2].contiguous(), xs[::2].contiguous(), w, ws, out_dtype=torch.float32))


@pytest.mark.parametrize("m", [1, 16, 40, 100, 300])
def test_block_matmul_rows_do_not_depend_on_the_others(cuda, m):
    """A row's result has the same bits whatever the rows beside it hold."""
    import cuda_decode_gemv as G

    (x, xs), (w, ws) = _operands(_gen(m), m, 512, 2048, cuda)
    y = G.block_matmul_fp8(x, xs, w, ws)
    x2 = x.clone()
    x2.view(torch.uint8)[1:] = 0x7F
    y2 = G.block_matmul_fp8(x2, xs, w, ws)
    assert torch.equal(y[0], y2[0])


# ---------------------------------------------------------------- the cache

def _new_tokens(g, b, s, hq, hkv):
    t = dict(q=_randn(g, b, s, hq, 128), k=_randn(g, b, s, hkv, 128), v=_randn(g, b, s, hkv, 128))
    t["v"] *= torch.exp2(torch.randint(-9, 7, (b, s, 1, 1), generator=g)).half()
    t.update(qw=_randn(g, 128, std=0.2, mean=1.0), kw=_randn(g, 128, std=0.2, mean=1.0))
    ang = torch.rand(b, s, 64, generator=g) * 6.28
    t.update(cos=torch.cat([ang, ang], -1).cos().half(), sin=torch.cat([ang, ang], -1).sin().half())
    return t


def _update(S, t, cache, pos, cuda):
    d = {n: v.to(cuda) for n, v in t.items()}
    cp = torch.tensor(pos, dtype=torch.int64, device=cuda)
    return S.fused_q_rope_kv_cache_update_fp8(d["q"], d["k"], d["v"], d["qw"], d["kw"], EPS, d["cos"], d["sin"], cache, cp)


def _rotated_check(out, x, w, cos, sin, what):
    """fp16 result: half a step, and the fp32 rotation's part of both its terms."""
    n = O.rms_norm(x, w, EPS)
    y = O.rope(n, cos, sin)
    size = O.rope(n.abs(), cos.abs(), sin.abs()) if False else (n * cos.double()[:, :, None]).abs() + (n.roll(64, -1) * sin.double()[:, :, None]).abs()
    off = (out.cpu().double() - y).abs() - (2.0 ** -11 * y.abs() + FP32 * size + 2.0 ** -25)
    assert (off <= 0).all(), what
    return y, size


def _check_update(before, cache, t, pos, what):
    """The cache after a write of S tokens at pos, against the one before it."""
    s, T = t["k"].shape[1], cache.k.shape[2]
    y = O.rope(O.rms_norm(t["k"], t["kw"], EPS), t["cos"], t["sin"])
    # per (sequence, head) views with rows first
    for name, new in (("k", y), ("v", t["v"].double())):
        vals, sc = getattr(cache, name).cpu(), getattr(cache, name + "_scale").cpu()
        old, osc = getattr(before, name).cpu(), getattr(before, name + "_scale").cpu()
        if name == "v":
            vals, old = (x.transpose(-1, -2).reshape(*x.shape[:2], -1, 128) for x in (vals, old))
        e, e_old = O.exponents(sc), O.exponents(osc)
        for b, p in enumerate(pos):
            for blk in range(T // 64):
                lo, hi = max(p, blk * 64), min(p + s, blk * 64 + 64)
                rows = slice(blk * 64, blk * 64 + 64)
                if lo >= hi:   # untouched
                    assert torch.equal(_bytes(vals[b, :, rows]), _bytes(old[b, :, rows])), f"{what}: block {blk} of {b}"
                    assert torch.equal(e[b, :, blk], e_old[b, :, blk])
                    continue
                for h in range(vals.shape[1]):
                    part = new[b, lo - p:hi - p, h]
                    floor = int(e_old[b, h, blk]) if lo > blk * 64 else O.KV_LOW
                    cand = {max(O.exponent(float(part.abs().max()) * f, O.KV_LOW), floor) for f in (1 - FP32, 1, 1 + FP32)}
                    ee = int(e[b, h, blk])
                    assert ee in cand, f"{what}: {name} scale of block {blk}: {ee} not in {cand}"
                    got = torch.ldexp(vals[b, h, lo:hi].double(), torch.tensor(ee))
                    if name == "v":
                        assert torch.equal(_bytes(vals[b, h, lo:hi]), _bytes(O.round_f8(part, torch.tensor(ee))))
                    else:
                        bound = (O.HALF_STEP + FP32) * part.abs() + O.TINY_STEP * 2.0 ** ee + FP32 * part.abs().max()
                        assert ((got - part).abs() <= bound).all(), f"{what}: K rows of block {blk}"
                    earlier = old[b, h, blk * 64:lo]
                    if lo > blk * 64:
                        kept = (earlier.float() * 2.0 ** (int(e_old[b, h, blk]) - ee)).to(O.F8)
                        assert torch.equal(_bytes(vals[b, h, blk * 64:lo]), _bytes(kept)), f"{what}: earlier rows"
                    assert torch.equal(_bytes(vals[b, h, hi:blk * 64 + 64]), _bytes(old[b, h, hi:blk * 64 + 64])), f"{what}: later rows"


def _snapshot(S, cache):
    return S.KVCacheFP8(*(t.clone() for t in cache))


def _filled(S, b, h, cap, cuda, seed=0):
    """A cache whose every byte holds something (no NaN), scales in a usual range."""
    c = S.new_kv_cache_fp8(b, h, cap, cuda)
    g = _gen(seed)
    for t in (c.k, c.v):
        r = torch.randint(0, 0x7F, t.shape, generator=g) | (torch.randint(0, 2, t.shape, generator=g) << 7)
        t.view(torch.uint8).copy_(r.to(torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.view(torch.uint8).copy_(torch.randint(127 - 12, 127 - 5, t.shape, generator=g).to(torch.uint8))
    return c


@pytest.mark.parametrize("s,pos", [(1, [0, 63, 64]), (1, [200, 5, 127]), (2, [63, 62, 191]), (7, [0, 60, 100]),
                                   (64, [0, 64, 1]), (65, [0, 63, 64]), (129, [0, 31, 63]), (1, [-1, 256, 255]),
                                   (3, [-2, 254, 400]), (70, [-5, 250, -200])])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (3, 1)])
def test_cache_update(cuda, s, pos, hq, hkv):
    import cuda_decode_small_ops as S

    t = _new_tokens(_gen(s + hq), 3, s, hq, hkv)
    cache = _filled(S, 3, hkv, 256, cuda, seed=s)
    before = _snapshot(S, cache)
    q = _update(S, t, cache, pos, cuda)
    _rotated_check(q, t["q"], t["qw"], t["cos"], t["sin"], "q")
    _check_update(before, cache, t, pos, f"S={s} pos={pos}")


def test_cache_token_by_token_and_at_once(cuda):
    """Rows appended one at a time to a fresh cache: the same scales in the end, and
    values that differ from a whole write only by the subnormals that a growing scale
    rounded again (at most half a subnormal step at each growth)."""
    import cuda_decode_small_ops as S

    n, b, hkv = 150, 2, 2
    t = _new_tokens(_gen(11), b, n, 4, hkv)
    whole, steps = S.new_kv_cache_fp8(b, hkv, n, cuda), S.new_kv_cache_fp8(b, hkv, n, cuda)
    assert whole.k.shape[2] == 192
    _update(S, t, whole, [0, 0], cuda)
    for i in range(n):
        one = {x: (v[:, i:i + 1] if v.ndim > 1 else v) for x, v in t.items()}
        _update(S, one, steps, [i, i], cuda)
    for name in ("k", "v"):
        sw, ss = getattr(whole, name + "_scale"), getattr(steps, name + "_scale")
        assert torch.equal(_bytes(sw), _bytes(ss))
        a, c = (O.cache_rows(getattr(x, name).cpu(), getattr(x, name + "_scale").cpu(), name == "v") for x in (whole, steps))
        step = torch.ldexp(torch.tensor(2.0 ** -9, dtype=torch.float64), O.exponents(sw.cpu())).repeat_interleave(64, 2)[..., None]
        # half a step now, and half a (finer) step at each growth before: under two half steps in all
        assert ((a - c).abs() <= step)[:, :, :n].all()


def test_cache_views_of_sequences_and_heads(cuda):
    """A write through a view of some sequences and heads touches nothing else."""
    import cuda_decode_small_ops as S

    cache = _filled(S, 4, 3, 128, cuda)
    before = _snapshot(S, cache)
    view = S.KVCacheFP8(*(t[1:3, 1:] for t in cache))
    t = _new_tokens(_gen(2), 2, 5, 4, 2)
    _update(S, t, view, [62, 3], cuda)
    _check_update(S.KVCacheFP8(*(x[1:3, 1:] for x in before)), view, t, [62, 3], "view")
    for a, c in zip(cache, before):
        a, c = a.view(torch.uint8).clone(), c.view(torch.uint8).clone()
        a[1:3, 1:], c[1:3, 1:] = 0, 0
        assert torch.equal(a, c)


def test_cache_update_takes_strided_inputs(cuda):
    """q, k, v as slices of one qkv product."""
    import cuda_decode_small_ops as S

    t = _new_tokens(_gen(8), 2, 9, 4, 2)
    qkv = torch.cat([t["q"].flatten(2), t["k"].flatten(2), t["v"].flatten(2)], -1).to(cuda).view(2, 9, 8, 128)
    a, b = _filled(S, 2, 2, 128, cuda), _filled(S, 2, 2, 128, cuda)
    q1 = _update(S, t, a, [60, 0], cuda)
    cp = torch.tensor([60, 0], device=cuda)
    q2 = S.fused_q_rope_kv_cache_update_fp8(qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:], t["qw"].to(cuda), t["kw"].to(cuda),
                                            EPS, t["cos"].to(cuda), t["sin"].to(cuda), b, cp)
    assert torch.equal(q1, q2)
    for x, y in zip(a, b):
        assert torch.equal(_bytes(x), _bytes(y))
    # operands at odd addresses are copied
    odd = {n: torch.empty(v.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(v.shape).copy_(v) for n, v in t.items()}
    c = _filled(S, 2, 2, 128, cuda)
    q3 = S.fused_q_rope_kv_cache_update_fp8(odd["q"], odd["k"], odd["v"], odd["qw"], odd["kw"], EPS, odd["cos"], odd["sin"], c, cp)
    assert torch.equal(q1, q3)
    for x, y in zip(a, c):
        assert torch.equal(_bytes(x), _bytes(y))


def test_cache_keeps_nonfinite_rows_apart(cuda):
    """NaN and infinities become NaN in their own places and do not move the scale."""
    import cuda_decode_small_ops as S

    t = _new_tokens(_gen(21), 1, 70, 2, 1)
    clean, cache = S.new_kv_cache_fp8(1, 1, 128, cuda), S.new_kv_cache_fp8(1, 1, 128, cuda)
    _update(S, t, clean, [0], cuda)
    big = t["v"][0, :64].abs().amax((1, 2))
    row = int(big.argmin())   # not the row that sets the scale
    t["v"][0, row, 0, 17], t["v"][0, row, 0, 99] = float("inf"), float("nan")
    _update(S, t, cache, [0], cuda)
    assert torch.equal(_bytes(clean.v_scale), _bytes(cache.v_scale))
    got = O.cache_rows(cache.v.cpu(), cache.v_scale.cpu(), True)
    assert got[0, 0, row, 17].isnan() and got[0, 0, row, 99].isnan() and int(got.isnan().sum()) == 2


@pytest.mark.parametrize("b,h,cap,rows", [(1, 1, 64, 1), (2, 3, 192, 130), (1, 8, 1024, 1024), (3, 2, 128, 65), (1, 2, 64, 0)])
def test_cache_read(cuda, b, h, cap, rows):
    import cuda_decode_small_ops as S

    cache = _filled(S, b, h, cap, cuda, seed=rows)
    k, v = S.read_kv_cache_fp8(cache, rows)
    for got, name in ((k, "k"), (v, "v")):
        ref = O.cache_rows(getattr(cache, name), getattr(cache, name + "_scale"), name == "v")[:, :, :rows]
        assert got.shape == (b, h, rows, 128) and torch.equal(got, ref.half())
    view = S.KVCacheFP8(*(t[:, -1:] for t in cache))
    assert torch.equal(S.read_kv_cache_fp8(view, rows)[1], v[:, -1:])


# ---------------------------------------------------------------- attention

SCALE = 128 ** -0.5


def _attend_check(q, cache, pos, window=0, sinks=0, scale=SCALE, workspace=None, what=""):
    import cuda_decode_attention as A

    cp = torch.tensor(pos, dtype=torch.int64, device=q.device)
    out = A.attn_fp8_kv_cache(q, cache, scale, cp, window=window, sinks=sinks, workspace=workspace)
    b, hq, sq, _ = q.shape
    assert out.shape == (b, sq, hq, 128) and out.dtype == torch.float16
    k, v = O.cache_rows(cache.k, cache.k_scale, False), O.cache_rows(cache.v, cache.v_scale, True)
    ref, mass, big = O.attention(q, k, v, pos, scale, window, sinks)
    assert torch.equal(out.isnan(), ref.isnan()), f"{what}: NaN in other places"
    off = ((out.double() - ref).abs() - O.attention_bound(ref, mass, big)).nan_to_num(nan=-1.0)
    rel = (out.double() - ref).nan_to_num().norm() / ref.nan_to_num().norm().clamp_min(1e-300)
    print(f"[parity] {what}: rel {rel.item():.2e}, worst {off.max().item():.2e} over its bound", flush=True)
    assert (off <= 0).all(), what
    return out


def _attend_inputs(S, cuda, b, hq, hkv, sq, cap, seed=1):
    """Rows in the sizes a model's have: unit K, V blocks of sizes 2^-6 to 2^6."""
    g = _gen(seed)
    cache = _filled(S, b, hkv, cap, cuda, seed)
    for t in (cache.k, cache.v):
        t.copy_((torch.randn(t.shape, generator=g) * 60).clamp(-448, 448).to(O.F8).to(cuda))
    cache.k_scale.view(torch.uint8).fill_(127 - 6)
    e = torch.randint(-12, 1, cache.v_scale.shape, generator=g)
    cache.v_scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))
    q = _randn(g, b, sq, hq, 128).to(cuda).transpose(1, 2)
    return q, cache


@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (8, 2), (3, 1), (16, 1), (40, 2)])
@pytest.mark.parametrize("lens", [[1, 2, 64], [65, 63, 400], [1029, 1, 700]])
def test_decode_attention(cuda, hq, hkv, lens):
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 3, hq, hkv, 1, -(-max(lens) // 64) * 64)
    _attend_check(q, cache, [n - 1 for n in lens], what=f"decode Hq={hq} Hkv={hkv} {lens}")


@pytest.mark.parametrize("sq", [2, 5, 8, 9, 16, 17, 32, 33, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("groups", [1, 2, 5])
def test_several_query_tokens(cuda, sq, groups):
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 2, 2 * groups, 2, sq, 768, seed=sq)
    _attend_check(q, cache, [0, 700 - sq], what=f"Sq={sq} G={groups}")


@pytest.mark.parametrize("sq", [1, 7, 40, 200])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (50, 4), (64, 64), (128, 70), (100, 1000), (5000, 3), (200, 0)])
def test_window_and_sinks(cuda, sq, window, sinks):
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 3, 4, 2, sq, 896, seed=window + sinks)
    _attend_check(q, cache, [0, 896 - sq, 333], window=window, sinks=sinks, what=f"Sq={sq} W={window} sinks={sinks}")


@pytest.mark.parametrize("sq", [1, 20, 150])
def test_rows_that_see_nothing_and_positions_past_the_cache(cuda, sq):
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 5, 4, 2, sq, 256, seed=sq)
    pos = [-1, -sq, -3 if sq > 3 else -10 ** 12, 256, 10 ** 9]
    out = _attend_check(q, cache, pos, what=f"empty Sq={sq}")
    assert (out[1, :sq - 1 if sq > 1 else 1] == 0).all()
    _attend_check(q, cache, pos, window=100, what=f"empty Sq={sq} W=100")   # a window past the end sees nothing
    q, cache = _attend_inputs(S, cuda, 1, 2, 1, sq, 64, seed=sq)
    _attend_check(q, cache, [1000], window=5, sinks=3, what="window behind the cache, sinks in it")


@pytest.mark.parametrize("sq", [1, 3, 40, 150])
@pytest.mark.parametrize("window", [0, 70])
def test_nan_in_rows_that_are_not_seen(cuda, sq, window):
    """NaN bytes behind the end, before the window and between the query tokens'
    own limits reach only the rows that see them."""
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 2, 4, 2, sq, 512, seed=7)
    pos = [300 - sq, 190]
    for b, p in enumerate(pos):
        cache.k.view(torch.uint8)[b, :, p + sq:] = 0x7F
        rows = cache.v.view(torch.uint8)[b].transpose(-1, -2)   # [H, blocks, 64, 128]
        for t in range(p + sq, 512):
            rows[:, t // 64, t % 64] = 0xFF
    # visible to the last token alone, in one dim of one head
    last = pos[0] + sq - 1
    cache.v.view(torch.uint8)[0, 1, last // 64, 77, last % 64] = 0x7F
    if window:
        old = pos[1] - window   # no token of sequence 1 sees it
        cache.v.view(torch.uint8)[1, 0, old // 64, :, old % 64] = 0x7F
        cache.k.view(torch.uint8)[1, 0, old] = 0x7F
    out = _attend_check(q, cache, pos, window=window, what=f"NaN Sq={sq} W={window}")
    assert int(out.isnan().sum()) == 2   # the two q heads of kv head 1, one dim, the last token


@pytest.mark.parametrize("sq", [1, 60])
def test_nan_in_a_key_or_query_that_is_seen(cuda, sq):
    """A visible K row or a query with a NaN makes its own rows NaN, all of them, and
    no others."""
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 1, 4, 2, sq, 256, seed=5)
    last = 200
    cache.k.view(torch.uint8)[0, 1, last, 9] = 0x7F       # seen by the last token only
    q[0, 1, 0, 3] = float("nan")                          # head 1, first token
    q[0, 0, 0, 5] = float("inf")
    out = _attend_check(q, cache, [last + 1 - sq], what=f"NaN in K, Sq={sq}")
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, -1, 2:], bad[0, 0, :2] = True, True
    assert torch.equal(out.isnan(), bad)


def test_rows_of_a_fresh_cache_count_as_zeros(cuda):
    """Rows that were never written are zeros with a weight like any other."""
    import cuda_decode_small_ops as S

    for sq in (1, 70):
        fresh = S.new_kv_cache_fp8(2, 2, 300, cuda)
        t = _new_tokens(_gen(3), 2, 80, 4, 2)
        _update(S, t, fresh, [0, 128], cuda)
        q = _randn(_gen(6), 2, sq, 4, 128).to(cuda).transpose(1, 2)
        _attend_check(q, fresh, [300 - sq, 299 - sq], what=f"fresh rows Sq={sq}")


def test_one_prefix_shared_by_a_batch(cuda):
    """One sequence's cache expanded to several is read; writing through it is refused."""
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 4, 4, 2, 2, 256, seed=8)
    shared = S.KVCacheFP8(*(t[:1].expand(4, *t.shape[1:]) for t in cache))
    pos = torch.tensor([100, 254, 3, 77], device=cuda)
    out = A.attn_fp8_kv_cache(q, shared, SCALE, pos)
    for b in range(4):
        one = A.attn_fp8_kv_cache(q[b:b + 1], S.KVCacheFP8(*(t[:1] for t in cache)), SCALE, pos[b:b + 1])
        assert torch.equal(out[b:b + 1], one)
    t = _new_tokens(_gen(2), 4, 1, 4, 2)
    with pytest.raises(RuntimeError, match="share"):
        _update(S, t, shared, [0, 1, 2, 3], cuda)
    with pytest.raises(RuntimeError, match="share"):   # rows of their own, one set of scales
        _update(S, t, S.KVCacheFP8(cache.k, cache.v, shared.k_scale, shared.v_scale), [0, 1, 2, 3], cuda)


@pytest.mark.parametrize("b", [3, 9, 17])
def test_a_batch_gives_each_sequence_its_own_bits(cuda, b):
    """8 kv heads of 3, 9 and 17 sequences: the dims of a head on four, two and one
    workgroups; the result is the same."""
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, b, 16, 8, 2, 1152, seed=b)
    cache.v.view(torch.uint8)[1, 2, 5, 77, 3] = 0x7F     # row 323 of a sequence that stops before it
    cache.v.view(torch.uint8)[2, 3, 1, 120, 9] = 0x7F    # row 73 of one that sees it
    pos = [int(x) for x in torch.randint(0, 1150, (b,), generator=_gen(b))]
    pos[:3] = [1150, 300, 500]
    out = _attend_check(q, cache, pos, window=900, sinks=70, what=f"{b} sequences")
    for i in range(b):
        one = A.attn_fp8_kv_cache(q[i:i + 1], S.KVCacheFP8(*(t[i:i + 1] for t in cache)), SCALE,
                                  torch.tensor(pos[i:i + 1], device=cuda), window=900, sinks=70)
        assert torch.equal(out[i:i + 1].nan_to_num(nan=9e4), one.nan_to_num(nan=9e4)), i


def test_one_visible_row_is_returned(cuda):
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 1, 4, 2, 1, 64)
    out = A.attn_fp8_kv_cache(q, cache, SCALE, torch.zeros(1, dtype=torch.int64, device=cuda))
    v = O.cache_rows(cache.v, cache.v_scale, True)[0, :, 0]
    assert torch.equal(out[0, 0], v.repeat_interleave(2, 0).half())


def test_block_scales_far_apart(cuda):
    """V blocks from the smallest scale to large ones, an all-zero block, and rows whose
    weight sits in the small ones."""
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 1, 2, 1, 1, 512, seed=13)
    e = torch.tensor([-32, 3, -20, -32, 5, -8, -31, 0])
    cache.v_scale.view(torch.uint8)[0, 0] = (e + 127).to(torch.uint8).to(cuda)
    cache.v[0, 0, 3].zero_()
    for p in (63, 100, 260, 511):
        _attend_check(q, cache, [p], what=f"scales far apart, pos {p}")
    q.mul_(20)   # one row takes nearly all the weight
    for p in (63, 100, 260, 511):
        _attend_check(q, cache, [p], what=f"scales far apart, sharp, pos {p}")


@pytest.mark.parametrize("length,sq", [(30001, 1), (30001, 6), (8192, 100), (20000, 40)])
def test_long_contexts(cuda, length, sq):
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 1, 4, 2, sq, -(-length // 64) * 64 + 128, seed=length)
    _attend_check(q, cache, [length - sq], what=f"length {length} Sq={sq}")


def test_offsets_beyond_32_bits(cuda):
    """A cache of 4.9e9 bytes per tensor: reads and writes behind 2^32."""
    import cuda_decode_small_ops as S

    T = 64 * 75000
    cache = S.new_kv_cache_fp8(1, 8, T, cuda)
    base, sq = T - 400, 5
    t = _new_tokens(_gen(1), 1, 330, 16, 8)
    _update(S, t, cache, [base], cuda)
    q = _randn(_gen(2), 1, sq, 16, 128).to(cuda).transpose(1, 2)
    small = S.new_kv_cache_fp8(1, 8, 448, cuda)
    shift = base - (T - 448)   # the same rows at the same places of their blocks
    _update(S, t, small, [shift], cuda)
    for a, b in zip(cache, small):
        n = b.shape[2]
        assert torch.equal(_bytes(a[:, :, -n:]), _bytes(b))
    import cuda_decode_attention as A

    far = A.attn_fp8_kv_cache(q, cache, SCALE, torch.tensor([base + 330 - sq], device=cuda), window=200)
    near = A.attn_fp8_kv_cache(q, small, SCALE, torch.tensor([shift + 330 - sq], device=cuda), window=200)
    k, v = O.cache_rows(small.k, small.k_scale, False), O.cache_rows(small.v, small.v_scale, True)
    ref, mass, big = O.attention(q, k, v, [shift + 330 - sq], SCALE, 200)
    for out in (far, near):
        assert ((out.double() - ref).abs() <= O.attention_bound(ref, mass, big)).all()
    del cache
    torch.cuda.empty_cache()


def test_strided_queries_and_cache_views(cuda):
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 3, 8, 4, 6, 256, seed=4)
    pos = torch.tensor([100, 3, 250], device=cuda)
    whole = A.attn_fp8_kv_cache(q, cache, SCALE, pos)
    assert torch.equal(A.attn_fp8_kv_cache(q.contiguous(), cache, SCALE, pos), whole)
    part = A.attn_fp8_kv_cache(q[1:, 2:6], S.KVCacheFP8(*(t[1:, 1:3] for t in cache)), SCALE, pos[1:])
    assert torch.equal(part, whole[1:, :, 2:6])
    odd = torch.empty(3, 6, 8, 132, dtype=torch.float16, device=cuda)[..., 1:129]
    odd.copy_(q.transpose(1, 2))
    assert torch.equal(A.attn_fp8_kv_cache(odd.transpose(1, 2), cache, SCALE, pos), whole)
    assert A.attn_fp8_kv_cache(q[:, :, :0], cache, SCALE, pos).shape == (3, 0, 8, 128)


def test_equal_calls_give_equal_bits(cuda):
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 2, 16, 8, 3, 8192, seed=4)
    pos = torch.tensor([8000, 4321], device=cuda)
    ws = {}
    first = A.attn_fp8_kv_cache(q, cache, SCALE, pos, workspace=ws)
    for t in ws.values():
        t.fill_(255)   # the workspace holds nothing between calls
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = A.attn_fp8_kv_cache(q, cache, SCALE, pos)
    for _ in range(3):
        assert torch.equal(A.attn_fp8_kv_cache(q, cache, SCALE, pos, workspace=ws), first)
    side.synchronize()
    assert torch.equal(other, first)


def test_a_captured_call_keeps_its_workspace(cuda):
    """A larger call replaces the dict's workspace; what a graph captured with the first
    one writes to is not handed to anyone else."""
    import cuda_decode_attention as A
    import cuda_decode_small_ops as S

    q, cache = _attend_inputs(S, cuda, 2, 16, 8, 3, 8192, seed=5)
    pos = torch.tensor([8000, 4321], device=cuda)
    small = [q[:1, :, :1], S.KVCacheFP8(*(t[:1] for t in cache)), SCALE, pos[:1]]
    ws = {}
    want = A.attn_fp8_kv_cache(*small, workspace=ws)
    size = sum(t.numel() for t in ws.values())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.attn_fp8_kv_cache(*small, workspace=ws)
    A.attn_fp8_kv_cache(q, cache, SCALE, pos, workspace=ws)
    others = [torch.full((size,), 7, dtype=torch.uint8, device=cuda) for _ in range(8)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all((o == 7).all() for o in others)
        A.attn_fp8_kv_cache(q, cache, SCALE, pos, workspace=ws)


def test_refusals_before_any_launch(cuda):
    import cuda_decode_attention as A
    import cuda_decode_gemv as G
    import cuda_decode_small_ops as S

    def h(*shape):
        return torch.ones(shape, dtype=torch.float16, device=cuda)

    x, w = h(2, 256), h(256)
    qx, sx = S.quantize_fp8(x)
    wq, wsc = S.quantize_fp8(h(130, 256), block_rows=128)
    cache = S.new_kv_cache_fp8(2, 2, 128, cuda)
    pos = torch.zeros(2, dtype=torch.int64, device=cuda)
    q, kv, cs = h(2, 1, 4, 128), h(2, 1, 2, 128), h(2, 1, 128)

    def update(q=q, k=kv, v=kv, qw=h(128), cos=cs, cache=cache, pos=pos):
        return S.fused_q_rope_kv_cache_update_fp8(q, k, v, qw, h(128), EPS, cos, cs, cache, pos)

    def attend(q=q.transpose(1, 2), cache=cache, scale=SCALE, pos=pos, **more):
        return A.attn_fp8_kv_cache(q, cache, scale, pos, **more)

    calls = [
        lambda: S.quantize_fp8(x.float()), lambda: S.quantize_fp8(x.cpu()), lambda: S.quantize_fp8(x, block_rows=64),
        lambda: S.quantize_fp8(x[None], block_rows=128), lambda: S.quantize_fp8(x[:, :0]),
        lambda: S.fused_silu_mul_fp8(x, x[:1]), lambda: S.fused_add_rms_norm_fp8(x, x[:1], w, EPS),
        lambda: S.rms_norm_fp8(x, w[:255], EPS), lambda: S.rms_norm_fp8(x, w.bfloat16(), EPS),
        lambda: G.block_matmul_fp8(x, sx, wq, wsc), lambda: G.block_matmul_fp8(qx, sx.view(torch.uint8), wq, wsc),
        lambda: G.block_matmul_fp8(qx, sx[:, :1], wq, wsc), lambda: G.block_matmul_fp8(qx, sx, wq, wsc[:1]),
        lambda: G.block_matmul_fp8(qx[:, :128], sx[:, :1], wq, wsc), lambda: G.block_matmul_fp8(qx, sx, wq, wsc, torch.bfloat16),
        lambda: G.block_matmul_fp8(qx[:, :24], sx[:, :1], wq[:, :24], wsc[:, :1]),
        lambda: G.block_matmul_fp8(qx[:1].expand((1 << 20) + 1, 256), sx[:1].expand((1 << 20) + 1, 2), wq, wsc),
        lambda: S.new_kv_cache_fp8(0, 2, 64, cuda), lambda: S.new_kv_cache_fp8(1, 2, 0, cuda),
        lambda: S.read_kv_cache_fp8(cache, 129), lambda: S.read_kv_cache_fp8(cache, -1),
        lambda: S.read_kv_cache_fp8(cache._replace(v=cache.v.transpose(3, 4)), 1),
        lambda: S.read_kv_cache_fp8(cache._replace(k=cache.k.view(torch.uint8)), 1),
        lambda: S.read_kv_cache_fp8(cache._replace(k=cache.k[:, :, :100]), 1),
        lambda: S.read_kv_cache_fp8(cache._replace(k_scale=cache.k_scale[:, :1]), 1),
        lambda: S.read_kv_cache_fp8(cache._replace(k=cache.k[:, :, ::2]), 1),
        lambda: update(q=h(2, 1, 3, 128)), lambda: update(q=h(2, 1, 2 * 65, 128)), lambda: update(k=h(2, 2, 2, 128)),
        lambda: update(v=kv.cpu()), lambda: update(qw=h(64)), lambda: update(cos=h(1, 1, 128)), lambda: update(pos=pos.int()),
        lambda: update(pos=pos[:1]), lambda: update(q=q[..., :64]),
        lambda: attend(q=h(2, 3, 1, 128)), lambda: attend(q=h(1, 4, 1, 128)), lambda: attend(q=q.transpose(1, 2).float()),
        lambda: attend(window=-1), lambda: attend(sinks=-1), lambda: attend(window=1 << 31), lambda: attend(sinks=(1 << 32) + 1),
        lambda: attend(scale=0.0), lambda: attend(scale=-1.0), lambda: attend(scale=float("nan")),
        lambda: attend(scale=float("inf")), lambda: attend(pos=pos.cpu()), lambda: attend(pos=pos[None]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            print(f"call {i} was not refused", flush=True)


# ---------------------------------------------------------------- together

def test_decoder_layer_in_8_bits(cuda):
    """A decoder layer's operators in a row, prompt and decode steps, each checked against
    64 bits on the inputs it was given; then the decode step in a HIP graph, replayed
    with eager work in between, bit for bit the eager one."""
    import cuda_decode_attention as A
    import cuda_decode_gemv as G
    import cuda_decode_small_ops as S

    g = _gen(77)
    b, hid, hq, hkv, inter, cap = 2, 512, 4, 2, 768, 256
    mats = {n: _randn(g, r, c, std=0.05).to(cuda) for n, r, c in
            (("qkv", (hq + 2 * hkv) * 128, hid), ("o", hid, hq * 128), ("gate_up", 2 * inter, hid), ("down", hid, inter))}
    W = {n: S.quantize_fp8(m, block_rows=128) for n, m in mats.items()}
    norms = {n: _randn(g, c, std=0.1, mean=1.0).to(cuda) for n, c in (("in", hid), ("post", hid), ("q", 128), ("k", 128))}
    cache = S.new_kv_cache_fp8(b, hkv, cap, cuda)
    ws = {}

    def product(x, name, check):
        y = G.block_matmul_fp8(*x, *W[name])
        if check:
            xd = O.widen(x[0].flatten(0, -2), x[1].flatten(0, -2), 1)
            wd = O.widen(*W[name], 128)
            ref = xd @ wd.T
            assert ((y.flatten(0, -2).double() - ref).abs() <= _product_bound(xd, wd, ref, y.dtype)).all(), name
        return y

    def layer(x, residual, cos, sin, pos, check=True):
        r1, *n1 = S.fused_add_rms_norm_fp8(residual, x, norms["in"], EPS)
        if check:
            y = O.rms_norm(residual.double() + x.double(), norms["in"], EPS)
            _check_quantized(n1[0].flatten(0, 1), n1[1].flatten(0, 1), y.flatten(0, 1), what="input norm")
        s = x.shape[1]
        qkv = product(n1, "qkv", check).view(b, s, hq + 2 * hkv, 128)
        before = _snapshot(S, cache) if check else None
        q = S.fused_q_rope_kv_cache_update_fp8(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:], norms["q"],
                                               norms["k"], EPS, cos, sin, cache, pos)
        if check:
            t = dict(q=qkv[:, :, :hq].cpu(), k=qkv[:, :, hq:hq + hkv].cpu(), v=qkv[:, :, hq + hkv:].cpu(), kw=norms["k"].cpu(),
                     cos=cos.cpu(), sin=sin.cpu())
            _rotated_check(q, t["q"], norms["q"].cpu(), t["cos"], t["sin"], "q")
            _check_update(before, cache, t, pos.tolist(), "layer")
            att = _attend_check(q.transpose(1, 2), cache, pos.tolist(), workspace=ws, what="layer attention")
        else:
            att = A.attn_fp8_kv_cache(q.transpose(1, 2), cache, SCALE, pos, workspace=ws)
        o = product(S.quantize_fp8(att.flatten(2)), "o", check)
        r2, *n2 = S.fused_add_rms_norm_fp8(r1, o, norms["post"], EPS)
        gate, up = product(n2, "gate_up", check).chunk(2, -1)
        h = S.fused_silu_mul_fp8(gate, up)
        if check:
            t = gate.double()
            _check_quantized(h[0].flatten(0, 1), h[1].flatten(0, 1), (t / (1 + torch.exp(-t)) * up.double()).flatten(0, 1), what="silu")
        return r2, product(h, "down", check)

    def angles(s):
        a = torch.rand(b, s, 64, generator=g) * 6.28
        return torch.cat([a, a], -1).cos().half().to(cuda), torch.cat([a, a], -1).sin().half().to(cuda)

    zero = torch.zeros(b, 70, hid, dtype=torch.float16, device=cuda)
    layer(_randn(g, b, 70, hid).to(cuda), zero, *angles(70), torch.zeros(b, dtype=torch.int64, device=cuda))
    pos = torch.tensor([70, 66], device=cuda)
    x, res, (cos, sin) = _randn(g, b, 1, hid).to(cuda), _randn(g, b, 1, hid).to(cuda), angles(1)
    layer(x, res, cos, sin, pos)

    start = _snapshot(S, cache)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(x, res, cos, sin, pos, check=False)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x, res, cos, sin, pos, check=False)
    for step in range(4):
        pos += 1
        x.copy_(_randn(g, b, 1, hid))
        for c, s0 in zip(cache, start):
            c.copy_(s0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (*got, *cache)]
        for c, s0 in zip(cache, start):
            c.copy_(s0)
        eager = [*layer(x, res, cos, sin, pos, check=False), *cache]
        for a, e in zip(replayed, eager):
            assert torch.equal(a.view(torch.uint8), e.contiguous().view(torch.uint8)), f"replay {step}"
