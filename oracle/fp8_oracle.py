"""64-bit restatement of the 8-bit operators, for tests: block quantisers, the
block-scaled product, the KV cache in 64-row blocks and the attention over it.
Works on the device its inputs are on; shares no code with the library."""

from __future__ import annotations

import math

import torch

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
ROW_LOW, KV_LOW, KV_BLOCK, COLS = -126, -32, 64, 128
HALF_STEP = 2.0 ** -4     # e4m3: half a step relative to a normal value
TINY_STEP = 2.0 ** -10    # half a step of its subnormals


def exponent(amax: float, low: int) -> int:
    """Least e >= low with amax <= 448 * 2^e."""
    e = low
    if amax > 0:
        e = max(low, math.ceil(math.log2(amax / 448)) - 1)
        while amax > 448 * 2.0 ** e:
            e += 1
    return e


def scale_bytes(e: torch.Tensor) -> torch.Tensor:
    return (e + 127).to(torch.uint8)


def exponents(scale: torch.Tensor) -> torch.Tensor:
    """Integer exponents of E8M0 scales."""
    return scale.view(torch.uint8).long() - 127


def block_exponents(y: torch.Tensor, rows: int, low: int = ROW_LOW) -> torch.Tensor:
    """Exponents of y [M, N] in blocks of rows x 128."""
    f = torch.where(y.isfinite(), y.double().abs(), torch.zeros_like(y, dtype=torch.float64))
    r, c = -(-y.shape[0] // rows), -(-y.shape[1] // COLS)
    out = torch.empty(r, c, dtype=torch.int64)
    for i in range(r):
        for j in range(c):
            out[i, j] = exponent(float(f[i * rows:(i + 1) * rows, j * COLS:(j + 1) * COLS].max()), low)
    return out.to(y.device)


def spread(e: torch.Tensor, rows: int, shape) -> torch.Tensor:
    """Block exponents to one per element."""
    return e.repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(COLS, 1)[:, :shape[1]]


def widen(q: torch.Tensor, scale: torch.Tensor, rows: int) -> torch.Tensor:
    """What 8-bit values [M, N] with scales per rows x 128 stand for."""
    return torch.ldexp(q.double(), spread(exponents(scale), rows, q.shape))


def round_f8(y: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """e4m3 values of y * 2^-e (y holds at most 24 significant bits, so fp32 holds the product)."""
    return torch.ldexp(y.double(), -e).float().to(F8)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    x = x.double()
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()


def rope(n: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """n [B, S, H, 128], cos / sin [B, S, 128]."""
    c, s = cos.double()[:, :, None], sin.double()[:, :, None]
    return n * c + torch.cat([-n[..., 64:], n[..., :64]], -1) * s


def cache_rows(values: torch.Tensor, scale: torch.Tensor, transposed: bool) -> torch.Tensor:
    """The rows [B, H, T, 128] that a cache's K (or, transposed, V) stands for."""
    v = values.double()
    if transposed:
        v = v.transpose(-1, -2).reshape(*v.shape[:2], -1, 128)
    return torch.ldexp(v, exponents(scale).repeat_interleave(KV_BLOCK, 2)[..., None])


def visible(pos: int, sq: int, T: int, window: int, sinks: int) -> torch.Tensor:
    """[sq, T]: which rows each query token sees."""
    p = pos + torch.arange(sq)[:, None]
    t = torch.arange(T)
    m = t <= p
    if window > 0:
        m &= (t > p - window) | (t < sinks)
    return m


def attention(q, k, v, positions, scale, window=0, sinks=0):
    """(out, sum of weight * |v|, largest |score| error factor): q [B, Hq, Sq, 128],
    k and v [B, Hkv, T, 128] in 64 bits; out [B, Sq, Hq, 128].  The last is
    sum_d |q_d k_d| * scale at its largest over the visible rows, per row."""
    b, hq, sq, _ = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(b, sq, hq, 128, dtype=torch.float64, device=q.device)
    mass, big = torch.zeros_like(out), torch.zeros(b, sq, hq, 1, dtype=torch.float64, device=q.device)
    for i, pos in enumerate(positions):
        n = max(0, min(pos + sq, k.shape[2]))
        if n == 0:
            continue
        m = visible(pos, sq, n, window, sinks).to(q.device)
        empty = ~m.any(-1)
        for h in range(hq):
            kk, vv, qq = k[i, h // g, :n], v[i, h // g, :n], q[i, h].double()
            s = (qq @ kk.T * scale).masked_fill(~m, -math.inf)
            w = torch.softmax(s, -1)
            w[empty] = 0
            # a row that nobody sees has no part, whatever it holds
            seen = torch.where(m.any(0)[:, None], vv, torch.zeros_like(vv))
            out[i, :, h] = _weighted(w, m, seen)
            mass[i, :, h] = w.nan_to_num() @ seen.abs().nan_to_num()
            big[i, :, h] = (qq.abs().nan_to_num() @ kk.abs().nan_to_num().T * scale).masked_fill(~m, 0).amax(-1, keepdim=True)
    return out, mass, big


def _weighted(w, m, v):
    """w @ v where a masked entry has no part even if v is NaN there."""
    bad = v.isnan()
    out = w @ torch.where(bad, torch.zeros_like(v), v)
    return torch.where(m.double() @ bad.double() > 0, torch.full_like(out, math.nan), out)


def attention_bound(out, mass, big):
    """Largest error of a correct kernel: its fp16 result (2^-11) and its
    probabilities' fp16 rounding (2^-11 of each term; below 2^-14 * 2^-9 of the
    largest an absolute 2^-34 of it), fp32 scores (128 products, each within
    2^-24 of its own, the sum's additions likewise: 129 * 2^-24 of sum |q_d k_d|) in
    the exponent, twice (numerator and denominator), and 2^-16 for exp2, its argument's
    rounding and the fp32 sums."""
    return 2.0 ** -11 * (out.abs() + mass) + 2 * (129 * 2.0 ** -24 * big + 2.0 ** -16) * mass + 2.0 ** -24
