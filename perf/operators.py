"""The 8-bit serving operators as measurable cases: row quantisers (add + RMSNorm,
SiLU * up, plain), the block-scaled product, the 8-bit KV cache (written and read
back) and the attention over it.

Values are e4m3, scales powers of two (E8M0): a block's exponent e is the least
integer with amax <= 448 * 2^e.  ``own = False`` computes the operators from
elementary torch operations in fp32; ``own = True`` calls the framework's.
Sizes are the Qwen3-VL-2B text decoder's: hidden 2048, intermediate 6144, 8 kv
heads of 128, qkv rows 4096, vocabulary 151936.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "aicasgc-2026_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

HIDDEN, INTER, VOCAB, QKV, D, EPS = 2048, 6144, 151936, 4096, 128, 1e-6
BLOCK = 64          # cache rows per scale
KV_LOW = -32        # least exponent of a cache block
LOW = -126          # least exponent of an activation or weight block
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------ the cases

def listed() -> list:
    return [
        # One decode token's residual add + RMSNorm: the smallest call, latency only.
        {"name": "norm_1", "path": "rows", "mode": "norm", "rows": 1, "cols": HIDDEN},
        # The same for every row of a long prompt.
        {"name": "norm_4001", "path": "rows", "mode": "norm", "rows": 4001, "cols": HIDDEN},
        # One decode token's qkv projection.
        {"name": "qkv_1", "path": "matmul", "m": 1, "n": QKV, "k": HIDDEN, "out": "f16"},
        # The tied lm_head over a batch of 8 sequences, fp32 logits: the largest weight.
        {"name": "lm_head_8", "path": "matmul", "m": 8, "n": VOCAB, "k": HIDDEN, "out": "f32"},
        # gate_up of a long prompt: the largest product.
        {"name": "gate_up_4001", "path": "matmul", "m": 4001, "n": 2 * INTER, "k": HIDDEN, "out": "f16"},
        # One token of each of 8 ragged sequences appended to the cache.
        {"name": "append_8", "path": "write", "batch": 8, "tokens": 1, "low": 700, "high": 4095, "groups": 2,
         "kv_heads": 8},
        # A long prompt written at once into a fresh cache.
        {"name": "write_4001", "path": "write", "batch": 1, "tokens": 4001, "low": 0, "high": 0, "groups": 2,
         "kv_heads": 8},
        # A long document's cache handed back to an fp16 path.
        {"name": "read_30001", "path": "read", "batch": 1, "rows": 30001, "kv_heads": 8},
        # Decode attention behind a 1024-position prompt.
        {"name": "attend_1029", "path": "attend", "batch": 1, "queries": 1, "low": 1029, "high": 1029, "capacity": 1344,
         "groups": 2, "kv_heads": 8, "window": 0, "sinks": 0},
        # Decode attention late in a long document.
        {"name": "attend_30001", "path": "attend", "batch": 1, "queries": 1, "low": 30001, "high": 30001,
         "capacity": 32768, "groups": 2, "kv_heads": 8, "window": 0, "sinks": 0},
        # One decode token of each of 8 ragged sequences.
        {"name": "attend_batch8", "path": "attend", "batch": 8, "queries": 1, "low": 2048, "high": 4096, "capacity": 4160,
         "groups": 2, "kv_heads": 8, "window": 0, "sinks": 0},
        # A 929-token question about a picture of 48 x 64 positions: a chunk behind a filled cache.
        {"name": "attend_chunk", "path": "attend", "batch": 1, "queries": 929, "low": 4001, "high": 4001, "capacity": 4032,
         "groups": 2, "kv_heads": 8, "window": 0, "sinks": 0},
    ]


def _log(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    path = rng.choice(["rows", "matmul", "matmul", "write", "read", "attend", "attend", "attend"])
    if path == "rows":
        # plain rows are quantised activations, weight a matrix in 128 x 128 blocks at load
        return {"path": path, "mode": rng.choice(["norm", "silu", "plain", "weight"]), "rows": _log(rng, 1, 4001),
                "cols": rng.choice([HIDDEN, INTER, _log(rng, 64, 4096)])}
    if path == "matmul":
        m = _log(rng, 1, 4001)
        k = rng.choice([HIDDEN, INTER, 16 * _log(rng, 4, 256)])
        n = min(_log(rng, 64, 20000), 4001 * 2 * INTER * HIDDEN // (m * k))
        return {"path": path, "m": m, "n": n, "k": k, "out": rng.choice(["f16", "f32"])}
    kv_heads = rng.choice([2, 4, 8])
    if path == "write":
        batch = rng.randrange(1, 9)
        tokens = rng.choice([1, rng.randrange(2, 17), _log(rng, 16, 4001 // batch)])
        low = rng.randrange(0, 2000)
        return {"path": path, "batch": batch, "tokens": tokens, "low": low, "high": low + rng.randrange(0, 2000),
                "groups": rng.choice([1, 2, 4]), "kv_heads": kv_heads}
    if path == "read":
        batch = rng.randrange(1, 9)
        return {"path": path, "batch": batch, "rows": _log(rng, 1, 30001 // batch), "kv_heads": kv_heads}
    groups = rng.choice([1, 2, 4])
    batch = rng.randrange(1, 9)
    high = _log(rng, 1, 32768 // batch)
    queries = rng.choice([1, 1, rng.randrange(2, 17), _log(rng, 16, 929)])
    queries = max(1, min(queries, high, 60_000_000 // (batch * groups * kv_heads * (high + 128))))
    low = max(queries, high // rng.randrange(1, 9))
    window = 0 if rng.random() < 0.5 else _log(rng, 16, 4096)
    return {"path": path, "batch": batch, "queries": queries, "low": low, "high": high,
            "capacity": BLOCK * ((high + BLOCK - 1) // BLOCK + rng.randrange(0, 5)), "groups": groups,
            "kv_heads": kv_heads, "window": window, "sinks": rng.randrange(0, 130) if window else 0}


# ------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std: float = 1.0, mean: float = 0.0) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.float16, device="cuda").normal_(mean, std, generator=g)


def _lengths(case: dict, seed: int) -> list:
    """One length per sequence: `high` first, the others spread over [low, high]."""
    r = torch.Generator().manual_seed(int(seed))
    more = torch.randint(case["low"], case["high"] + 1, (case["batch"] - 1,), generator=r).tolist()
    return [case["high"]] + more


def _cache(g, batch: int, kv_heads: int, capacity: int) -> dict:
    """A cache whose every row holds something: behind a sequence's end what an
    earlier one left.  K rows are normalised and rotated (unit variance), V rows'
    size differs from block to block."""
    nb = capacity // BLOCK
    k = _randn(g, batch, kv_heads, nb, BLOCK, D).float()
    v = _randn(g, batch, kv_heads, nb, D, BLOCK).float() * torch.exp2(_randn(g, batch, kv_heads, nb, 1, 1).float())
    out = {}
    for name, t in (("k", k), ("v", v)):
        e = _exponent(t.abs().amax((-1, -2)), KV_LOW)
        out[name] = (t * _pow2(-e)[..., None, None]).to(F8)
        out[name + "_scale"] = _byte(e)
    out["k"] = out["k"].view(batch, kv_heads, capacity, D)
    return out


def _rope(positions: torch.Tensor):
    f = positions[..., None].double() * 5e6 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    e = torch.cat([f, f], -1)
    return e.cos().half(), e.sin().half()


def prepare(case: dict, seed: int) -> dict:
    g, path = _gen(seed), case["path"]
    st = {"case": case}
    if path == "rows":
        r, c = case["rows"], case["cols"]
        if case["mode"] == "norm":
            st.update(residual=_randn(g, r, c), x=_randn(g, r, c), weight=_randn(g, c, std=0.02, mean=1.0))
        elif case["mode"] == "silu":
            st["gate_up"] = _randn(g, r, 2 * c)     # one product's output, gate and up side by side
        else:
            st["x"] = _randn(g, r, c, std=0.02 if case["mode"] == "weight" else 1.0)
    elif path == "matmul":
        st["x"], st["x_scale"] = _quantize(_randn(g, case["m"], case["k"]).float(), 1)
        st["w"], st["w_scale"] = _quantize(_randn(g, case["n"], case["k"], std=0.02).float(), 128)
    elif path == "write":
        b, s, h = case["batch"], case["tokens"], case["kv_heads"]
        pos = torch.tensor(_lengths(case, seed), dtype=torch.int64, device="cuda")
        capacity = BLOCK * ((case["high"] + s + BLOCK - 1) // BLOCK + 1)
        st.update(_cache(g, b, h, capacity), pos=pos,
                  q=_randn(g, b, s, h * case["groups"], D), knew=_randn(g, b, s, h, D), vnew=_randn(g, b, s, h, D),
                  q_weight=_randn(g, D, std=0.02, mean=1.0), k_weight=_randn(g, D, std=0.02, mean=1.0))
        st["cos"], st["sin"] = _rope(pos[:, None] + torch.arange(s, device="cuda"))
    elif path == "read":
        st.update(_cache(g, case["batch"], case["kv_heads"], BLOCK * ((case["rows"] + BLOCK - 1) // BLOCK)))
    else:
        b, s = case["batch"], case["queries"]
        lens = torch.tensor(_lengths(case, seed), dtype=torch.int64, device="cuda")
        st.update(_cache(g, b, case["kv_heads"], case["capacity"]), pos=lens - s, ws={},
                  q=_randn(g, b, s, case["kv_heads"] * case["groups"], D).transpose(1, 2))
    return st


# ------------------------------------------------------------------ one pass

def run(st: dict):
    case = st["case"]
    return (_run_own if own else _run_plain)(st, case, case["path"])


def _run_own(st: dict, case: dict, path: str):
    import cuda_decode_attention as attention
    import cuda_decode_gemv as gemv
    import cuda_decode_small_ops as small

    if path == "rows":
        mode = case["mode"]
        if mode == "norm":
            return small.fused_add_rms_norm_fp8(st["residual"], st["x"], st["weight"], EPS)
        if mode == "silu":
            gate, up = st["gate_up"].chunk(2, -1)
            return small.fused_silu_mul_fp8(gate, up)
        return small.quantize_fp8(st["x"], block_rows=128 if mode == "weight" else 1)
    if path == "matmul":
        return gemv.block_matmul_fp8(st["x"], st["x_scale"], st["w"], st["w_scale"],
                                     out_dtype=torch.float16 if case["out"] == "f16" else torch.float32)
    cache = small.KVCacheFP8(st["k"], st["v"], st["k_scale"], st["v_scale"])
    if path == "write":
        q = small.fused_q_rope_kv_cache_update_fp8(st["q"], st["knew"], st["vnew"], st["q_weight"], st["k_weight"], EPS,
                                                   st["cos"], st["sin"], cache, st["pos"])
        return [q, *cache]
    if path == "read":
        return small.read_kv_cache_fp8(cache, case["rows"])
    return attention.attn_fp8_kv_cache(st["q"], cache, D ** -0.5, st["pos"], window=case["window"], sinks=case["sinks"],
                                       workspace=st["ws"])


# ------------------------------------------------------------------ the plain form

def _exponent(amax: torch.Tensor, low: int) -> torch.Tensor:
    """The least integer e >= low with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 8 - (m <= 0.875).int(), torch.full_like(x, low)).clamp_min(low)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.int() + 127) << 23).view(torch.float32)


def _byte(e: torch.Tensor) -> torch.Tensor:
    return (e + 127).to(torch.uint8).view(E8)


def _unbyte(s: torch.Tensor) -> torch.Tensor:
    return s.view(torch.uint8).int() - 127


def _amax(y: torch.Tensor, dims) -> torch.Tensor:
    return torch.where(y.isfinite(), y.abs(), torch.zeros_like(y)).amax(dims)


def _quantize(y: torch.Tensor, block_rows: int):
    """e4m3 values and E8M0 scales of y [rows, cols] in blocks of block_rows x 128."""
    r, c = y.shape
    rb, cb = -(-r // block_rows), -(-c // 128)
    t = torch.nn.functional.pad(y, (0, cb * 128 - c, 0, rb * block_rows - r)).view(rb, block_rows, cb, 128)
    e = _exponent(_amax(t, (1, 3)), LOW)
    q = (t * _pow2(-e)[:, None, :, None]).to(F8).view(rb * block_rows, cb * 128)[:r, :c]
    return q.contiguous(), _byte(e)


def _widen(q: torch.Tensor, scale: torch.Tensor, block_rows: int) -> torch.Tensor:
    s = _pow2(_unbyte(scale))
    s = s.repeat_interleave(block_rows, 0)[:q.shape[0]] if block_rows > 1 else s
    return q.float() * s.repeat_interleave(128, 1)[:, :q.shape[1]]


def _head_norm_rope(x, w, cos, sin):
    y = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + EPS) * w.float()
    c, s = cos.float()[:, :, None], sin.float()[:, :, None]
    return y * c + torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1) * s


def _write_blocks(cache, scale, new, pos, tokens):
    """`new` [B, H, S, D] quantised into the blocks of `cache` [B, H, nb, 64, D] (a view)."""
    b = new.shape[0]
    first = pos // BLOCK
    rows = torch.arange((tokens + 126) // BLOCK * BLOCK, device="cuda") + first[:, None] * BLOCK     # [B, n]
    src = rows - pos[:, None]
    fresh = ((src >= 0) & (src < tokens)).view(b, 1, -1, BLOCK, 1)
    index = src.clamp(0, tokens - 1)[:, None, :, None].expand(-1, new.shape[1], -1, D)
    t = new.gather(2, index).view(b, new.shape[1], -1, BLOCK, D) * fresh
    blocks = rows.view(b, -1, BLOCK)[:, :, 0] // BLOCK     # within the capacity: it has a block to spare
    at = (torch.arange(b, device="cuda")[:, None], slice(None), blocks)
    old = cache.view(torch.uint8)[at].transpose(1, 2)
    e_old = _unbyte(scale)[at].transpose(1, 2)
    earlier = (rows < pos[:, None]).view(b, 1, -1, BLOCK, 1)
    e_new = _exponent(_amax(t, (-1, -2)), KV_LOW)
    e = torch.where(earlier.any(3).squeeze(-1), torch.maximum(e_new, e_old), e_new)
    e = torch.where(fresh.any(3).squeeze(-1), e, e_old)
    kept = (old.view(F8).float() * _pow2(e_old - e)[..., None, None]).to(F8).view(torch.uint8)
    put = (t * _pow2(-e)[..., None, None]).to(F8).view(torch.uint8)
    cache.view(torch.uint8)[at] = torch.where(fresh, put, torch.where(earlier, kept, old)).transpose(1, 2)
    scale.view(torch.uint8)[at] = (e + 127).to(torch.uint8).transpose(1, 2)


def _run_plain(st: dict, case: dict, path: str):
    if path == "rows":
        if case["mode"] == "norm":
            y = st["residual"].float() + st["x"].float()
            n = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * st["weight"].float()
            return y.half(), *_quantize(n, 1)
        if case["mode"] == "silu":
            gate, up = st["gate_up"].float().chunk(2, -1)
            return _quantize(gate / (1 + torch.exp(-gate)) * up, 1)
        return _quantize(st["x"].float(), 128 if case["mode"] == "weight" else 1)
    if path == "matmul":
        y = _widen(st["x"], st["x_scale"], 1) @ _widen(st["w"], st["w_scale"], 128).T
        return y.half() if case["out"] == "f16" else y
    b, h = st["k"].shape[:2]
    kb, vb = st["k"].view(b, h, -1, BLOCK, D), st["v"].transpose(-1, -2)
    if path == "write":
        k = _head_norm_rope(st["knew"], st["k_weight"], st["cos"], st["sin"]).transpose(1, 2)
        _write_blocks(kb, st["k_scale"], k, st["pos"], case["tokens"])
        _write_blocks(vb, st["v_scale"], st["vnew"].float().transpose(1, 2), st["pos"], case["tokens"])
        q = _head_norm_rope(st["q"], st["q_weight"], st["cos"], st["sin"]).half()
        return [q, st["k"], st["v"], st["k_scale"], st["v_scale"]]
    k = (kb.float() * _pow2(_unbyte(st["k_scale"]))[..., None, None]).view(b, h, -1, D)
    v = (vb.float() * _pow2(_unbyte(st["v_scale"]))[..., None, None]).reshape(b, h, -1, D)
    if path == "read":
        return k[:, :, :case["rows"]].half(), v[:, :, :case["rows"]].half()
    n, groups = case["queries"], case["groups"]
    p = st["pos"][:, None] + torch.arange(n, device="cuda")
    t = torch.arange(k.shape[2], device="cuda")
    seen = t <= p[..., None]
    if case["window"]:
        seen &= (t > p[..., None] - case["window"]) | (t < case["sinks"])
    q = st["q"].float().reshape(b, h, groups * n, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, h, groups, n, -1) * D ** -0.5
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).view(b, h, groups * n, -1)
    return torch.matmul(w, v).view(b, h * groups, n, D).transpose(1, 2).contiguous().half()


# ------------------------------------------------------------------ bounds

def _visible(case: dict, length: int):
    """(cache rows that some query sees, query-row pairs) of one sequence."""
    n, w, sinks = case["queries"], case["window"], case["sinks"]
    pairs = union = 0
    low = None
    for p in range(length - n, length):
        first = max(0, p - w + 1) if w else 0
        low = first if low is None else low
        pairs += p + 1 - first + min(sinks if w else 0, first)
    union = length - low + min(sinks if w else 0, low)
    return union, pairs


def work(case: dict) -> dict:
    """Each input read and each output written once; two flops per multiply-add."""
    path = case["path"]
    if path == "rows":
        r, c = case["rows"], case["cols"]
        per = {"norm": 6 + 1, "silu": 4 + 1, "plain": 2 + 1, "weight": 2 + 1}[case["mode"]]
        return {"bytes": r * c * per + r * c / 128, "flops": 8 * r * c}
    if path == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + m * k + m * n * (2 if case["out"] == "f16" else 4), "flops": 2 * m * n * k}
    h = case["kv_heads"]
    if path == "write":
        rows = case["batch"] * case["tokens"]
        return {"bytes": rows * D * (4 * h * case["groups"] + 2 * h * (2 + 1) + 4), "flops": 8 * rows * D * h * 4}
    if path == "read":
        return {"bytes": case["batch"] * h * case["rows"] * D * 6, "flops": 2 * case["batch"] * h * case["rows"] * D}
    # the ragged lengths follow the seed; their mean here
    seen = [_visible(case, n) for n in [case["high"]] + [(case["low"] + case["high"]) // 2] * (case["batch"] - 1)]
    heads = h * case["groups"]
    return {"bytes": sum(u for u, _ in seen) * 2 * D * h + case["batch"] * case["queries"] * heads * D * 4,
            "flops": 4 * D * heads * sum(p for _, p in seen)}


# ------------------------------------------------------------------ the same in 64 bits

def _step(amax: torch.Tensor, low: int) -> torch.Tensor:
    """2^e of blocks in 64 bits: e = ceil(log2(amax / 448)), at least `low`."""
    e = torch.log2(amax.clamp_min(1e-300) / 448).ceil().clamp_min(low)
    e = torch.where(amax > 448 * 2.0 ** e, e + 1, torch.where((amax <= 224 * 2.0 ** e) & (e > low), e - 1, e))
    return 2.0 ** e


def _blocked64(y: torch.Tensor, rows: int):
    """y over its blocks' scales, not rounded, and the scales."""
    out = torch.empty_like(y)
    scale = torch.empty(-(-y.shape[0] // rows), -(-y.shape[1] // 128), dtype=torch.float64, device=y.device)
    for j in range(scale.shape[1]):
        part = y[:, 128 * j:128 * j + 128].abs().amax(1)
        part = torch.nn.functional.pad(part, (0, -len(part) % rows)).view(-1, rows).amax(1)
        scale[:, j] = _step(part, LOW)
        out[:, 128 * j:128 * j + 128] = y[:, 128 * j:128 * j + 128] / scale[:, j].repeat_interleave(rows)[:len(y), None]
    return out, scale


def _rotate64(x, w, cos, sin):
    x = x.double()
    n = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
    a, b = n[..., :D // 2], n[..., D // 2:]
    c, s = cos.double()[:, :, None, :D // 2], sin.double()[:, :, None, :D // 2]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _rows64(st, name):
    """The cache's rows [B, H, T, D] in 64 bits."""
    scale = 2.0 ** (st[name + "_scale"].view(torch.uint8).double() - 127)
    t = st[name].double()
    t = t if name == "k" else t.permute(0, 1, 2, 4, 3).reshape(*t.shape[:2], -1, D)
    return t * scale.repeat_interleave(BLOCK, 2)[..., None]


def _append64(st, name, new, pos):
    """The stored values (not rounded) and scales with `new` [B, S, H, D] written from pos[b]."""
    scale = 2.0 ** (st[name + "_scale"].view(torch.uint8).double() - 127)
    rows = _rows64(st, name)
    held = rows / scale.repeat_interleave(BLOCK, 2)[..., None]
    for b, p in enumerate(pos):
        end = p + new.shape[1]
        for blk in range(p // BLOCK, (end - 1) // BLOCK + 1):
            lo, hi = max(p, blk * BLOCK), min(end, blk * BLOCK + BLOCK)
            part = new[b, lo - p:hi - p].transpose(0, 1)
            s = _step(part.abs().amax((1, 2)), KV_LOW)
            if lo > blk * BLOCK:
                s = torch.maximum(s, scale[b, :, blk])
                held[b, :, blk * BLOCK:lo] = rows[b, :, blk * BLOCK:lo] / s[:, None, None]
            held[b, :, lo:hi] = part / s[:, None, None]
            scale[b, :, blk] = s
    if name == "v":
        held = held.view(*held.shape[:2], -1, BLOCK, D).transpose(-1, -2).contiguous()
    return held, scale


def exact(case: dict, seed: int):
    st, path = prepare(case, seed), case["path"]
    if path == "rows":
        if case["mode"] == "norm":
            y = st["residual"].double() + st["x"].double()
            n = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * st["weight"].double()
            return y, *_blocked64(n, 1)
        if case["mode"] == "silu":
            t = st["gate_up"].double()
            c = case["cols"]
            return _blocked64(t[:, :c] * torch.sigmoid(t[:, :c]) * t[:, c:], 1)
        return _blocked64(st["x"].double(), 128 if case["mode"] == "weight" else 1)
    if path == "matmul":
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for j in range(st["x_scale"].shape[1]):
            k = slice(128 * j, 128 * j + 128)
            sx = 2.0 ** (st["x_scale"][:, j].view(torch.uint8).double() - 127)
            sw = 2.0 ** (st["w_scale"][:, j].view(torch.uint8).double() - 127)
            w = st["w"][:, k].double() * sw.repeat_interleave(128)[:case["n"], None]
            y += (st["x"][:, k].double() * sx[:, None]) @ w.T
        return y
    if path == "write":
        pos = st["pos"].tolist()
        k = _append64(st, "k", _rotate64(st["knew"], st["k_weight"], st["cos"], st["sin"]), pos)
        v = _append64(st, "v", st["vnew"].double(), pos)
        return [_rotate64(st["q"], st["q_weight"], st["cos"], st["sin"]), k[0], v[0], k[1], v[1]]
    k, v = _rows64(st, "k"), _rows64(st, "v")
    if path == "read":
        return k[:, :, :case["rows"]], v[:, :, :case["rows"]]
    out = torch.empty(case["batch"], case["queries"], st["q"].shape[1], D, dtype=torch.float64, device="cuda")
    for b, p in enumerate(st["pos"].tolist()):
        at = p + torch.arange(case["queries"], device="cuda")[:, None]
        t = torch.arange(p + case["queries"], device="cuda")
        gone = t > at
        if case["window"]:
            gone |= (t <= at - case["window"]) & (t >= case["sinks"])
        for head in range(st["q"].shape[1]):
            kv = head // case["groups"]
            s = st["q"][b, head].double() @ k[b, kv, :len(t)].T / math.sqrt(D)
            out[b, :, head] = torch.softmax(s.masked_fill(gone, -math.inf), -1) @ v[b, kv, :len(t)]
    return out
