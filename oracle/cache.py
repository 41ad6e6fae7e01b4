"""Rotary positions, the FP8 key/value cache and the attention over it, in numpy float64 (test infrastructure; see
``oracle/__init__.py``). The operators are not in the reference's scope of this library, so nothing of it restates
them; each function is the operator's definition, and is pinned in tests/test_oracle_cache.py by properties a mistake
would break (lengths kept, angles added, a brute-force softmax, hand-worked places).

quantize restates ``quant.per_group_quant_fp8``'s fp32 steps with one group a vector, plus the rule for vectors that
hold a NaN or an infinity: zero codes under a NaN scale.
"""
from __future__ import annotations

import numpy as np

from .formats import f32_to_e4m3fn
from .quant import AMAX_FLOOR, INV448

E4M3 = np.array([(1 - 2 * (c >> 7)) * (np.nan if c & 127 == 127 else
                                       (c & 7) * 2.0**-9 if c & 0x78 == 0 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                 for c in range(256)])


def rotate(x, positions, frequencies, interleaved=False, magnitude=1.0):
    """x [tokens, heads, head_dim] with the first 2 * len(frequencies) values of every head turned."""
    x = np.array(x, dtype=np.float64)
    r = 2 * len(frequencies)
    angle = np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(frequencies, dtype=np.float64)
    cos, sin = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., lo].copy(), x[..., hi].copy()
    x[..., lo], x[..., hi] = a * cos - b * sin, b * cos + a * sin
    return x


def quantize(x):
    """fp32 vectors [..., head_dim] -> (e4m3fn codes uint8, fp32 scales [...])."""
    x = np.asarray(x, dtype=np.float32)
    bad = ~np.isfinite(x).all(-1)
    y = np.where(bad[..., None], np.float32(0), x)
    scale = (np.maximum(np.abs(y).max(-1), AMAX_FLOOR) * INV448).astype(np.float32)
    with np.errstate(over="ignore"):
        inv = (np.float32(1) / scale).astype(np.float32)
        code = f32_to_e4m3fn(np.clip((y * inv[..., None]).astype(np.float32), np.float32(-448), np.float32(448)))
    return np.where(bad[..., None], np.uint8(0), code), np.where(bad, np.float32(np.nan), scale)


def gather(codes, scales, block_table, seq, length):
    """Values [length, kv_heads, head_dim] of a sequence's first positions, and which of them the cache has."""
    pages, heads, page, dim = codes.shape
    out = np.zeros((length, heads, dim))
    there = np.zeros(length, dtype=bool)
    for p in range(length):
        col = p // page
        if col < block_table.shape[1] and 0 <= block_table[seq, col] < pages:
            at = block_table[seq, col]
            out[p] = E4M3[codes[at, :, p % page]] * scales[at, :, p % page].astype(np.float64)[:, None]
            there[p] = True
    return out, there


def attention(q, k_codes, v_codes, k_scales, v_scales, block_table, lens, starts, mask, scale):
    """(out, lse, bound): bound[token, head, d] is the softmax-weighted sum of |v| (what a relative error of the
    weights can do), and bound_score[token, head] the largest scale * sum |q_d k_d|."""
    tokens, heads, dim = q.shape
    kv = k_codes.shape[1]
    out, lse = np.zeros((tokens, heads, dim)), np.full((tokens, heads), -np.inf)
    weighed, score_size = np.zeros((tokens, heads, dim)), np.zeros((tokens, heads))
    q = np.asarray(q, dtype=np.float64)
    for b in range(len(lens)):
        lo, hi = int(starts[b]), int(starts[b + 1])
        n = min(int(lens[b]), block_table.shape[1] * k_codes.shape[2])
        k, there = gather(k_codes, k_scales, block_table, b, n)
        v, _ = gather(v_codes, v_scales, block_table, b, n)
        ctx = n - (hi - lo)
        for i in range(lo, hi):
            sees = there.copy()
            for p in range(max(ctx, 0), n):
                j = p - ctx
                sees[p] &= bool(j < mask.shape[1] and mask[i, j]) if mask is not None else j <= i - lo
            if not sees.any():
                continue
            for h in range(heads):
                kk, vv = k[sees, h * kv // heads], v[sees, h * kv // heads]
                s = kk @ q[i, h] * scale
                top = s.max()
                w = np.exp(s - top)
                out[i, h] = w @ vv / w.sum()
                lse[i, h] = top + np.log(w.sum())
                weighed[i, h] = w @ np.abs(vv) / w.sum()
                score_size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, lse, weighed, score_size
