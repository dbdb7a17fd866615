"""Plain 64-bit restatements of the cache-maintenance operators (numpy), for tests.

The reference project has no counterpart of these operators; the formulas are those of
include/kvssd_b200.h. Quantization follows the format's rule (src/kvssd/quant.py:28-65): FP32 step
and quotient, round half to even, FP16 scales.
"""

from __future__ import annotations

import numpy as np


def rotate(x, positions, frequencies, interleaved=False, magnitude=1.0):
    """x [T, H, D] -> float64 [T, H, D]."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    half = len(frequencies)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    c, s = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


def quantize(x32, bits, group):
    """FP32 [..., D] -> (codes uint8 [..., D], scales FP16 [..., D / group])."""
    mid = 1 << (bits - 1)
    g = np.asarray(x32, np.float32)
    g = g.reshape(*g.shape[:-1], -1, group)
    step = np.maximum(np.abs(g).max(-1), np.float32(1e-8)) / np.float32(mid - 1)
    codes = np.clip(np.rint(g / step[..., None]), -mid, mid - 1) + mid
    with np.errstate(over="ignore"):
        scales = step.astype(np.float16)
    return codes.astype(np.uint8).reshape(x32.shape), scales


def pack(codes, bits):
    per = 8 // bits
    lanes = codes.reshape(*codes.shape[:-1], -1, per).astype(np.uint32)
    return (lanes << (np.arange(per, dtype=np.uint32) * bits)).sum(-1).astype(np.uint8)


def unpack(packed, bits):
    shifts = np.arange(8 // bits, dtype=np.uint8) * bits
    codes = (packed[..., None] >> shifts) & ((1 << bits) - 1)
    return codes.reshape(*packed.shape[:-1], -1)


def values(codes, scales, bits, group):
    """(code - midpoint) * scale in float64."""
    centred = codes.astype(np.float64) - (1 << (bits - 1))
    return centred * np.repeat(scales.astype(np.float64), group, -1)


def attention_weights(query, packed_k, scales_k, valid, bits, group, sm_scale, lse=None,
                      table=None, visible=None, previous=None):
    """query [T, QH, D] -> (weights [KVH, places], lse [T, QH], bound [KVH, places]) in float64; bound
    is the largest sum |q||k| * sm_scale of a place's scores (for tolerances)."""
    t, qh, d = query.shape
    blocks = np.arange(packed_k.shape[0]) if table is None else np.asarray(table)
    bt, kvh = packed_k.shape[1], packed_k.shape[2]
    k = values(unpack(packed_k[blocks], bits), scales_k[blocks], bits, group).reshape(-1, kvh, d)
    n = k.shape[0]
    seen = (np.arange(bt) < np.clip(valid[blocks], 0, bt)[:, None]).reshape(1, n).repeat(t, 0)
    if visible is not None:
        seen &= np.arange(n) < np.asarray(visible)[:, None]
    q = np.asarray(query, np.float64).reshape(t, kvh, qh // kvh, d)
    k = np.where(seen.any(0)[:, None, None], k, 0.0)  # masked rows may hold anything
    score = np.einsum("thgd,nhd->htgn", q, k) * sm_scale
    bound = np.einsum("thgd,nhd->htgn", np.abs(q), np.abs(k)).max((1, 2)) * abs(sm_scale)
    score = np.where(seen[None, :, None], score, -np.inf)
    if lse is None:
        top = score.max(-1, keepdims=True)
        safe = np.where(np.isinf(top), 0.0, top)
        with np.errstate(divide="ignore"):
            full = np.log(np.exp(score - safe).sum(-1)) + safe[..., 0]
    else:
        full = np.asarray(lse, np.float64).reshape(t, kvh, -1).transpose(1, 0, 2)
    with np.errstate(invalid="ignore"):
        p = np.where((full == -np.inf)[..., None] | ~seen[None, :, None], 0.0, np.exp(score - full[..., None]))
    w = p.sum((1, 2))
    if previous is not None:
        w = w + previous
    return w, full.transpose(1, 0, 2).reshape(t, qh), bound


def evict(weights, positions, n, keep, sink, recent_from, shared):
    """Which place each of the first `keep` places takes its token from: int [KVH, keep]."""
    kvh = weights.shape[0]
    source = np.empty((kvh, keep), np.int64)
    total = weights[:, :n].astype(np.float64).sum(0).astype(np.float32)
    for h in range(kvh):
        w = (total if shared else weights[h, :n]).astype(np.float64)
        pos = positions[0 if shared else h, :n]
        w = np.where(np.isnan(w), -np.inf, w)
        nan = np.isnan(total if shared else weights[h, :n])
        safe = (pos < sink) | (pos >= recent_from)
        # protected first, then numbers by weight, then NaN; all by place within equals
        order = sorted(range(n), key=lambda i: (not safe[i], nan[i], -w[i] if not safe[i] else 0, i))
        kept = np.zeros(n, bool)
        kept[order[:keep]] = True
        source[h] = np.arange(keep)
        source[h, ~kept[:keep]] = keep + np.nonzero(kept[keep:])[0]
    return source
