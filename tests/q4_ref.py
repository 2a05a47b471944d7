"""Q4_0 blocks and the rotation written from their definitions in 64 bits, for the tests of the 4-bit cache and of the pass that fills
the caches."""
from __future__ import annotations

import numpy as np


def quantize_q4_0(x):
    """float32 (..., n) -> uint8 (..., n/32*18): d = m / -8 with m the first value of largest magnitude of a block, nibble =
    trunc(x * (1/d) + 8.5) at most 15 with 1/d in fp32, byte i = nibble i | nibble 16+i << 4."""
    x = np.ascontiguousarray(x, np.float32)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    m = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
    d = m / np.float32(-8)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d)
        q = np.trunc(b.astype(np.float64) * inv.astype(np.float64) + 8.5)
    q = np.clip(q, 0, 15).astype(np.uint8)
    out = np.concatenate([d.astype(np.float16).view(np.uint8), q[..., :16] | (q[..., 16:] << 4)], -1)
    return out.reshape(x.shape[:-1] + (-1,))


def dequantize_q4_0(rows):
    """uint8 (..., n/32*18) -> float32 (..., n): d * (nibble - 8), exact in fp32."""
    b = np.ascontiguousarray(rows).reshape(rows.shape[:-1] + (-1, 18))
    d = b[..., :2].copy().view(np.float16).astype(np.float32)
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float32) - 8
    return (d * q).reshape(rows.shape[:-1] + (-1,))


def random_q4_0(rng, shape):
    """Rows as quantising N(0,1) values leaves them: (..., n) -> uint8 (..., n/32*18)."""
    return quantize_q4_0(rng.standard_normal(shape).astype(np.float32))


def attention_f64(q, k, v, scale, kv_len=None, q_len=None, causal=False, n_past=0):
    """q (B,H,Tq,hd) rounded to F16 as the operator does; k, v (Bk,Hkv,Lk,hd) values.  -> (B,Tq,H,hd) float64."""
    B, H, Tq, hd = q.shape
    Bk, Hkv, Lk, _ = k.shape
    out = np.zeros((B, Tq, H, hd))
    q = q.astype(np.float16).astype(np.float64)
    for b in range(B):
        n = Lk if kv_len is None else min(max(int(kv_len[b]), 0), Lk)
        live = Tq if q_len is None else min(max(int(q_len[b]), 0), Tq)
        past = n - live if (q_len is not None and kv_len is not None) else n_past
        for h in range(H):
            kk, vv = (x[b // (B // Bk), h // (H // Hkv), :n].astype(np.float64) for x in (k, v))
            s = q[b, h, :live] @ kk.T * scale
            if causal:
                s = np.where(np.arange(n)[None, :] <= past + np.arange(live)[:, None], s, -np.inf)
            if n == 0 or live == 0:
                continue
            m = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(m), m, 0))
            total = p.sum(-1, keepdims=True)
            out[b, :live, h] = p @ vv / np.where(total == 0, 1, total)
    return out


def norm_rope_f64(x, weight, pos, *, n_dims, base=10000.0, scale=1.0, neox=True, eps=1e-6):
    """x (S,H,n,hd), pos (S,) the position of row 0 of each stream.  -> float64 of the same shape."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    i = np.arange(n_dims // 2)
    p = np.asarray(pos, np.float64)[:, None] + np.arange(x.shape[2])
    t = (p[..., None] * float(np.float32(scale)) * float(np.float32(base)) ** (-2.0 * i / max(n_dims, 1)))[:, None]
    c, s = np.cos(t), np.sin(t)
    a, b = (i, i + n_dims // 2) if neox else (2 * i, 2 * i + 1)
    out = y.copy()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    return out
