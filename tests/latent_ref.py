"""Latent rows in pages (include/crabml_paged.h) in plain numpy, 64 bits: the append and the attention, from their formulas."""
import numpy as np

F = np.float64


def f16(x):
    """rounded to 16 bits; finite numbers beyond its range become its largest"""
    x = np.asarray(x, F)
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(x), np.clip(x, -65504.0, 65504.0), x).astype(np.float16)


def turn(x, pos, freq, pairing, mag):
    """x [T, ..., columns]: the first 2 P columns of the last axis turned by their token's position"""
    x, P = np.array(x, F), len(freq)
    if not P:
        return x
    a = np.asarray(pos, F)[:, None] * np.asarray(freq, np.float32).astype(F)
    a = a.reshape(a.shape[0], *[1] * (x.ndim - 2), P)
    i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if pairing == 0 else (slice(0, P), slice(P, 2 * P))
    u, v = x[..., i].copy(), x[..., j].copy()
    x[..., i], x[..., j] = mag * (u * np.cos(a) - v * np.sin(a)), mag * (v * np.cos(a) + u * np.sin(a))
    return x


def row(kv, rank, w, eps, pos, freq, pairing, mag):
    """rows of a cache before their rounding"""
    kv = np.asarray(kv, F)
    c = kv[:, :rank] / np.sqrt((kv[:, :rank] ** 2).mean(1, keepdims=True) + eps)
    return np.concatenate([c if w is None else c * np.asarray(w, F), turn(kv[:, rank:], pos, freq, pairing, mag)], 1)


def attention(rows, pos0, q, uk, uv, rank, H, scale, window=0, sink=None):
    """one sequence: rows [L, rank + rest] as cached, q [n, H, dim + rest] of its last n positions -> [n, H, vdim]; NaN where a visible row or the query is not finite.
    Also, for the tolerance: the largest of sum(|w| |v|) over a head's columns' worth, [n, H, vdim]"""
    rows, q = np.asarray(rows, F), np.asarray(q, F)
    n, dim, vdim = q.shape[0], uk.shape[0] // H, uv.shape[0] // H
    U, V = np.asarray(uk, F).reshape(H, dim, rank), np.asarray(uv, F).reshape(H, vdim, rank)
    out, size = np.full((n, H, vdim), np.nan), np.full((n, H, vdim), np.nan)
    wild = ~np.isfinite(rows).all(1)
    clean = np.where(wild[:, None], 0.0, rows)
    for h in range(H):
        k, v = np.concatenate([clean[:, :rank] @ U[h].T, clean[:, rank:]], 1), clean[:, :rank] @ V[h].T
        for t in range(n):
            i = pos0 + t
            lo = max(0, i - window + 1) if window > 0 else 0
            if wild[lo:i + 1].any() or not np.isfinite(q[t, h]).all():
                continue
            z = scale * (k[lo:i + 1] @ q[t, h])
            top = z.max() if sink is None else max(z.max(), float(sink[h]))
            w = np.exp(z - top)
            total = w.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - top))
            out[t, h], size[t, h] = (w / total) @ v[lo:i + 1], (w / total) @ np.abs(v[lo:i + 1])
    return out, size
