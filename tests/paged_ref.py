"""Plain 64-bit reference of include/crabml_paged.h and of cc_product_i8, written from their definitions (numpy)."""
import numpy as np

F = np.float64


def f16(x):
    """32-bit numbers as the cache's 16-bit ones: nearest, and what is finite stays finite"""
    x = np.asarray(x, np.float32)
    with np.errstate(over="ignore"):
        h = x.astype(np.float16)
    top = np.float16(65504)
    return np.where(np.isinf(h) & np.isfinite(x), np.where(x > 0, top, -top), h).astype(np.float16)


def turn(x, pos, freq, pairing, offset, mag):
    """x [T, heads, d]; pairing 0: neighbours, 1: halves.  In 64 bits"""
    out = np.array(x, F)
    if freq is None:
        return out
    n = len(freq)
    i = np.arange(n)
    a, b = (offset + 2 * i, offset + 2 * i + 1) if pairing == 0 else (offset + i, offset + i + n)
    ang = np.asarray(pos, F)[:, None, None] * np.asarray(freq, np.float32).astype(F)
    u, v = out[..., a].copy(), out[..., b].copy()
    m = float(np.float32(mag))
    out[..., a] = m * (u * np.cos(ang) - v * np.sin(ang))
    out[..., b] = m * (v * np.cos(ang) + u * np.sin(ang))
    return out


def codes(x):
    """x: one block of one head, 16-bit numbers -> (int8 codes, 32-bit factor)"""
    if not np.isfinite(x).all():
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    x32 = x.astype(F)
    a = np.abs(x32).max()
    if a == 0:
        return np.zeros(x.shape, np.int8), np.float32(0)
    return np.rint(x32 * 127 / a).astype(np.int8), np.float32(a) / np.float32(127)


class Cache:
    """the pages of a layer; arrays as the framework lays them out"""

    def __init__(self, n_pages, G, P, dk, dv, i8, n_slots=0, fill=None):
        r = np.random.default_rng(5 if fill is None else fill)
        self.P, self.G, self.i8 = P, G, i8
        self.a = {}
        for n, d in (("k", dk), ("v", dv)):
            if i8:
                self.a[n] = r.integers(-127, 128, (n_pages, G, P, d)).astype(np.int8)
                self.a[n + "_scale"] = r.uniform(0.5, 1.5, (n_pages, G)).astype(np.float32)
                self.a[n + "_open"] = r.normal(size=(2 * n_slots, G, P, d)).astype(np.float16)
            else:
                self.a[n] = r.normal(size=(n_pages, G, P, d)).astype(np.float16)

    def append(self, table, pos0, slots, rows):
        """rows: {"k": [n, G, dk], "v": ..} 32-bit rows of one sequence (turned)"""
        P = self.P
        for n, x in rows.items():
            x, end = f16(x), pos0 + len(x)
            started = self.a[n + "_open"].copy() if self.i8 else None
            for b in range(pos0 // P, (end - 1) // P + 1 if len(x) else 0):
                lo, hi = max(pos0, b * P), min(end, (b + 1) * P)
                new = x[lo - pos0:hi - pos0].swapaxes(0, 1)
                if not self.i8:
                    self.a[n][table[b], :, lo - b * P:hi - b * P] = new
                    continue
                at = 2 * slots + b % 2
                block = started[at].copy()
                block[:, lo - b * P:hi - b * P] = new
                if hi == (b + 1) * P:
                    for g in range(self.G):
                        self.a[n][table[b], g], self.a[n + "_scale"][table[b], g] = codes(block[g])
                if b >= end // P - 1:
                    self.a[n + "_open"][at, :, lo - b * P:hi - b * P] = new

    def rows(self, name, table, end, slot):
        """the sequence's rows as numbers, [G, end, d]"""
        P, out = self.P, []
        for b in range((end + P - 1) // P):
            if not self.i8:
                x = self.a[name][table[b]].astype(F)
            elif (b + 1) * P <= end:
                x = self.a[name][table[b]].astype(F) * self.a[name + "_scale"][table[b]].astype(F)[:, None, None]
            else:
                x = self.a[name + "_open"][2 * slot + b % 2].astype(F)
            out.append(x)
        d = self.a[name].shape[3]
        return np.concatenate(out, 1)[:, :end] if out else np.zeros((self.G, 0, d))


def attention(q, k, v, pos0, scale, window=0, softcap=0.0, sink=None):
    """q [n, H, dk] at positions pos0 .., k [G, end, dk], v [G, end, dv] -> ([n, H, dv], sums of |weight x value|, largest sum of |q x key| x scale).  Keys that a
    query does not see take no part at all"""
    n, H, _ = q.shape
    G, end, _ = k.shape
    out, mass, reach = np.zeros((n, H, v.shape[2])), np.zeros((n, H, v.shape[2])), np.zeros((n, H))
    for t in range(n):
        i = pos0 + t
        lo = max(0, i - window + 1) if window > 0 else 0
        for h in range(H):
            kk, vv = k[h // (H // G), lo:i + 1], v[h // (H // G), lo:i + 1]
            s = kk @ q[t, h].astype(F) * scale
            reach[t, h] = (np.abs(kk) @ np.abs(q[t, h].astype(F))).max() * abs(scale)
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
            top = s.max() if sink is None else max(s.max(), float(sink[h]))
            p = np.exp(s - top)
            p /= p.sum() + (0 if sink is None else np.exp(float(sink[h]) - top))
            out[t, h], mass[t, h] = p @ vv, p @ np.abs(vv)
    return out, mass, reach


def attention_bound(mass, reach, dk, keys):
    """How far the 32-bit result may be from the exact one.  Scores: h + l leave out 2^-22 of a product, and a step of 16 products adds to a 24-bit sum that may be cut
    off, 2^-23 of the sum of magnitudes for each of the dk / 8 steps (h and l), and a handful of 32-bit operations.  A score's error moves its weight by itself and the
    denominator by as much.  Weights and values likewise: keys / 16 steps, h and l, of at most a slice, a dozen 32-bit operations behind them."""
    score = reach * (2.0 ** -22 + dk / 8 * 2.0 ** -23 + 8 * 2.0 ** -24)
    return mass * (2 * score[..., None] + 2.0 ** -22 + 2 * (min(keys, 2048) / 16 + 1) * 2.0 ** -23 + 16 * 2.0 ** -23) + 1e-30


def product(w, ws, x):
    x = np.asarray(x, np.float32).astype(F)
    a = np.abs(x).max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.where(a > 0, np.rint(x * 127 / a), 0.0)
    return (c @ w.astype(F).T) * (a / 127) * ws.astype(F), c
