"""The 4-bit KV cache restated in numpy: what its codes and scales are for given rows, where they lie, and attention over the values
they stand for, in 64 bits."""
import numpy as np


def rotate(x, heads, pos0, theta):
    """[B, heads * hd], adjacent pairs by (pos0 + b) * theta^(-2m / hd), in 64 bits"""
    B, hd = x.shape[0], x.shape[1] // heads
    if not theta:
        return x.astype(np.float64)
    a = (pos0 + np.arange(B, dtype=np.float64))[:, None] * np.float64(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    y = x.astype(np.float64).reshape(B, heads, hd // 2, 2)
    return np.stack([y[..., 0] * c - y[..., 1] * s, y[..., 0] * s + y[..., 1] * c], -1).reshape(B, heads * hd)


def quantise(x):
    """codes uint8 [..., hd] and scales fp16 [..., hd / 32] of FP32 rows"""
    y = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = np.abs(y).max(-1)
    bad = ~np.isfinite(y).all(-1)
    with np.errstate(all="ignore"):
        s = np.minimum(np.where(bad, np.float32(0), amax) * (np.float32(1) / np.float32(7)), np.float32(8192)).astype(np.float16)
        inv = np.where(s > 0, np.float32(1) / s.astype(np.float32), np.float32(0)).astype(np.float32)
        c = np.clip(np.rint(np.where(bad[..., None], np.float32(0), y) * inv[..., None]), -7, 7)
    s[bad] = np.nan
    return (c + 8).astype(np.uint8).reshape(x.shape), s


def order(hd, key):
    """order[place] = which value of the row lies there"""
    ng, pieces = hd // 32, 4 if key else 8
    per = 32 // pieces
    return np.array([32 * j + per * t + i for t in range(pieces) for j in range(ng) for i in range(per)])


def pack(codes, key):
    c = codes[..., order(codes.shape[-1], key)]
    return c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(b, key):
    hd = b.shape[-1] * 2
    c = np.empty((*b.shape[:-1], hd), np.uint8)
    c[..., 0::2], c[..., 1::2] = b & 15, b >> 4
    out = np.empty_like(c)
    out[..., order(hd, key)] = c
    return out


def values(codes, s):
    return (codes.astype(np.float64) - 8) * np.repeat(s.astype(np.float64), 32, axis=-1)


def random_planes(rng, n_kv, hd, max_rows, rows, loud=3.0):
    """planes of a cache whose first `rows` rows hold quantised values and whose rest holds garbage: random codes, NaN scales"""
    k = rng.integers(0, 256, (n_kv, max_rows, hd // 2), dtype=np.uint8)
    v = rng.integers(0, 256, (n_kv, max_rows, hd // 2), dtype=np.uint8)
    s = np.full((n_kv, max_rows, hd // 16), np.nan, np.float16)
    x = rng.standard_normal((n_kv, rows, hd), dtype=np.float32)
    x[..., ::max(8, hd // 4)] *= loud
    kc, ks = quantise(x)
    vc, vs = quantise(rng.standard_normal((n_kv, rows, hd), dtype=np.float32))
    k[:, :rows], v[:, :rows] = pack(kc, True), pack(vc, False)
    s[:, :rows, :hd // 32], s[:, :rows, hd // 32:] = ks, vs
    return k, v, s


def plane_values(k, v, s):
    ng = s.shape[-1] // 2
    return values(unpack(k, True), s[..., :ng]), values(unpack(v, False), s[..., ng:])


def attention(q, kv_values, n_heads, row0):
    """q [B, n_heads * hd] (64 bits), values of rows 0..row0+B-1 -> out [B, n_heads * hd], weight [n_kv, rows], and a bound on what FP32
    arithmetic may be off by in each of the two.

    A score is a sum of hd products: any order of FP32 additions is off by at most hd half steps of the sum of magnitudes; queries and
    weights split into two pieces of 11 bits lose 2^-22 more of each. With d the largest such error of a score, a weight is off by a factor of at
    most exp(2 d) from the scores, and the sums over rows by the number of additions on a path: at most 64 partial sums of 512
    rows meet, so 600 half steps; exp and the quotient add a few."""
    K, V = kv_values
    n_kv, R, hd = K.shape
    B, group = q.shape[0], n_heads // n_kv
    qh = q.reshape(B, n_heads, hd)
    out, weight = np.zeros((B, n_heads, hd)), np.zeros((n_kv, R))
    tol, wtol = np.zeros((B, n_heads, 1)), np.zeros((n_kv, R))
    seen = np.arange(R)[None, :] <= row0 + np.arange(B)[:, None]
    half = 2.0 ** -24
    for h in range(n_heads):
        n = h // group
        sc = np.where(seen, qh[:, h] @ K[n].T / np.sqrt(hd), -np.inf)
        p = np.exp(sc - sc.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ V[n]
        weight[n] += p.sum(0)
        mag = np.where(seen, np.abs(qh[:, h]) @ np.abs(K[n]).T / np.sqrt(hd), 0.0).max(1)
        rel = np.expm1(2 * (hd + 8) * half * mag) + 640 * half                    # of a weight
        tol[:, h] = (rel[:, None] * (p @ np.abs(V[n]))).max(1, keepdims=True) + 1e-30
        wtol[n] += (rel[:, None] * p).sum(0)
    return out.reshape(B, -1), weight, np.repeat(tol, hd, axis=2).reshape(B, -1), wtol + B * group * half * weight


def choose(weight, keep, sink, recent):
    """rows kept of one head, ascending"""
    rows = len(weight)
    w = weight.astype(np.float64).copy()
    w[np.isnan(w)] = -np.inf
    isnan = np.isnan(weight)
    mid = np.arange(sink, rows - recent)
    best = mid[np.lexsort((mid, isnan[mid], -w[mid]))][:keep - sink - recent]
    return np.sort(np.concatenate([np.arange(sink), best, np.arange(rows - recent, rows)]).astype(np.int32))
