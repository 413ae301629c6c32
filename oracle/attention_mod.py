"""Oracle for paged attention with score modifications and for the rotary
append (test infrastructure, never shipped).

The reference has neither (its RoPE is tests/test_fusion.py:30-38's half-split
rotation, and there is no attention kernel), so these float64 restatements of
the definitions in include/krt.h are unpinned by reference vectors; the CPU
tests check them against torch's own attention and complex arithmetic.
"""
import numpy as np

from .attention import gather_kv


def visible_range(pos, length, window=0, kv_start=0, prefix=0):
    """Half-open range of positions that the query at `pos` sees."""
    lo = max(0, kv_start, pos - window + 1 if window > 0 else 0)
    return lo, min(length, max(pos + 1, prefix))


def attention_row(q, k, v, pos, lo, hi, scale, softcap=0.0, slope=0.0):
    """One query row and head over keys lo .. hi - 1 of k, v [n, 128] (float64):
    (out [128], lse, weight of |v| [128], error scale of the scores)."""
    if lo >= hi:
        return np.zeros(v.shape[1]), -np.inf, np.zeros(v.shape[1]), 0.0
    kk, vv = k[lo:hi], v[lo:hi]
    s = (kk @ q) * scale
    x = softcap * np.tanh(s / softcap) if softcap > 0 else s
    x = x - slope * np.abs(pos - np.arange(lo, hi))
    top = x.max()
    e = np.exp(x - top)
    w = e / e.sum()
    # fp32 error of a score: 128 products and sums, and a few roundings of x itself
    fuzz = 2.0 ** -24 * (130 * scale * (np.abs(kk) @ np.abs(q)).max() + 4 * np.abs(x).max() + 8 * softcap)
    return w @ vv, top + np.log(e.sum()), w @ np.abs(vv), fuzz


def paged_attention_mod(q, pool, table, rows, n_heads, n_kv_heads, tokens_per_block, softcap=0.0, window=0,
                        slopes=None, scale=None):
    """rows: per query row (sequence, position, length, kv_start, prefix) or
    None (left out).  q [T, n_heads, 128], pool [blocks, tokens, 2, n_kv_heads,
    128] (float).  Returns (out [T, H, 128], lse [T, H], tol_out, tol_lse)."""
    scale = 1.0 / np.sqrt(q.shape[-1]) if scale is None else scale
    T, group = len(rows), n_heads // n_kv_heads
    out, lse = np.zeros((T, n_heads, 128)), np.full((T, n_heads), -np.inf)
    tol_out, tol_lse = np.zeros_like(out), np.zeros((T, n_heads))
    cache = {}
    for t, row in enumerate(rows):
        if row is None:
            continue
        s, pos, length, start, prefix = row
        if (s, length) not in cache:
            k, v = gather_kv(pool, table[s], length, tokens_per_block)
            cache[s, length] = k.astype(np.float64), v.astype(np.float64)
        k, v = cache[s, length]
        lo, hi = visible_range(pos, length, window, start, prefix)
        for h in range(n_heads):
            o, z, a, fuzz = attention_row(q[t, h].astype(np.float64), k[:, h // group], v[:, h // group], pos, lo, hi,
                                          scale, softcap, 0.0 if slopes is None else float(slopes[h]))
            out[t, h], lse[t, h] = o, z
            # weights to bf16 (2^-8 each), their fp32 errors on both sides of the quotient, one bf16 rounding
            rel = 2.0 ** -8 + 2 * (fuzz + 2.0 ** -20 + (hi - lo) * 2.0 ** -24)
            tol_out[t, h] = rel * a + 2.0 ** -8 * np.abs(o) + 1e-30
            tol_lse[t, h] = fuzz + 2.0 ** -20 + (hi - lo) * 2.0 ** -24 + 2.0 ** -22 * abs(z) if hi > lo else 0.0
    return out, lse, tol_out, tol_lse


def rope(x, positions, inv_freq, rotary_dim, interleaved, factor=1.0):
    """x [T, heads, 128] float64, rotated."""
    x = np.array(x, dtype=np.float64)
    turn = factor * np.exp(1j * np.outer(positions, inv_freq))[:, None, :]
    a = slice(0, rotary_dim, 2) if interleaved else slice(0, rotary_dim // 2)
    b = slice(1, rotary_dim, 2) if interleaved else slice(rotary_dim // 2, rotary_dim)
    z = (x[..., a] + 1j * x[..., b]) * turn
    x[..., a], x[..., b] = z.real, z.imag
    return x
