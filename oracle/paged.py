"""CPU oracle of batched attention serving (paged KV caches, packed prompts) -- TEST INFRASTRUCTURE ONLY.

The definitions of include/nmi_fp8_linear.h in float64, one sequence, token and head after another.  No
counterpart in the reference (one sequence, contiguous caches); ``decode`` and ``prefill`` are pinned
against oracle.attention (itself pinned against torch's attention) in tests/test_paged_cpu.py, and
``rotate`` against complex multiplication.
"""
from __future__ import annotations

import numpy as np

HEAD = 128
E4M3_MAX = 448.0


def rotate(x: np.ndarray, pos: np.ndarray, inv_freq: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [T, heads, 128] float64 rotated by position: pair i by pos * inv_freq[i]."""
    out = np.array(x, np.float64)
    r = 2 * len(inv_freq)
    for i, f in enumerate(np.asarray(inv_freq, np.float64)):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        c, s = np.cos(pos * f)[:, None], np.sin(pos * f)[:, None]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return out


def partner_sum(x: np.ndarray, rotary: int, interleaved: bool) -> np.ndarray:
    """|x| + |its partner in the rotation| of every element (dims that are not rotated: 0)."""
    out = np.zeros_like(x, dtype=np.float64)
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        out[..., a] = out[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return out


def positions(T: int, start, cu=None):
    """[(row, sequence, position)] of the rows that belong to a sequence in use."""
    if cu is None:
        return [(t, t, int(start[t])) for t in range(T) if start[t] >= 0]
    return [(t, b, int(start[b]) + t - int(cu[b])) for b in range(len(start)) if start[b] >= 0
            for t in range(int(cu[b]), int(cu[b + 1]))]


def gather(pages: np.ndarray, table_row, n: int) -> np.ndarray:
    """The first n positions of a sequence: pages [n_pages, n_kv, page_size, 128] -> [n_kv, n, 128]."""
    page = pages.shape[2]
    if n == 0:
        return pages[:1, :, :0].transpose(1, 0, 2, 3).reshape(pages.shape[1], 0, HEAD)
    got = [pages[table_row[i]] for i in range(-(-n // page))]
    return np.concatenate(got, axis=1)[:, :n]


def decode(q: np.ndarray, k_pages: np.ndarray, v_pages: np.ndarray, table, lens, scale=HEAD ** -0.5) -> np.ndarray:
    """q [B, H, 128]; pages float64 (scales applied).  o [B, H, 128]; a length of 0 gives zeros."""
    B, H, _ = q.shape
    n_kv = k_pages.shape[1]
    out = np.zeros((B, H, HEAD))
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        K, V = gather(k_pages, table[b], n), gather(v_pages, table[b], n)
        for h in range(H):
            e = scale * (K[h * n_kv // H] @ q[b, h])
            w = np.exp(e - e.max())
            out[b, h] = (w @ V[h * n_kv // H]) / w.sum()
    return out


def prefill(q: np.ndarray, k: np.ndarray, v: np.ndarray, cu, scale=HEAD ** -0.5) -> np.ndarray:
    """q [T, H, 128], k, v [T, n_kv, 128]; causal attention in each of the packed sequences; rows of no
    sequence are NaN."""
    T, H, _ = q.shape
    n_kv = k.shape[1]
    out = np.full((T, H, HEAD), np.nan)
    for b in range(len(cu) - 1):
        s = slice(int(cu[b]), int(cu[b + 1]))
        n = s.stop - s.start
        for h in range(H):
            e = scale * (q[s, h] @ k[s, h * n_kv // H].T)
            e[np.triu_indices(n, 1)] = -np.inf
            if n:
                vh = v[s, h * n_kv // H]
                if np.isfinite(vh).all() and np.isfinite(k[s, h * n_kv // H]).all():
                    w = np.exp(e - e.max(axis=1, keepdims=True))
                    out[s, h] = (w @ vh) / w.sum(axis=1, keepdims=True)
                    continue
                for i in range(n):              # a row takes no part in the keys after it (0 * NaN is NaN)
                    w = np.exp(e[i, :i + 1] - e[i, :i + 1].max())
                    out[s.start + i, h] = (w @ vh[:i + 1]) / w.sum()
    return out


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """To the nearest e4m3 value (ties to even), saturating at +-448; NaN stays."""
    x = np.clip(np.asarray(x, np.float64), -E4M3_MAX, E4M3_MAX)
    unit = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.rint(x / unit) * unit
