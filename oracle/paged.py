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


# --- a cache under scales of blocks, pages handed out, pages selected -------------------------------

BLOCK = 16


def block_scale(amax: float) -> float:
    """The smallest power of two s, 2^-126 at least, with amax <= 448 s."""
    s = 2.0 ** -126
    while amax > E4M3_MAX * s:
        s *= 2
    return s


def append_blocks(values: np.ndarray, scales: np.ndarray, x: np.ndarray, rows, table, page: int) -> None:
    """x [T, n_kv, 128] float64 stored in values [n_pages, n_kv, page, 128] (what the codes stand for without
    their scale) under scales [n_pages, n_kv, page / 16], both in place; rows: [(row, sequence, position)]."""
    blocks = {}
    for t, b, pos in rows:
        blocks.setdefault((b, pos // BLOCK), []).append((pos, t))
    for (b, _), new in blocks.items():
        new.sort()
        pos0 = new[0][0]
        p, r0 = int(table[b][pos0 // page]), pos0 % page // BLOCK * BLOCK
        before = pos0 % BLOCK
        for h in range(values.shape[1]):
            got = np.stack([x[t, h] for _, t in new])
            finite = np.abs(got[np.isfinite(got)])
            s = block_scale(finite.max() if finite.size else 0.0)
            if before:
                was = float(scales[p, h, r0 // BLOCK])
                s = max(s, 2.0 ** max(-126, int(np.ceil(np.log2(was)))) if 0 < was < np.inf else 0.0)
                values[p, h, r0:r0 + before] = round_e4m3(values[p, h, r0:r0 + before] * (was / s))
            scales[p, h, r0 // BLOCK] = s
            for (pos, _), v in zip(new, got):
                values[p, h, pos % page] = np.where(np.isfinite(v), round_e4m3(np.where(np.isfinite(v), v, 0.0) / s), np.nan)


def assign(lens, new_lens, table, free_pages, free_count: int, page: int, packed: bool):
    """One step of the pages' life, one sequence after another; table and free_pages (lists) in place."""
    stack = list(free_pages[:free_count])
    new = [1] * len(lens) if new_lens is None else [int(n) for n in new_lens]
    for b, n in enumerate(new):
        if n < 0 <= lens[b]:
            stack += [int(i) for i in table[b][:-(-int(lens[b]) // page)]]
    free_pages[:len(stack)] = stack
    room = len(stack)
    start, kv, after, slots, cu = [], [], [], [], [0]
    for b, n in enumerate(new):
        have, total = -(-max(0, int(lens[b])) // page), int(lens[b]) + max(0, n)
        ok = lens[b] >= 0 and n > 0 and total <= len(table[b]) * page
        need = -(-total // page) - have if ok else 0
        room -= need
        ok = ok and (need == 0 or room >= 0)
        if ok:
            for j in range(need):
                table[b][have + j] = stack.pop()
        start.append(int(lens[b]) if ok else -1)
        kv.append(total if ok else 0)
        after.append(-1 if lens[b] >= 0 and n < 0 else total if ok else int(lens[b]))
        n_rows = max(0, n) if packed else 1
        slots += [int(table[b][(int(lens[b]) + i) // page]) * page + (int(lens[b]) + i) % page if ok else -1 for i in range(n_rows)]
        cu.append(cu[-1] + n_rows)
    return {"start_pos": start, "kv_lens": kv, "cu_seqlens": cu if packed else None, "slots": slots, "lens": after,
            "free_count": [len(stack)]}


def page_bounds(values: np.ndarray) -> np.ndarray:
    """Minimum and maximum over the positions of pages [n, n_kv, page, 128]; NaN where one is.  [n, n_kv, 2, 128]."""
    return np.stack((values.min(axis=2), values.max(axis=2)), axis=2)


def select(q: np.ndarray, bounds: np.ndarray, table_row, n: int, page: int, n_select: int):
    """The places of the pages that a token attends: q [H, 128], bounds [n_pages, n_kv, 2, 128]; a list per KV head."""
    P, n_kv = -(-n // page), bounds.shape[1]
    if P <= n_select:
        return [list(range(P))] * n_kv
    group, kept = q.shape[0] // n_kv, []
    for g in range(n_kv):
        lo, hi = (bounds[np.asarray(table_row[:P - 1]), g, i] for i in range(2))
        score = np.full(P - 1, -np.inf, np.float32)
        for x in q[g * group:(g + 1) * group]:
            score = np.maximum(score, (hi @ np.maximum(x, 0) + lo @ np.minimum(x, 0)).astype(np.float32))
        order = sorted(range(P - 1), key=lambda p: (0, 0.0, p) if np.isnan(score[p]) else (1, -score[p], p))
        kept.append(sorted(order[:n_select - 1]) + [P - 1])
    return kept


def decode_selected(q, k_pages, v_pages, table, lens, kept, scale=HEAD ** -0.5) -> np.ndarray:
    """decode over the pages kept[b][g] of each sequence and KV head."""
    B, H, _ = q.shape
    n_kv, page = k_pages.shape[1:3]
    out = np.zeros((B, H, HEAD))
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        for g in range(n_kv):
            end = len(kept[b][g]) * page - (-(-n // page) * page - n)
            heads = slice(g * (H // n_kv), (g + 1) * (H // n_kv))
            ids = [[int(table[b][p]) for p in kept[b][g]]]
            out[b, heads] = decode(q[b:b + 1, heads], k_pages[:, g:g + 1], v_pages[:, g:g + 1], ids, [end], scale)[0]
    return out
