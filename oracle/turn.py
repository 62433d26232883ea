"""Reference results of the operators for a further turn over cached rows (CPU, 64 bits; test
infrastructure only): norm and rotation of q and k, pages shared, freed, moved and copied, and
attention of each row's newest tokens over its pages.

Written from the operators' definitions, row by row and in plain loops.
"""
from __future__ import annotations

import math

import numpy as np

HEAD_DIM = 128


def norm_rope(x, weight, cos_sin, positions, eps, interleaved):
    """x [tokens, heads, 128] normed (weight [128] or [heads, 128]; None: not) and rotated: the
    result, and for tolerances the sum of the magnitudes that each element is made of."""
    x = np.array(x, dtype=np.float64)
    cos_sin = np.asarray(cos_sin, dtype=np.float64)
    half = cos_sin.shape[1] // 2
    with np.errstate(invalid="ignore", over="ignore"):
        if weight is not None:
            mean = (x * x).sum(axis=2, keepdims=True) / HEAD_DIM
            x = x * (1.0 / np.sqrt(mean + eps)) * np.asarray(weight, dtype=np.float64)
        out, size = x.copy(), np.abs(x)
        for t, pos in enumerate(positions):
            pos = min(max(int(pos), 0), cos_sin.shape[0] - 1)
            for i in range(half):
                c, s = cos_sin[pos, i], cos_sin[pos, half + i]
                a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
                out[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
                out[t, :, b] = x[t, :, b] * c + x[t, :, a] * s
                size[t, :, a] = np.abs(x[t, :, a] * c) + np.abs(x[t, :, b] * s)
                size[t, :, b] = np.abs(x[t, :, b] * c) + np.abs(x[t, :, a] * s)
    return out, size


def fork_rows(parents, children, lens, block_table, page_shares, free_pages, num_free, page_size):
    """(block_table, page_shares, num_free_out, copy_src, copy_dst)"""
    table, shares = np.array(block_table, dtype=np.int64), np.array(page_shares, dtype=np.int64)
    batch, columns = table.shape
    avail = min(max(int(num_free), 0), len(free_pages))

    def tokens(p, c):
        if not (0 <= p < batch and 0 <= c < batch and p != c):
            return 0
        return min(max(int(lens[p]), 0), columns * page_size)

    need = sum(tokens(p, c) % page_size > 0 for p, c in zip(parents, children))
    src, dst = [-1] * len(parents), [-1] * len(parents)
    if need > avail:
        return table, shares, avail - need, src, dst
    taken = 0
    for i, (p, c) in enumerate(zip(parents, children)):
        n = tokens(p, c)
        for column in range(n // page_size):
            page = table[c, column] = table[p, column]
            if 0 <= page < len(shares):
                shares[page] += 1
        if n % page_size:
            taken += 1
            src[i], dst[i] = int(table[p, n // page_size]), int(free_pages[avail - taken])
            table[c, n // page_size] = dst[i]
    return table, shares, avail - need, src, dst


def free_rows(rows, lens, block_table, page_shares, free_pages, num_free, page_size):
    """(page_shares, free_pages, num_free_out)"""
    shares, free = np.array(page_shares, dtype=np.int64), list(free_pages)
    batch, columns = np.shape(block_table)
    avail = min(max(int(num_free), 0), len(free))
    seen = set()
    for row in rows:
        if not 0 <= row < batch or row in seen:
            continue
        seen.add(row)
        for column in range(min(-(-max(int(lens[row]), 0) // page_size), columns)):
            page = block_table[row][column]
            if 0 <= page < len(shares):
                shares[page] -= 1
    gone = [p for p in range(len(shares)) if shares[p] < 0]
    for p in gone:
        shares[p] = 0
        if avail < len(free):
            free[avail] = p
            avail += 1
    return shares, free, avail


def compact_pages(block_table, page_shares, free_pages, num_free, copies):
    """(page_map, block_table, page_shares, free_pages, num_free_out, copy_src, copy_dst)"""
    pages = len(page_shares)
    listed = {int(p) for p in free_pages[:min(max(int(num_free), 0), len(free_pages))]}
    used = [p for p in range(pages) if p not in listed]
    holes = [p for p in range(len(used)) if p in listed]
    movers = [p for p in used if p >= len(used)][::-1]
    to = {p: p for p in used}
    to.update(zip(movers, holes))
    page_map = [to.get(p, -1) for p in range(pages)]
    table = [[page_map[p] if 0 <= p < pages else p for p in row] for row in block_table]
    shares = [0] * pages
    for p in used:
        shares[to[p]] = int(page_shares[p])
    free = list(free_pages)
    free[:pages - len(used)] = range(pages - 1, len(used) - 1, -1)
    pad = [-1] * (copies - len(holes))
    return page_map, table, shares, free, pages - len(used), movers + pad, holes + pad


def paged_prefill(q, k_pages, v_pages, block_table, seq_lens, offsets):
    """Attention of each row's newest tokens over its pages: float64 output (NaN outside every
    row's tokens), and as prompt.prefill per element sum_j p_j |v_j|, the largest |v| of the keys
    seen, and per (token, head) the largest sum |q k_j| / sqrt(128)."""
    q, k_pages, v_pages = (np.asarray(x, dtype=np.float64) for x in (q, k_pages, v_pages))
    pages, hkv, ps, _ = k_pages.shape
    group = q.shape[1] // hkv
    out, weight, vmax = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape)
    score = np.zeros(q.shape[:2])
    for b in range(len(offsets) - 1):
        s, e = int(offsets[b]), int(offsets[b + 1])
        if e <= s:
            continue
        total = max(int(seq_lens[b]), 0)
        n = min(total, block_table.shape[1] * ps)
        ids = np.clip(np.asarray(block_table[b][:-(-n // ps)], dtype=np.int64), 0, pages - 1)
        pos = total - (e - s) + np.arange(e - s)
        mask = np.arange(n)[None, :] <= pos[:, None]
        out[s:e] = 0.0
        sees = np.nonzero(mask.any(axis=1))[0]
        if not sees.size:
            continue
        for h in range(q.shape[1]):
            kh = k_pages[ids, h // group].reshape(-1, HEAD_DIM)[:n]
            vh = v_pages[ids, h // group].reshape(-1, HEAD_DIM)[:n]
            with np.errstate(invalid="ignore", over="ignore"):
                x = np.where(mask, q[s:e, h] @ kh.T / math.sqrt(HEAD_DIM), -np.inf)[sees]
                p = np.exp(x - x.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
            finite = np.where(np.isfinite(vh), vh, 0.0)
            o = p @ finite
            for j, d in zip(*np.nonzero(~np.isfinite(vh))):  # it reaches the tokens that see it
                with np.errstate(invalid="ignore"):
                    o[mask[sees, j], d] += vh[j, d]
            out[s + sees, h] = o
            weight[s + sees, h] = p @ np.abs(finite)
            vmax[s + sees, h] = np.abs(finite).max()
            score[s + sees, h] = np.where(mask, np.abs(q[s:e, h]) @ np.abs(kh).T, 0.0).max(axis=1)[sees] / math.sqrt(HEAD_DIM)
    return out, weight, vmax, score
