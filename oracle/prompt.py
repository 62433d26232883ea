"""Reference results of the operators between a prompt and the cache (CPU, 64 bits; test
infrastructure only): block tables and slots, causal attention over packed prompts, packed
K/V writes into 2-byte and block-scaled fp8 pools, and decode over the latter.

Written from the operators' definitions, row by row and in plain loops.
"""
from __future__ import annotations

import math

import numpy as np

HEAD_DIM = 128
INT32_MAX = 2 ** 31 - 1
SCALE_EXP = 60
E4M3_MAX = 448.0


def build_block_tables(cached_lens, seq_lens, free_pages, num_free, block_table, slots, page_size):
    """(block_table, token_offsets, slot_mapping, num_free_out) as int lists / arrays."""
    table = np.array(block_table, dtype=np.int64)
    batch, columns = table.shape
    avail = min(max(int(num_free), 0), len(free_pages))
    taken, offsets, out = 0, [0], []
    for b in range(batch):
        cached = max(int(cached_lens[b]), 0)
        length = max(int(seq_lens[b]), cached)
        held = min(-(-cached // page_size), columns)
        want = min(-(-length // page_size), columns)
        for column in range(held, want):
            at = avail - 1 - taken
            table[b, column] = free_pages[at] if at >= 0 else -1
            taken += 1
        for pos in range(cached, length):
            column, slot = pos // page_size, -1
            if column < columns and table[b, column] >= 0:
                slot = int(table[b, column]) * page_size + pos % page_size
            out.append(slot if slot <= INT32_MAX else -1)
        offsets.append(offsets[-1] + length - cached)
    out = (out + [-1] * slots)[:slots]
    return table, np.array(offsets), np.array(out, dtype=np.int64), avail - taken


def prefill(q, k, v, offsets):
    """Causal attention of the packed sequences: float64 output (NaN outside every
    sequence) and, for tolerances, per element sum_j p_j |v_j|, the largest |v| of the
    tokens attended to, and per (token, head) the largest sum |q k_j| / sqrt(128)."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    tokens, hq, _ = q.shape
    group = hq // k.shape[1]
    out = np.full(q.shape, np.nan)
    weight, vmax = np.zeros(q.shape), np.zeros(q.shape)
    score = np.zeros(q.shape[:2])
    for b in range(len(offsets) - 1):
        s, e = int(offsets[b]), int(offsets[b + 1])
        if e <= s:
            continue
        mask = np.tril(np.ones((e - s, e - s), dtype=bool))
        for h in range(hq):
            kh, vh = k[s:e, h // group], v[s:e, h // group]
            with np.errstate(invalid="ignore", over="ignore"):
                x = np.where(mask, q[s:e, h] @ kh.T / math.sqrt(HEAD_DIM), -np.inf)
                p = np.exp(x - x.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
            finite = np.where(np.isfinite(vh), vh, 0.0)
            o = p @ finite
            # Values that are not finite reach the tokens from theirs on, and no other.
            for j, d in zip(*np.nonzero(~np.isfinite(vh))):
                with np.errstate(invalid="ignore"):
                    o[j:, d] += vh[j, d]
            out[s:e, h] = o
            weight[s:e, h] = p @ np.abs(finite)
            vmax[s:e, h] = np.maximum.accumulate(np.abs(finite), axis=0)
            score[s:e, h] = np.where(mask, np.abs(q[s:e, h]) @ np.abs(kh).T, 0.0).max(axis=1) / math.sqrt(HEAD_DIM)
    return out, weight, vmax, score


def write_kv(pages, new, slots):
    """The pool [pages, hkv, ps, 128] after the new tokens [tokens, hkv, 128]."""
    pages, new = np.array(pages, dtype=np.float64), np.asarray(new, dtype=np.float64)
    ps = pages.shape[2]
    for t, slot in enumerate(slots):
        if 0 <= slot < pages.shape[0] * ps:
            pages[slot // ps, :, slot % ps] = new[t]
    return pages


def e4m3_round(y):
    """y (float64) to the nearest e4m3 value, ties to even, saturating at 448; NaN stays."""
    y = np.asarray(y, dtype=np.float64)
    mag = np.abs(np.where(np.isfinite(y), y, 0.0))
    e = np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -200))), -6)
    step = 2.0 ** (e - 3)
    r = np.minimum(np.round(mag / step) * step, E4M3_MAX)
    r = np.where(np.isinf(y), E4M3_MAX, r)
    return np.where(np.isnan(y), np.nan, np.copysign(r, y))


def power_of_two(x):
    """The smallest power of two >= x in [2^-60, 2^60], by comparison."""
    for e in range(-SCALE_EXP, SCALE_EXP):
        if not x > 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** SCALE_EXP


def clamp_scale(s):
    return min(max(s, 2.0 ** -SCALE_EXP), 2.0 ** SCALE_EXP) if s == s else 2.0 ** -SCALE_EXP


def write_kv_fp8_block(pages, scales, new, slots):
    """(pool values, scales) of one tensor (K or V) after the new tokens: ``pages``
    [pages, hkv, ps, 128] e4m3 values as float64, ``scales`` [pages, hkv].  A page's tokens
    must be one run of consecutive slots: anything else has no defined result."""
    pages, scales = np.array(pages, dtype=np.float64), np.array(scales, dtype=np.float64)
    new = np.asarray(new, dtype=np.float64)
    ps = pages.shape[2]
    runs = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < pages.shape[0] * ps:
            runs.setdefault(int(slot) // ps, []).append((int(slot) % ps, t))
    for page, run in runs.items():
        first = run[0][0]
        if any(b[0] != a[0] + 1 or b[1] != a[1] + 1 for a, b in zip(run, run[1:])):
            raise ValueError(f"page {page}: tokens that are not one run of consecutive slots")
        for h in range(pages.shape[1]):
            x = np.stack([new[t, h] for _, t in run])
            amax = np.abs(np.where(np.isfinite(x), x, 0.0)).max()
            scale = power_of_two(amax / E4M3_MAX)
            if first > 0:
                old = clamp_scale(scales[page, h])
                scale = max(scale, power_of_two(old))
                if scale != old:
                    pages[page, h, :first] = e4m3_round(pages[page, h, :first] * (old / scale))
            for i, (offset, _) in enumerate(run):
                pages[page, h, offset] = e4m3_round(x[i] / scale)
            scales[page, h] = scale
    return pages, scales


def fp8_block_decode(q, k_pages, v_pages, scales, block_table, seq_lens):
    """Decode over block-scaled pools (values as float64): float64 output and, for
    tolerances, per element sum_j p_j |v_j|; per (row, head) the largest sum |q k_j| /
    sqrt(128), and the largest scale of V times weight relation max_j vs_j p_j."""
    q, k_pages, v_pages, scales = (np.asarray(x, dtype=np.float64) for x in (q, k_pages, v_pages, scales))
    batch, hq, _ = q.shape
    pages, hkv, ps, _ = k_pages.shape
    group = hq // hkv
    scales = np.vectorize(clamp_scale)(scales)
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    score, lead = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for b in range(batch):
        n = min(max(int(seq_lens[b]), 0), block_table.shape[1] * ps)
        if n == 0:
            continue
        ids = np.clip(np.asarray(block_table[b][: -(-n // ps)], dtype=np.int64), 0, pages - 1)
        for h in range(hkv):
            ks = np.repeat(scales[ids, h, 0], ps)[:n]
            vs = np.repeat(scales[ids, h, 1], ps)[:n]
            k = k_pages[ids, h].reshape(-1, HEAD_DIM)[:n] * ks[:, None]
            v = v_pages[ids, h].reshape(-1, HEAD_DIM)[:n] * vs[:, None]
            qh = q[b, h * group:(h + 1) * group]
            x = qh @ k.T / math.sqrt(HEAD_DIM)
            p = np.exp(x - x.max(axis=1, keepdims=True))
            total = p.sum(axis=1, keepdims=True)
            p /= total
            at = slice(h * group, (h + 1) * group)
            out[b, at] = p @ v
            weight[b, at] = p @ np.abs(v)
            score[b, at] = (np.abs(qh) @ np.abs(k).T).max(axis=1) / math.sqrt(HEAD_DIM)
            lead[b, at] = (p * vs).max(axis=1)
    return out, weight, score, lead
