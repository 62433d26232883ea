"""How paged_prefill_attention cuts rows into parts, restated from its comments: for tests that hold the
parts against the workspace and the grid, and against what the kernels write."""
from __future__ import annotations

import numpy as np

KEYS, ROWS, WAVE_ROWS, MIN_TILES, LONG_PART, FINER = 32, 128, 32, 2, 192, 4
F = np.float32


def parts_wanted(units=256):
    return 2 * units


def states_at_most(tokens, group, units=256):
    """Rows of states in the workspace, from its size: 130 floats each beside the plan of many rows."""
    small, large = min(tokens * group, WAVE_ROWS), min(tokens * group, ROWS)
    few = tokens * group <= WAVE_ROWS
    return 2 * parts_wanted(units) * small + (0 if few else -(-4 * FINER * parts_wanted(units) * large // 3))


def plan_floats(batch):
    return (5 + 4 * batch + 3) // 4 * 4 if batch > 64 else 0


def grid(batch, tokens, group, hkv, units=256):
    parts = parts_wanted(units) * (1 if tokens * group <= WAVE_ROWS else 1 + FINER)
    return (tokens * group // ROWS + batch) * hkv + (parts // hkv + 1 + FINER) * hkv


def cut(lens, new, group, hkv, units=256):
    """The most tiles of a part, of large and of small rows, and each row's (blocks, tiles, small)."""
    rows = [(-(-n * group // ROWS), -(-size // KEYS), n * group <= WAVE_ROWS) for size, n in zip(lens, new)]
    scale = F(F(hkv) / F(parts_wanted(units)) * F(1.0001))
    large, small = (F(F(sum(b * t for b, t, s in rows if s == which)) * scale) for which in (False, True))
    whole = lambda c: max(MIN_TILES, int(np.ceil(c)))
    return whole(max(large * F(1 / FINER), min(large, F(LONG_PART)))), whole(small), rows


def parts(lens, new, group, hkv, units=256):
    """For each row its number of parts and their tiles."""
    large, small, rows = cut(lens, new, group, hkv, units)
    out = []
    for blocks, tiles, is_small in rows:
        most = small if is_small else large
        count = max((tiles + (most - 1 if is_small else most // 2)) // most, 1)
        out.append((count, max(-(-tiles // count), 1)))
    return out


def states(lens, new, group, hkv, units=256):
    """Rows of states of one KV head, and units of work of one."""
    counts = [c for c, _ in parts(lens, new, group, hkv, units)]
    return (sum(n * group * c for n, c in zip(new, counts) if c > 1), sum(-(-n * group // ROWS) * c for n, c in zip(new, counts)))


def written_states(lens, new, group, hkv, units=256):
    """Which rows of states (of each KV head alike) the parts write: not those of parts behind the last key
    that a block of 128 (token, head) rows sees, nor those of blocks that one part holds."""
    total, _ = states(lens, new, group, hkv, units)
    out, first = np.zeros(total, dtype=bool), 0
    for size, n, (count, tiles) in zip(lens, new, parts(lens, new, group, hkv, units)):
        if count == 1:
            continue
        rows = n * group
        for block in range(-(-rows // ROWS)):
            at, end = block * ROWS, min((block + 1) * ROWS, rows)
            seen = -(-max(min(size - n + (end - 1) // group, size - 1) + 1, 0) // KEYS)
            for part in range(count):
                if seen > tiles and part * tiles < seen:
                    out[first + part * rows + at:first + part * rows + end] = True
        first += rows * count
    return out
