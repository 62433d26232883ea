"""Seeded inputs and tolerances shared by the tests of the operators between a prompt and the
cache (CPU tensors)."""
from __future__ import annotations

import numpy as np
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
F32 = 2.0 ** -24


def packed_inputs(lengths, hq, hkv, dtype, seed, lead=0, trail=0):
    """Column ranges q, k, v of one fused projection [lead + tokens + trail, (hq + 2 hkv), 128],
    and the sequences' offsets."""
    gen = torch.Generator().manual_seed(seed)
    tokens = lead + sum(lengths) + trail
    qkv = torch.randn(tokens, hq + 2 * hkv, 128, generator=gen).to(dtype)
    offsets = np.concatenate([[0], np.cumsum(lengths)]) + lead
    return qkv, torch.tensor(offsets, dtype=torch.int32)


def split_qkv(qkv, hq, hkv):
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def attention_tolerance(out, weight, score, tokens, dtype, p_step, tiny):
    """Bound on |kernel - exact| per element.

    * The output's rounding: half a step of its type, and below its normal range half a step of
      the subnormals, which are 2^-24 apart in fp16 and 2^-133 in bf16.
    * Weights p_j enter the product with V rounded to `p_step` relative (half a step of the
      product's operands): p_step * sum p_j |v_j| in the numerator, and at most p_step * |out|
      more where the sum is of the rounded weights.
    * A score is a sum of 128 products in 32 bits, off by at most 128 * 2^-24 * sum |q k| /
      sqrt(128) (order free), and then scaled, shifted and exponentiated with a few more
      roundings of values of up to |x| + 100 in log2: delta.  Relative errors of the weights of
      up to delta move the quotient by at most 2 delta sum p_j |v_j|.
    * The sums over the tokens in 32 bits: each at most (tokens + 16) 2^-24 of its weights,
      numerator and denominator.
    * `tiny`: what weights below the operand type's normal range may lose in all.
    """
    delta = 130 * F32 * score[..., None] + 64 * F32 * (1 + score[..., None]) + 200 * F32
    sums = 2 * (tokens + 16) * F32
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    return U[dtype] * np.abs(out) + least + (1 + U[dtype]) * ((p_step + 2 * delta + sums) * weight + p_step * np.abs(out) + tiny)


def assert_within(got, want, bound, what=""):
    got = got.double().cpu().numpy()
    finite = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN in other places"
    assert (got[~finite & ~np.isnan(want)] == want[~finite & ~np.isnan(want)]).all(), what
    ratio = np.abs(got[finite] - want[finite]) / np.broadcast_to(bound, want.shape)[finite]
    worst = float(ratio.max()) if ratio.size else 0.0
    print(f"{what}: at most {worst:.3f} of the bound")
    assert worst <= 1.0, (what, worst)


def shortage_and_retry(build):
    """The documented answer to a list that runs out: the step is not used, rows are left out or
    pages returned, and it is built again from the same lengths and table.  `build(cached, lens,
    free, num_free, table, slots, page_size)` gives (table, offsets, slots, num_free_out) as lists."""
    ps, columns, free = 16, 6, [7, 3, 9, 4, 1, 8] + [-99] * 6  # 3 are held by row 0, 5 and 6 by row 1
    table = [[0, 2, 11, -1, -1, -1], [5, 6, -1, -1, -1, -1], [-1] * columns]
    cached, lens = [45, 20, 0], [50, 70, 33]  # 1 + 3 + 3 pages, and 6 are free

    def step(table, lens, free, num_free):
        new = [max(n - c, 0) for n, c in zip(lens, cached)]
        table, offsets, slots, left = build(cached, lens, free, num_free, table, sum(new), ps)
        assert offsets == [sum(new[:i]) for i in range(4)]
        return table, slots, left

    table, slots, left = step(table, lens, free, 6)
    assert left == -1 and slots[-1] == -1
    # row 1 waits: the others have their pages, and its own are untouched
    t1, slots, left = step(table, [50, 20, 33], free, 6)
    held = [t1[0][:4], t1[1][:2], t1[2][:3]]
    assert left == 2 and min(slots) >= 0 and held == [[0, 2, 11, 8], [5, 6], [1, 4, 9]]
    # or two pages come back, at free_pages[num_free] on: everything fits, each page once
    free[6:8] = [20, 21]
    t2, slots, left = step(table, lens, free, 8)
    held = t2[0][:4] + t2[1][:5] + t2[2][:3]
    assert left == 1 and min(slots) >= 0 and len(set(held)) == len(held) and min(held) >= 0
    assert t2[0][:3] == [0, 2, 11] and t2[1][:2] == [5, 6]
    want = [t2[b][p // ps] * ps + p % ps for b in range(3) for p in range(cached[b], lens[b])]
    assert slots == want
