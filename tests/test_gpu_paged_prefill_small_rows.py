"""paged_prefill_attention of rows whose (token, head) pairs are one wave's (at most 32 of a KV head: decoding
rows, guessed tokens): in bf16 the weights enter the product in two terms, as in the decode ops, alone and
in calls that hold larger rows too."""
import numpy as np
import pytest
import torch

from prompt_cases import U, assert_within, attention_tolerance
from turn_cases import Cache, run_chunk

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _check(cache, out, what):
    """Half a step of each product's operands: two bf16 terms hold 2^-16 of a weight."""
    want, weight, vmax, score = cache.want()
    group, longest = cache.hq // cache.hkv, max(cache.lens)
    tiny = longest * 2.0 ** -25 * vmax if cache.dtype == F16 else np.zeros_like(vmax)
    small = np.zeros(len(want), dtype=bool)
    for s, e in zip(cache.offsets, cache.offsets[1:]):
        small[s:e] = (e - s) * group <= 32
    for rows, p_step, name in ((small, 2.0 ** -16 if cache.dtype == BF16 else U[F16], "small"), (~small, U[cache.dtype], "large")):
        if rows.any():
            bound = attention_tolerance(want[rows], weight[rows], score[rows], longest, cache.dtype, p_step, tiny[rows])
            assert_within(out.cpu()[torch.from_numpy(rows)], want[rows], bound, f"{what}, {name}")


ROWS = [([2011], [5]), ([1], [1]), ([33, 64, 65], [1, 2, 3]), ([900, 40, 2000, 1], [1] * 4), ([1500, 700] + [100 + 37 * i for i in range(20)], [200, 130] + [1] * 20),
        ([300] * 70, [1] * 70), ([50 + 11 * i for i in range(90)], [1 + i % 4 for i in range(90)]), ([8, 31, 32], [8, 8, 8])]


@pytest.mark.parametrize("lens,new", ROWS, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("hq,hkv,page", [(8, 2, 16), (32, 1, 24), (5, 5, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weights_of_small_rows(ext, gpu, lens, new, hq, hkv, page, dtype):
    cache = Cache(lens, new, hq, hkv, page, dtype, seed=sum(lens) + hq)
    _check(cache, run_chunk(ext, cache, gpu), f"{len(lens)} rows up to {max(lens)}, {hq} / {hkv}")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_token_a_row_as_exact_as_the_decode_op(ext, gpu, dtype):
    """Both within the bound of two-term weights (bf16) of the exact result."""
    cache = Cache([900, 40, 2000, 1, 333], [1] * 5, 8, 2, 16, dtype, seed=12, stale=0.0)
    _check(cache, run_chunk(ext, cache, gpu), "attention over pages")
    q, k, v, table, lens, _ = cache.on(gpu)
    ref = torch.zeros_like(q)
    ws = torch.empty(ext.workspace_floats(5, 8, 4), device=gpu)
    ext.paged_attention_masked(q, k, v, table, lens, ref, ws, 2000, 16, 4)
    _check(cache, ref, "decode")


@pytest.mark.parametrize("hq,hkv,more", [(8, 2, 0), (16, 1, 40)])
def test_nonfinite_values_beside_two_terms(ext, gpu, hq, hkv, more):
    """Values that are not finite reach the tokens that see them, in small rows too."""
    cache = Cache([150, 64, 70] + [5] * more, [2, 1, 2] + [1] * more, hq, hkv, 16, BF16, seed=5)
    want, weight, vmax, score = cache.want()
    bound = attention_tolerance(want, weight, score, 150, BF16, 2.0 ** -16, 0.0)
    group = hq // hkv
    for row, pos, head, dim, x, sees in ((0, 149, 0, 3, float("inf"), [1]), (0, 0, 0, 9, float("nan"), [0, 1]), (2, 69, hkv - 1, 0, -float("inf"), [4]),
                                           (0, 50, 0, 40, float("inf"), [0, 1]), (0, 20, 0, 41, -float("inf"), [0, 1]), (1, 63, 0, 1, float("inf"), [2])):
        page, off = cache.place(row, pos)
        cache.v[page, head, off, dim] = x
        for t in sees:
            want[t, head * group:(head + 1) * group, dim] = x
    out = run_chunk(ext, cache, gpu)
    assert_within(out, want, bound, "nonfinite")
