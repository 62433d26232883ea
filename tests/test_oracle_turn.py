"""The reference of the operators for a further turn, held against other ways to the same results."""
import numpy as np
import pytest
import torch

from oracle import prompt, turn
from turn_cases import Cache, angles


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", [16, 96, 128])
def test_rotation_is_a_complex_product_that_keeps_lengths_and_distances(pairs, rot):
    rng = np.random.default_rng(rot)
    x, table = rng.standard_normal((6, 2, 128)), angles(50, rot).double().numpy()
    got, size = turn.norm_rope(x, None, table, range(6), 0.0, pairs)
    view = (lambda a: a[..., :rot].reshape(6, 2, -1, 2)) if pairs else (lambda a: np.stack([a[..., :rot // 2], a[..., rot // 2:rot]], -1))
    turned = (view(x) @ [1, 1j]) * (table[:6, :rot // 2] + 1j * table[:6, rot // 2:])[:, None]
    assert np.allclose(view(got) @ [1, 1j], turned) and (got[..., rot:] == x[..., rot:]).all()
    assert (size >= np.abs(got) - 1e-12).all()
    # products of a query and a key depend on the distance of their positions
    q, k = rng.standard_normal((2, 1, 1, 128))
    dots = [float((turn.norm_rope(q, None, table, [p], 0.0, pairs)[0] * turn.norm_rope(k, None, table, [p + 7], 0.0, pairs)[0]).sum())
            for p in (0, 3, 40)]
    assert np.allclose(dots, dots[0], atol=1e-5)


def test_norm_and_weights():
    rng = np.random.default_rng(1)
    x, w, still = rng.standard_normal((3, 4, 128)), rng.standard_normal((4, 128)), np.concatenate([np.ones((9, 64)), np.zeros((9, 64))], 1)
    got, _ = turn.norm_rope(x, w, still, [0, 5, 99], 0.5, False)
    assert np.allclose(got, w * x / np.sqrt(np.mean(x ** 2, -1, keepdims=True) + 0.5))


def test_whole_rows_are_the_prompt_attention():
    cache = Cache([40, 7, 100], [40, 7, 100], 4, 2, 16, torch.float16, seed=3)
    got = cache.want()[0]
    k, v = (np.concatenate([np.stack([pool.double().numpy()[cache.table[b, i // 16], :, i % 16] for i in range(n)])
                            for b, n in enumerate(cache.lens)]) for pool in (cache.k, cache.v))
    assert np.allclose(got, prompt.prefill(cache.q.double().numpy(), k, v, cache.offsets)[0])


def test_forked_rows_hold_what_their_parents_held_and_return_every_page():
    """Forks, frees in any order and a compaction: no page is lost, given twice, or freed while held."""
    rng = np.random.default_rng(5)
    page, columns, pages = 16, 8, 60
    table, shares = np.full((12, columns), -1), [0] * pages
    free, lens = list(rng.permutation(pages)), [0] * 12
    num, content = pages, np.arange(pages)
    for row, n in ((0, 50), (1, 96)):
        lens[row] = n
        for c in range(-(-n // page)):
            num -= 1
            table[row, c] = free[num]
    held = lambda r: [content[p] for p in table[r, :lens[r] // page]]
    for parents, children in (([0, 0, 1], [2, 3, 4]), ([2, 4, 4], [5, 6, 7])):
        table, shares, left, src, dst = turn.fork_rows(parents, children, lens, table, shares, free, num, page)
        for p, c, s, d in zip(parents, children, src, dst):
            lens[c] = lens[p]
            assert held(c) == held(p) and (d >= 0) == (lens[p] % page > 0)
            if d >= 0:
                content[d] = content[s]
        num = left
    in_use = {int(p) for r in range(12) for p in table[r, :-(-lens[r] // page)]}
    assert len(in_use) == pages - num and not in_use & {int(p) for p in free[:num]}
    before = [held(r) for r in range(8)]
    page_map, table, shares, free, num, src, dst = turn.compact_pages(table, shares, free, num, pages // 2)
    table = np.array(table)
    for s, d in zip(src, dst):
        if d >= 0:
            content[d] = content[s]
    assert [held(r) for r in range(8)] == before and sorted(free[:num]) == list(range(pages - num, pages))
    for rows in ([0, 4], [1, 1, 3], [7, 6, 5, 2]):
        shares, free, num = turn.free_rows(rows, lens, table, shares, free, num, page)
        for r in rows:
            lens[r] = 0
    assert num == pages and sorted(free) == list(range(pages)) and not any(shares)
