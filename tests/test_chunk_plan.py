"""The parts of paged_prefill_attention fit its workspace and its grid, whatever the lengths: random rows
and rows just past the cut, in every class and layout, against the sizes that the library gives."""
import random

import pytest

import pkv_native
from chunk_plan import cut, grid, plan_floats, states, states_at_most


def _rows(rng):
    hkv = rng.choice([1, 1, 2, 3, 4, 8, 16, 32])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16, 31, 32])
    batch = rng.choice([1, 1, 2, 3, 7, 20, 64, 65, 200, 1000])
    longest = 2 ** rng.randint(5, 24 if batch < 20 else 18)
    most = 2 ** rng.randint(0, 13 if batch < 20 else 7)
    kind = rng.choice(["any", "equal", "one", "small", "one size"])
    lens = [rng.randint(1, longest) if kind == "any" else longest for _ in range(batch)]
    new = [rng.randint(0, most) if kind != "one size" else most for _ in range(batch)]
    if kind == "small":
        new = [rng.randint(0, max(32 // group, 1)) for _ in range(batch)]
    if kind == "one":
        lens[1:] = [rng.randint(1, 64) for _ in lens[1:]]
    new = [min(n, size) for size, n in zip(lens, new)]
    if not sum(new):
        new[0] = 1
    return lens, new, group, hkv


def _past_the_cut(rng, lens, new, group, hkv, small):
    """Rows of a class brought to where they just have one part more."""
    for _ in range(6):
        large, little, rows = cut(lens, new, group, hkv)
        most = little if small else large
        edge = 32 * (most if small else 2 * most - most // 2 - 1) + 1
        moved = [max(min(edge + rng.randint(-40, 40), 2 ** 30), n) if r[2] == small and n else size for size, n, r in zip(lens, new, rows)]
        if moved == lens:
            break
        lens = moved
    return lens


@pytest.mark.parametrize("seed", range(40))
def test_parts_fit(seed):
    rng = random.Random(seed)
    seen = set()
    for _ in range(150):
        lens, new, group, hkv = _rows(rng)
        if rng.random() < 0.5:
            lens = _past_the_cut(rng, lens, new, group, hkv, rng.random() < 0.5)
        tokens, batch = sum(new), len(lens)
        rows, units = states(lens, new, group, hkv)
        assert rows * hkv <= states_at_most(tokens, group), (lens[:5], new[:5], group, hkv)
        assert units * hkv <= grid(batch, tokens, group, hkv), (lens[:5], new[:5], group, hkv)
        large = cut(lens, new, group, hkv)[0]
        seen.add("short" if large < 192 else "long" if large == 192 else "longer")
    assert len(seen) > 1


@pytest.mark.parametrize("batch", [1, 64, 65, 1000])
@pytest.mark.parametrize("tokens,group", [(1, 1), (8, 4), (9, 4), (31, 4), (32, 4), (5000, 4), (3, 32)])
def test_workspaces_hold_a_state_for_each(batch, tokens, group):
    """Sizes as without a GPU, where 256 compute units are assumed."""
    size = pkv_native.lib().pkv_paged_prefill_workspace_bytes(batch, tokens, 2 * group, 2)
    assert size == 4 * (plan_floats(batch) + 130 * states_at_most(tokens, group))
    assert size < 200 * 10 ** 6 and states_at_most(tokens, group) * 130 < 2 ** 32
