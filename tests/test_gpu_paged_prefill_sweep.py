"""Seeded random calls of paged_prefill_attention against 64 bits: rows of any length and number of
new tokens, single tokens among them, head layouts, page sizes, rows before and behind; the
workspace ends exactly where the call is told, and nothing behind it is written."""
import random

import numpy as np
import pytest
import torch

from prompt_cases import assert_within
from turn_cases import Cache, run_chunk

pytestmark = pytest.mark.gpu


def _case(seed):
    rng = random.Random(seed)
    hkv = rng.choice([1, 1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8, 16, 32] if hkv < 3 else [1, 2, 4])
    rows = rng.choice([1, 2, 3, 5, 9, 30, 64, 65, 66, 100, 190])
    longest = rng.choice([5, 40, 200, 700, 2500]) if rows < 20 else rng.choice([5, 40, 200, 500])
    kind = rng.choice(["single", "few", "all", "mixed", "mixed"])
    lens, new = [], []
    for i in range(rows):
        n = rng.randint(0, longest) if rng.random() < 0.9 else longest
        most = {"single": 1, "few": 6, "all": n, "mixed": n if i % 7 == 0 else 1}[kind]
        lens.append(n)
        new.append(min(n, rng.randint(0, most) if kind == "few" else most))
    if sum(new) * hq > 40000:  # the reference's time
        new = [min(x, max(1, 40000 // hq // rows)) if x else 0 for x in new]
    if not sum(new):
        lens[0], new[0] = max(lens[0], 1), 1
    page = rng.choice([1, 3, 8, 16, 16, 24, 32, 40, 100, 128])
    return Cache(lens, new, hq, hkv, page, rng.choice([torch.float16, torch.bfloat16]), seed, lead=rng.choice([0, 3]), trail=rng.choice([0, 5]))


@pytest.mark.parametrize("seed", range(60))
def test_random_calls(ext, gpu, seed):
    cache = _case(seed)
    floats = ext.paged_prefill_workspace_floats(len(cache.lens), cache.q.shape[0], cache.hq, cache.hkv)
    space = torch.full((floats + 4096,), 7.0, device=gpu)
    space[:floats] = float("nan")
    out = run_chunk(ext, cache, gpu, workspace=space[:floats])
    again = run_chunk(ext, cache, gpu, workspace=space[:floats])
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert (space[floats:] == 7.0).all()
    want, *rest = cache.want()
    inside = np.zeros(len(want), dtype=bool)
    for s, e in zip(cache.offsets, cache.offsets[1:]):
        inside[s:e] = True
    assert (out[~torch.from_numpy(inside)].float() == 7.0).all()
    what = f"seed {seed}: {len(cache.lens)} rows up to {max(cache.lens)}, {sum(cache.new)} tokens, {cache.hq} / {cache.hkv}, pages of {cache.page}"
    assert_within(out.cpu()[torch.from_numpy(inside)], want[inside], cache.bound(want, *rest)[inside], what)


def test_many_rows_just_past_a_part(ext, gpu):
    """Rows whose tiles pass the cut by little, of both classes: the most states a call can have."""
    for rows, new, n in ((64, 1, 2100), (64, 40, 300), (200, 8, 70), (150, 9, 1000)):
        cache = Cache([n] * rows, [new] * rows, 4, 1, 16, torch.bfloat16, rows + n)
        floats = ext.paged_prefill_workspace_floats(rows, rows * new, 4, 1)
        space = torch.full((floats + 4096,), 7.0, device=gpu)
        out = run_chunk(ext, cache, gpu, workspace=space[:floats])
        assert (space[floats:] == 7.0).all()
        want, *rest = cache.want()
        assert_within(out, want, cache.bound(want, *rest), f"{rows} rows of {n}, {new} new")
