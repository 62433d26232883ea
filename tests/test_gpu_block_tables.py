"""build_block_tables against plain loops: integers, so every entry must be equal."""
import numpy as np
import pytest
import torch

from oracle import prompt
from prompt_cases import shortage_and_retry

pytestmark = pytest.mark.gpu


def _i32(x, gpu):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=gpu)


def _check(ext, gpu, cached, lens, free, num_free, table, slots, page_size):
    table = np.asarray(table, dtype=np.int64)
    t, out = _i32(table, gpu), torch.full((slots,), 77, dtype=torch.int32, device=gpu)
    off, left = _i32([77] * (len(cached) + 1), gpu), _i32([77], gpu)
    given = [_i32(x, gpu) for x in (cached, lens, free)] + [_i32([num_free], gpu)]
    before = [x.clone() for x in given]
    want = prompt.build_block_tables(cached, lens, free, num_free, table, slots, page_size)
    for _ in range(2):  # a repeated call gives the same
        ext.build_block_tables(*given, t, off, out, left, page_size)
        for got, w in zip((t, off, out, left), want):
            assert torch.equal(got.cpu().long().reshape(-1), torch.as_tensor(w).reshape(-1).long())
    assert all(torch.equal(a, b) for a, b in zip(given, before))


def _random(rng, rows, hi, page_size, columns, grow):
    cached = rng.integers(0, hi + 1, rows) * (rng.random(rows) < 0.5)
    lens = np.minimum(cached + (1 if grow == "step" else rng.integers(0, hi + 1, rows)), columns * page_size + 5)
    lens = np.maximum(lens, 0)
    free = rng.permutation(rows * columns)
    table = rng.integers(0, rows * columns, (rows, columns))
    return cached, lens, free, table


@pytest.mark.parametrize("rows,hi,page_size,columns,grow", [
    (1, 1, 16, 1, "step"), (1, 40, 16, 7, "prompt"), (3, 100, 8, 30, "prompt"), (64, 300, 16, 40, "step"),
    (65, 50, 24, 5, "prompt"), (513, 60, 16, 8, "prompt"), (1500, 9, 1, 20, "prompt"), (2, 5000, 128, 90, "prompt")])
def test_tables_match_the_loops(ext, gpu, rows, hi, page_size, columns, grow):
    rng = np.random.default_rng(rows * 7 + hi)
    cached, lens, free, table = _random(rng, rows, hi, page_size, columns, grow)
    new = int(np.maximum(lens - cached, 0).sum())
    for slots in (new, new + 37, max(new - 3, 0)):
        _check(ext, gpu, cached, lens, free, len(free), table, slots, page_size)


def test_no_rows_no_tokens_no_pages(ext, gpu):
    _check(ext, gpu, [], [], [1, 2], 2, np.zeros((0, 4)), 5, 16)
    _check(ext, gpu, [0, 3], [0, 3], [1, 2], 2, np.zeros((2, 4)), 0, 16)
    _check(ext, gpu, [0], [3], [], 0, np.zeros((1, 4)), 3, 16)


def test_the_list_runs_out(ext, gpu):
    _check(ext, gpu, [0, 5, 0], [20, 50, 90], [3, 1, 2, 9, 8], 4, np.full((3, 8), 6), 160, 16)
    _check(ext, gpu, [0], [20], [3, 1], -3, np.full((1, 8), 6), 20, 16)   # counts as none
    _check(ext, gpu, [0], [50], [3, 1], 99, np.full((1, 8), 6), 50, 16)   # at most the list


def test_a_step_is_built_again_after_a_shortage(ext, gpu):
    def build(cached, lens, free, num_free, table, slots, page_size):
        t, out, off, left = _i32(table, gpu), _i32([77] * slots, gpu), _i32([77] * (len(cached) + 1), gpu), _i32([77], gpu)
        ext.build_block_tables(_i32(cached, gpu), _i32(lens, gpu), _i32(free, gpu), _i32([num_free], gpu), t, off, out, left, page_size)
        return t.tolist(), off.tolist(), out.tolist(), left.item()

    shortage_and_retry(build)


def test_shrinking_negative_and_unassigned_rows(ext, gpu):
    # a row that shrinks, negative lengths, a cached page without an id, a row past its table
    _check(ext, gpu, [40, -7, 10, 0], [8, 12, 20, 200], list(range(50)), 50,
           [[5, 6, 7], [-9, -9, -9], [-1, -9, -9], [-9, -9, -9]], 250, 16)


def test_slots_past_int32_are_dropped(ext, gpu):
    page = (2 ** 31 - 1) // 16
    _check(ext, gpu, [0, 3], [40, 20], [1, page, page + 1, page - 1], 4, [[0] * 3, [page, 0, 0]], 57, 16)


def test_a_captured_call_follows_its_inputs(ext, gpu):
    rng = np.random.default_rng(5)
    rows, columns, ps, slots = 33, 20, 16, 1200
    cached, lens, free, table = _random(rng, rows, 60, ps, columns, "prompt")
    c, l, f, n = _i32(cached, gpu), _i32(lens, gpu), _i32(free, gpu), _i32([len(free)], gpu)
    t, off, out, left = _i32(table, gpu), _i32([0] * (rows + 1), gpu), _i32([0] * slots, gpu), _i32([0], gpu)

    def call():
        ext.build_block_tables(c, l, f, n, t, off, out, left, ps)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(4):
        cached, lens, free, table = _random(np.random.default_rng(seed), rows, 60, ps, columns, "prompt")
        for dst, src in ((c, cached), (l, lens), (f, free), (t, table)):
            dst.copy_(_i32(src, gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = prompt.build_block_tables(cached, lens, free, len(free), table, slots, ps)
        for got, w in zip((t, off, out, left), want):
            assert torch.equal(got.cpu().long().reshape(-1), torch.as_tensor(w).reshape(-1).long())
